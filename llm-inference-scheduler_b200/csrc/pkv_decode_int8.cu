// pkv_decode_int8.cu -- decode attention (one query row per sequence) over int8
// pools with one power-of-two scale per (block, KV head).
//
// Replaces the gather of append_and_fetch and _attention with num_new == 1 of
// the reference (mini_engine/paged/block_manager.py:136-141,
// mini_engine/model/qwen2.py:98-128) for such pools.
//
// Mathematics.  With k_j = 2^a_b K_j and v_j = 2^c_b V_j (K, V integers, b the
// block of token j), x_j = (scale 2^a_b) (q . K_j) and
//   o = sum_j softmax(x)_j 2^c_b V_j.
// Scores.  S^T = K Q^T on the integer tensor cores (m16n8k32, 16 tokens as M, the
// 8 query heads of a GQA group as N), which take K's bytes as they lie.  A q row
// is brought by a power of two to integers below 2^22 and split into three signed
// bytes, q = 2^e (65536 A + 256 B + C): exact for fp16 / bf16 elements down to
// 2^-11 / 2^-14 of the row's largest, off by at most 2^-22 of it below and for fp32.  The
// three int32 products are exact; they are joined in fp32.
// Values.  O^T += V^T P^T in fp16 with fp32 sums (m16n8k16).  V's integers are
// exact in fp16, and no conversion instruction makes them: x ^ 0x80 = x + 128
// becomes the low byte of the fp16 1024 + 128 + x (a byte permute), and
// subtracting 1152 is exact.  (fp8 bytes need the conversion pipe, which bounds
// the fp8 kernel at about half of the HBM rate.)  The V scale goes into P as
// P' = p 2^(c_b + n), n per head such that the largest P' so far, the largest
// product of a probability and a scale, lies in 2^6 .. 2^15: fp16 keeps 11 bits of
// the keys down to 2^-20 of that one and an error of 2^-31 of it below.  (With n by
// the largest scale alone, a loud block of no weight took the others' bits: 2.3% off
// at a ratio of 2^20.)  n moves where P' passes 2^15 or the maximum moves, O with it,
// exactly; the row sum takes p itself.  An error of 2^-11 a key is of the size of the
// output's own rounding for 16-bit q; for fp32 q, P' is split into two fp16 parts
// (22 bits) and each product is two MMAs.
// Maximum, sums and O are fp32.
//
// Work split.  The 16-token tiles of all sequences are cut into one contiguous
// range per CTA and the range into one sub-range per team of warps (one warp per
// KV head and chunk of query heads, so the heads of a token are read at about
// the same time).  Each warp streams its tiles through its own ring of
// shared-memory stages by TMA: it fills a stage once its own lanes are done with
// it, so no warp waits for another.  Partial (m, l, O) of a sequence that several
// teams share meet in shared memory at the end of the CTA, those of a sequence
// that several CTAs share in the workspace, joined in CTA order by a second
// launch.
//
// What bounds it: HBM where heads are wide (64 sequences of 4,096 tokens, 32 / 8 x
// 128: 93.5 us, 5.8 TB/s of 6.5 measured for a copy), the instructions of the two
// kinds of tiles at 64 dims and 7 query heads a KV head (64 x 8,192 tokens, 14 / 2
// x 64: 34.0 us, 4.0 TB/s; 64 x 4,096 22.0, with fp32 q 23.0), and for small steps
// the fixed part: about 2 us to the first tile, 1.3 for the join in the CTA, 2.5 for
// the second launch (256 x 1,024: 22.9 us for 67 MB; one sequence of 131,072: 16.0 us
// for 34 MB; of 16: 5.3 us).
#include <algorithm>
#include <atomic>
#include <type_traits>

#include "pkv_common.cuh"
#include "pkv_internal.h"

namespace pkv {

namespace {

constexpr int kD8MaxSeqs = 1024;   // per launch
constexpr int kD8MaxCtas = 296;    // per launch and head group
constexpr float kD8Log2e = 1.4426950408889634f;
constexpr float kD8Slack = 8.f;    // the reference maximum moves by more than this (log2)
// log2 of P' = p vs 2^gain: the largest is brought to 2^kD8LeadP when the gain is set
// and never passes 2^kD8MostP (fp16 ends at 2^16)
constexpr float kD8LeadP = 7.f, kD8MostP = 15.f;
constexpr float kD8MostGain = 119.f;  // p 2^gain stays finite (p <= 2^8)

struct D8Params {
  void* out;
  const void* q;
  int64_t out_stride, q_stride;
  const int8_t* k_pool;
  const int8_t* v_pool;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  int64_t bt_stride;
  const int32_t* context_lens;
  int n_seqs, max_blocks, num_blocks, tiles_per_block;
  int n_q_heads, n_kv_heads, group, chunks;  // chunks of 8 NT query heads per KV head
  int n_groups;                              // n_kv_heads * chunks
  int teams;                                 // per CTA
  int min_tiles;                             // of a CTA's range
  int per_cta;                               // head groups per CTA
  int q_vec;  // q rows take 8-byte (fp32: 16-byte) loads of four elements
  float scale_log2;
  float* part_o;   // [2 * grid][n_q_heads][D]
  float* part_ml;  // [2 * grid][n_q_heads][2]
  int* err;
};

// D = A B + C on int8 (16 x 32 by 32 x 8, int32 sums)
__device__ __forceinline__ void mma16832_s8(int (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k32.row.col.s32.s8.s8.s32 {%0, %1, %2, %3}, {%4, %5, %6, %7},"
      " {%8, %9}, {%0, %1, %2, %3};"
      : "+r"(d[0]), "+r"(d[1]), "+r"(d[2]), "+r"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t pack_s8(int a, int b, int c, int d) {
  return __byte_perm(__byte_perm(a, b, 0x0040), __byte_perm(c, d, 0x0040), 0x5410);
}
// bytes (biased by 128) -> fp16 pairs; magic = 0x64646464
__device__ __forceinline__ uint32_t sub1152(uint32_t h) {
  const __half2 c = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
  const __half2 r = __hsub2(*reinterpret_cast<__half2*>(&h), c);
  return *reinterpret_cast<const uint32_t*>(&r);
}
__device__ __forceinline__ uint32_t i8_lo(uint32_t biased) { return sub1152(__byte_perm(biased, 0x64646464u, 0x4140)); }
__device__ __forceinline__ uint32_t i8_hi(uint32_t biased) { return sub1152(__byte_perm(biased, 0x64646464u, 0x4342)); }

// 2^n for whole n <= 127, exactly; 0 below the normal range
__device__ __forceinline__ float exp2_whole(float n) {
  return __int_as_float((static_cast<int>(fmaxf(n, -127.f)) + 127) << 23);
}

// last s in [0, n) with prefix[s] <= x
__device__ __forceinline__ int d8_find(const int* prefix, int n, int x) {
  int lo = 0, hi = n - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (prefix[mid] <= x) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// stage: K tile, V tile (16 rows x D bytes each, TMA's 64- or 128-byte swizzle)
template <int D> __host__ __device__ constexpr int d8_stage() { return 2 * 16 * D; }
// position of the 16-byte chunk c of row r.  The lanes read K as row g, chunk t
// (D = 128: 2t, 2t + 1) and V 8 bytes at a time in rows 2t + {0, 1, 8, 9}, in an
// order that depends on t's parity: all of them fill all banks.
template <int D> __device__ __forceinline__ int d8_chunk(int r, int c) {
  return D == 64 ? r * 64 + ((c ^ ((r >> 1) & 3)) << 4) : r * 128 + ((c ^ (r & 7)) << 4);
}
// a sum that starts at this int32 is, read as fp32, 1.5 * 2^23 + the sum (up to 2^22)
constexpr int kIntBase = 0x4b400000;
constexpr float kFloatBase = 12582912.f;

template <typename T, int D, int NT, int LIMBS, int WARPS, int STAGES>
__global__ void __launch_bounds__(WARPS * 32, 1)
    decode_int8_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const D8Params p) {
  constexpr int KS = D / 16;          // k-steps of the scores, and m-tiles of O
  constexpr int kHeads = 8 * NT;      // query heads of a warp
  constexpr int kSlot = kHeads * (D + 2);  // floats of a partial: O, then (m, l)
  constexpr int kStage = d8_stage<D>();
  constexpr int kRing = STAGES * kStage;
  static_assert(kRing >= kSlot * 4, "a warp's ring holds its last partial");
  extern __shared__ uint8_t d8_raw[];
  uint8_t* d8_smem = d8_raw + ((1024u - (smem_u32(d8_raw) & 1023u)) & 1023u);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int B = p.n_seqs;
  uint8_t* ring = d8_smem + warp * kRing;
  float* heads_part = reinterpret_cast<float*>(d8_smem + WARPS * kRing);  // [WARPS][kSlot]
  int* prefix = reinterpret_cast<int*>(heads_part + WARPS * kSlot);       // [B + 1] tiles before each sequence
  int* ctxs = prefix + B + 1;                                             // [B]
  __shared__ __align__(8) uint64_t full[WARPS][STAGES];  // a stage's copies are in
  __shared__ int wsum[WARPS];
  __shared__ int slot_seq[2 * WARPS];  // sequence of each team's partials (-1: none)

  if (lane == 0) {  // the warp's own barriers
    for (int i = 0; i < STAGES; ++i) mbar_init(&full[warp][i], 1);
    fence_barrier_init();
    if (warp == 0) {
      prefetch_tensormap(&kmap);
      prefetch_tensormap(&vmap);
    }
  }
  pdl_wait();  // the metadata, q and the pools may come from the kernel before this one
  pdl_trigger();  // (after the wait: the merge reads the lengths before its own)

  // ---- tiles of each sequence, and their prefix
  {
    const int64_t room = static_cast<int64_t>(p.max_blocks) * p.tiles_per_block * 16;
    const int per = (B + WARPS * 32 - 1) / (WARPS * 32);
    const int lo = min(B, tid * per), hi = min(B, lo + per);
    int sum = 0;
    for (int i = lo; i < hi; ++i) {
      int c = max(p.context_lens[i], 0);
      if (c > room) {
        if (blockIdx.x == 0 && blockIdx.y == 0) raise_flag(p.err, PKV_FLAG_CONTEXT_EXCEEDS_TABLE);
        c = static_cast<int>(room);
      }
      ctxs[i] = c;
      sum += (c + 15) >> 4;
    }
    int x = sum;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    if (lane == 31) wsum[warp] = x;
    __syncthreads();
    int run = x - sum;
    for (int w = 0; w < warp; ++w) run += wsum[w];
    for (int i = lo; i < hi; ++i) {
      prefix[i] = run;
      run += (ctxs[i] + 15) >> 4;
    }
    if (hi == B && lo < B) prefix[B] = run;
    if (tid < 2 * WARPS) slot_seq[tid] = -1;
    __syncthreads();
  }
  const int total = prefix[B];
  const int per = max((total + static_cast<int>(gridDim.x) - 1) / static_cast<int>(gridDim.x), p.min_tiles);
  const int c0 = min(total, static_cast<int>(blockIdx.x) * per), c1 = min(total, c0 + per);
  const int team = warp / p.per_cta;
  const int hg = blockIdx.y * p.per_cta + (warp - team * p.per_cta);
  const int sub = (c1 - c0 + p.teams - 1) / p.teams;
  const bool works = team < p.teams && hg < p.n_groups;
  const int r0 = works ? min(c1, c0 + team * sub) : c1, r1 = works ? min(c1, r0 + sub) : c1;
  const int kvh = hg / p.chunks, head0 = kvh * p.group + (hg - kvh * p.chunks) * kHeads;
  const int nh = works ? min(kHeads, (kvh + 1) * p.group - head0) : 0;  // this warp's query heads

  if (r0 < r1) {
    // ---- the ring: tiles of the range in order, STAGES - 1 ahead
    const int n_tiles = r1 - r0;
    int fill = 0;  // the stage the next copies go to
    // lane l: pool row / 16 and scales of tile 32 b + l of the range
    int ids = 0, ids_next = 0;
    float ks_ids = 0.f, vs_ids = 0.f, ks_next = 0.f, vs_next = 0.f;
    int batch = 0;                                 // of ids
    const uint64_t policy = l2_evict_first_policy();  // every byte is read once
    auto load_ids = [&](int b, int& row16, float& ks, float& vs) {
      const int i = b * 32 + lane;
      if (i < n_tiles) {
        const int s = d8_find(prefix, B, r0 + i);
        const int tile = r0 + i - prefix[s];
        const int jb = p.tiles_per_block == 1 ? tile : tile / p.tiles_per_block;
        int id = p.block_tables[static_cast<int64_t>(s) * p.bt_stride + jb];
        if (id < 0 || id >= p.num_blocks) {
          raise_flag(p.err, PKV_FLAG_BLOCK_OUT_OF_RANGE);
          id = 0;
        }
        row16 = id * p.tiles_per_block + (tile - jb * p.tiles_per_block);
        ks = p.k_scale[static_cast<int64_t>(id) * p.n_kv_heads + kvh];
        vs = p.v_scale[static_cast<int64_t>(id) * p.n_kv_heads + kvh];
      }
    };
    load_ids(0, ids, ks_ids, vs_ids);
    if (n_tiles > 32) load_ids(1, ids_next, ks_next, vs_next);
    auto issue = [&](int i) {
      if (i < n_tiles) {
        // the copies run at most 31 tiles ahead, so i is in this batch or the next
        const int row16 = __shfl_sync(0xffffffffu, (i >> 5) == batch ? ids : ids_next, i & 31);
        if (elect_one()) {
          uint8_t* st = ring + fill * kStage;
          mbar_arrive_expect_tx(&full[warp][fill], kStage);
          tma_load_3d_hint(st, &kmap, &full[warp][fill], 0, kvh, row16 * 16, policy);
          tma_load_3d_hint(st + 16 * D, &vmap, &full[warp][fill], 0, kvh, row16 * 16, policy);
        }
        __syncwarp();
        fill = fill + 1 == STAGES ? 0 : fill + 1;
      }
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) issue(i);

    int s = d8_find(prefix, B, r0), pos = r0;
    int use = 0, i = 0;  // the stage of the tile at pos, its number in the range
    uint32_t use_ph = 0;
    bool dead = false;
    while (pos < r1) {
      const int seg_end = min(prefix[s + 1], r1);
      const int ctx = ctxs[s];
      const bool first = pos == r0;  // the range's first segment
      // ---- Q^T fragments: column n = g is head head0 + 8 nt + g; this lane's
      // dims are those of its K chunks: 16 from 16t (D = 128: 32 from 32t), in
      // words of four, of which k-step kk takes words 2 kk and 2 kk + 1
      uint32_t qb[NT][3][D / 32][2];
      float c_head[NT][2];  // score factor of heads 2t, 2t + 1
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const bool on = 8 * nt + g < nh;
        const T* row = static_cast<const T*>(p.q) + static_cast<int64_t>(s) * p.q_stride +
                       static_cast<int64_t>(head0 + 8 * nt + g) * D + t * (D / 4);
        float f[D / 16][4];
        float amax = 0.f;
#pragma unroll
        for (int w = 0; w < D / 16; ++w) {
          if (on && p.q_vec) {
            load4_f<T>(row + 4 * w, f[w]);
          } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) f[w][e] = on ? Elem<T>::to_f(row[4 * w + e]) : 0.f;
          }
#pragma unroll
          for (int e = 0; e < 4; ++e) amax = fmaxf(amax, fabsf(f[w][e]));
        }
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
        amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
        // the power of two that brings amax to [2^21, 2^22): sums of the top bytes
        // then stay below 2^22 at any head_dim here.  Rows of zeros and tiny rows
        // go by 2^-100; a row that is not finite gives NaN
        const uint32_t ex = max(__float_as_uint(amax) >> 23, 27u);
        const float inv = __uint_as_float((275u - min(ex, 254u)) << 23);
        float back = __uint_as_float((min(ex, 254u) - 21u) << 23);
        bool fine = amax < INFINITY;
#pragma unroll
        for (int w = 0; w < D / 16; ++w) {
          int A[4], Bv[4], C[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            fine = fine && f[w][e] == f[w][e];
            const int q = __float2int_rn(f[w][e] * inv);
            A[e] = (q + 32768 + 128) >> 16;
            const int rest = q - (A[e] << 16);
            Bv[e] = (rest + 128) >> 8;
            C[e] = rest - (Bv[e] << 8);
          }
          qb[nt][0][w / 2][w & 1] = pack_s8(A[0], A[1], A[2], A[3]);
          qb[nt][1][w / 2][w & 1] = pack_s8(Bv[0], Bv[1], Bv[2], Bv[3]);
          qb[nt][2][w / 2][w & 1] = pack_s8(C[0], C[1], C[2], C[3]);
        }
        const unsigned bad = __ballot_sync(0xffffffffu, !fine);
        if ((bad >> (4 * g)) & 15u) back = NAN;
        // lanes 4n .. hold head n's factor
        c_head[nt][0] = p.scale_log2 * __shfl_sync(0xffffffffu, back, 8 * t);
        c_head[nt][1] = p.scale_log2 * __shfl_sync(0xffffffffu, back, 8 * t + 4);
      }
      // mu: the reference of the exponentials, at most kD8Slack (log2) below the
      // running maximum; it moves when some score passes that, which a vote of the
      // lanes' own scores tells, so most tiles need no maximum across lanes
      float mu[NT][2], l[NT][2], o[NT][KS][4];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mu[nt][0] = mu[nt][1] = l[nt][0] = l[nt][1] = 0.f;
#pragma unroll
        for (int j = 0; j < KS; ++j) o[nt][j][0] = o[nt][j][1] = o[nt][j][2] = o[nt][j][3] = 0.f;
      }
      // gain: P' = p vs 2^gain goes into the products (vs: V's scale of the tile)
      float gain[NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) gain[nt][0] = gain[nt][1] = 0.f;
      bool fresh = true;  // no tile of the segment yet

      int left = ctx - (pos - prefix[s]) * 16;  // tokens from this tile on
      for (; pos < seg_end; ++pos, ++i, left -= 16) {
        if (!dead && !mbar_wait(&full[warp][use], use_ph)) dead = true;
        __syncwarp();  // every lane is done with the tile before, whose stage is filled again
        issue(i + STAGES - 1);
        if ((i >> 5) != batch) {  // (uniform) the next 32 tiles
          batch = i >> 5;
          ids = ids_next;
          ks_ids = ks_next;
          vs_ids = vs_next;
          if ((batch + 1) * 32 < n_tiles) load_ids(batch + 1, ids_next, ks_next, vs_next);
        }
        const float ks = __shfl_sync(0xffffffffu, ks_ids, i & 31), vs = __shfl_sync(0xffffffffu, vs_ids, i & 31);
        const uint8_t* st = ring + use * kStage;
        // ---- S^T = K Q^T, one product for each byte of q
        int si[NT][3][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int lb = 0; lb < 3; ++lb) si[nt][lb][0] = si[nt][lb][1] = si[nt][lb][2] = si[nt][lb][3] = kIntBase;
#pragma unroll
        for (int half = 0; half < D / 64; ++half) {
          const int c = D == 64 ? t : 2 * t + half;
          const uint4 k0 = *reinterpret_cast<const uint4*>(st + d8_chunk<D>(g, c));
          const uint4 k1 = *reinterpret_cast<const uint4*>(st + d8_chunk<D>(g + 8, c));
#pragma unroll
          for (int k2 = 0; k2 < 2; ++k2) {
            const uint32_t a[4] = {k2 ? k0.z : k0.x, k2 ? k1.z : k1.x, k2 ? k0.w : k0.y, k2 ? k1.w : k1.y};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int lb = 0; lb < 3; ++lb)
                mma16832_s8(si[nt][lb], a, qb[nt][lb][half * 2 + k2][0], qb[nt][lb][half * 2 + k2][1]);
          }
        }
        float2 sc[NT][2];  // tokens g, g + 8
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float2 v[3];
#pragma unroll
            for (int lb = 0; lb < 3; ++lb)
              v[lb] = __fadd2_rn(make_float2(__int_as_float(si[nt][lb][2 * r]), __int_as_float(si[nt][lb][2 * r + 1])),
                                 make_float2(-kFloatBase, -kFloatBase));
            sc[nt][r] = __ffma2_rn(v[0], make_float2(65536.f, 65536.f), __ffma2_rn(v[1], make_float2(256.f, 256.f), v[2]));
          }
        // ---- x - mu of the lane's scores (tokens g, g + 8; heads 2t, 2t + 1)
        float2 x0[NT], x1[NT];
        float top = -INFINITY, top_w = -INFINITY;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 f = __fmul2_rn(make_float2(c_head[nt][0], c_head[nt][1]), make_float2(ks, ks));
          const float2 nm = make_float2(-mu[nt][0], -mu[nt][1]);
          x0[nt] = __ffma2_rn(sc[nt][0], f, nm);
          x1[nt] = __ffma2_rn(sc[nt][1], f, nm);
        }
        if (left < 16) {  // a sequence's last tile
          const float2 none = make_float2(-INFINITY, -INFINITY);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (g >= left) x0[nt] = none;
            if (g + 8 >= left) x1[nt] = none;
          }
        }
        // the largest x - mu, and the largest of P' without vs
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 m = make_float2(fmaxf(x0[nt].x, x1[nt].x), fmaxf(x0[nt].y, x1[nt].y));
          const float2 w = __fadd2_rn(m, make_float2(gain[nt][0], gain[nt][1]));
          top = fmax3(top, m.x, m.y);
          top_w = fmax3(top_w, w.x, w.y);
        }
        const float v_exp = __uint_as_float(0x4b000000u | (__float_as_uint(vs) >> 23)) - (8388608.f + 127.f);  // vs < 2^(v_exp + 1)
        if (__any_sync(0xffffffffu, top > kD8Slack || top_w + v_exp > kD8MostP - 1.f) || fresh) {
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float mx[2] = {fmaxf(x0[nt].x, x1[nt].x), fmaxf(x0[nt].y, x1[nt].y)}, cf[2];
#pragma unroll
            for (int c = 0; c < 2; ++c) {
#pragma unroll
              for (int off = 4; off < 32; off <<= 1) mx[c] = fmaxf(mx[c], __shfl_xor_sync(0xffffffffu, mx[c], off));
              // the reference moves up to mx, in whole steps (the segment's first tile: to its
              // maximum, unless that is not finite)
              float up = ceilf(fresh ? mx[c] : fmaxf(mx[c], 0.f));
              if (!(fabsf(up) < INFINITY)) up = 0.f;
              mu[nt][c] += up;
              // gain: what it was, raised by what the older p fall by, or as low as this tile's largest P' asks for
              const float want = kD8LeadP - ceilf(mx[c] - up) - v_exp;
              const float to = fmaxf(fminf(fresh ? want : fminf(gain[nt][c] + up, want), kD8MostGain), -126.f);
              cf[c] = exp2_whole(to - gain[nt][c] - up);
              gain[nt][c] = to;
              if (!fresh) l[nt][c] *= exp2_whole(-up);
              mx[c] = up;
            }
            const float2 nu = make_float2(-mx[0], -mx[1]);
            x0[nt] = __fadd2_rn(x0[nt], nu);
            x1[nt] = __fadd2_rn(x1[nt], nu);
            if (!fresh) {
#pragma unroll
              for (int j = 0; j < KS; ++j) {
                o[nt][j][0] *= cf[0];
                o[nt][j][1] *= cf[1];
                o[nt][j][2] *= cf[0];
                o[nt][j][3] *= cf[1];
              }
            }
          }
          fresh = false;
        }
        const float2 vs2 = make_float2(vs, vs);
        uint32_t pb[NT][LIMBS][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
          const float2 p0 = make_float2(ex2_approx(x0[nt].x), ex2_approx(x0[nt].y));
          const float2 p1 = make_float2(ex2_approx(x1[nt].x), ex2_approx(x1[nt].y));
          l[nt][0] += p0.x + p1.x;
          l[nt][1] += p0.y + p1.y;
          // (the gain first: its product with vs alone may pass fp32's range)
          const float2 n = __fadd2_rn(make_float2(gain[nt][0], gain[nt][1]), make_float2(kFloatBase + 127.f, kFloatBase + 127.f));
          const float2 g2 = make_float2(__int_as_float(__float_as_int(n.x) << 23), __int_as_float(__float_as_int(n.y) << 23));
          const float2 e0 = __fmul2_rn(__fmul2_rn(p0, g2), vs2), e1 = __fmul2_rn(__fmul2_rn(p1, g2), vs2);
          float e[4] = {e0.x, e0.y, e1.x, e1.y};
          pb[nt][0][0] = movmatrix_t(pack2<__half>(e[0], e[1]));
          pb[nt][0][1] = movmatrix_t(pack2<__half>(e[2], e[3]));
          if constexpr (LIMBS == 2) {
#pragma unroll
            for (int c = 0; c < 4; ++c) e[c] -= __half2float(__float2half_rn(e[c]));
            pb[nt][LIMBS - 1][0] = movmatrix_t(pack2<__half>(e[0], e[1]));
            pb[nt][LIMBS - 1][1] = movmatrix_t(pack2<__half>(e[2], e[3]));
          }
        }
        // ---- O^T += V^T P^T: row g of m-tile mt is dim 8g + 2mt (of a half of 64), row g + 8 the next
        const int sw = t & 1;
        const uint32_t flip_sel = sw ? 0x4444u : 0u;
#pragma unroll
        for (int half = 0; half < D / 64; ++half) {
          uint2 r[4];
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const int row = 2 * t + (k >> 1) * 8 + ((k & 1) ^ sw);
            r[k] = *reinterpret_cast<const uint2*>(st + 16 * D + d8_chunk<D>(row, half * 4 + (g >> 1)) + (g & 1) * 8);
            r[k].x ^= 0x80808080u;
            r[k].y ^= 0x80808080u;
          }
#pragma unroll
          for (int mt = 0; mt < 4; ++mt) {
            const uint32_t sel = ((mt & 1) ? 0x7362u : 0x5140u) ^ flip_sel;
            const uint32_t x01 = __byte_perm(mt < 2 ? r[0].x : r[0].y, mt < 2 ? r[1].x : r[1].y, sel);
            const uint32_t x23 = __byte_perm(mt < 2 ? r[2].x : r[2].y, mt < 2 ? r[3].x : r[3].y, sel);
            const uint32_t a[4] = {i8_lo(x01), i8_hi(x01), i8_lo(x23), i8_hi(x23)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int lb = 0; lb < LIMBS; ++lb)
                mma16816<__half>(o[nt][half * 4 + mt], a, pb[nt][lb][0], pb[nt][lb][1]);
          }
        }
        if (++use == STAGES) {
          use = 0;
          use_ph ^= 1;
        }
      }

      // ---- segment end
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int c = 0; c < 2; ++c)
#pragma unroll
          for (int off = 4; off < 32; off <<= 1) l[nt][c] += __shfl_xor_sync(0xffffffffu, l[nt][c], off);
      const bool complete = prefix[s] >= r0 && prefix[s + 1] <= r1;
      if (complete) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int hh = 8 * nt + 2 * t + c;
            if (hh >= nh) continue;
            const float f = 1.f / l[nt][c], back = exp2_whole(-gain[nt][c]);
            T* orow = static_cast<T*>(p.out) + static_cast<int64_t>(s) * p.out_stride +
                      static_cast<int64_t>(head0 + hh) * D;
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              const int d = (j >> 2) * 64 + 8 * g + 2 * (j & 3);
              orow[d] = Elem<T>::from_f(o[nt][j][c] * f * back);
              orow[d + 1] = Elem<T>::from_f(o[nt][j][c + 2] * f * back);
            }
          }
      } else {
        // the range's first partial goes to its own slot, a later (last) one
        // into the ring, which no copy in flight uses any more
        float* slot = first ? heads_part + warp * kSlot : reinterpret_cast<float*>(ring);
        if (!first) __syncwarp();  // every lane is done with the last tile
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const int hh = 8 * nt + 2 * t + c;
            const float f = 1.f / l[nt][c], back = exp2_whole(-gain[nt][c]);  // a partial holds its own softmax's O
#pragma unroll
            for (int j = 0; j < KS; ++j) {
              const int d = (j >> 2) * 64 + 8 * g + 2 * (j & 3);
              slot[hh * D + d] = o[nt][j][c] * f * back;
              slot[hh * D + d + 1] = o[nt][j][c + 2] * f * back;
            }
            if (g == 0) {
              slot[kHeads * D + 2 * hh] = mu[nt][c];
              slot[kHeads * D + 2 * hh + 1] = l[nt][c];
            }
          }
        if (lane == 0 && warp == team * p.per_cta) slot_seq[2 * team + (first ? 0 : 1)] = s;
      }
      ++s;
      while (s < B && prefix[s + 1] == prefix[s]) ++s;  // empty sequences
    }
    if (dead && lane == 0) raise_flag(p.err, PKV_FLAG_PIPELINE_TIMEOUT);
  }
  __syncthreads();

  // ---- join the teams' partials: runs of slots of one sequence, in order
  static_assert(2 * WARPS <= 32, "a lane for each slot");
  __shared__ int n_runs;
  __shared__ unsigned run_mask[2 * WARPS];  // the slots of each run
  if (warp == 0) {
    const int v = lane < 2 * p.teams ? slot_seq[lane] : -1;
    const unsigned used = __ballot_sync(0xffffffffu, v >= 0);
    const unsigned below = used & ((1u << lane) - 1u);
    const int before = __shfl_sync(0xffffffffu, v, below ? 31 - __clz(below) : 0);
    const unsigned starts = __ballot_sync(0xffffffffu, v >= 0 && (below == 0 || before != v));
    if ((starts >> lane) & 1) {
      const unsigned later = starts & ~((2u << lane) - 1u);  // starts of later runs (lane 31: 2 << 31 is 0)
      const unsigned upto = later ? (1u << (__ffs(later) - 1)) - 1u : 0xffffffffu;
      run_mask[__popc(starts & ((1u << lane) - 1u))] = used & upto & ~((1u << lane) - 1u);
    }
    if (lane == 0) n_runs = __popc(starts);
  }
  __syncthreads();
  constexpr int kVec = D / 4;
  const int per_run = p.per_cta * kHeads * kVec;  // four dims at a time
  for (int e = tid; e < n_runs * per_run; e += WARPS * 32) {
    const int r = e / per_run, w = (e - r * per_run) / (kHeads * kVec), hh = (e / kVec) % kHeads, v = e % kVec;
    const int hgw = blockIdx.y * p.per_cta + w;
    if (hgw >= p.n_groups) continue;
    const int kv = p.chunks == 1 ? hgw : hgw / p.chunks, head = kv * p.group + (hgw - kv * p.chunks) * kHeads + hh;
    if (head >= (kv + 1) * p.group) continue;
    float mm = 0.f, ll = 0.f;
    float4 oo = make_float4(0.f, 0.f, 0.f, 0.f);
    unsigned todo = run_mask[r];
    const int s = slot_seq[__ffs(todo) - 1];
    for (bool one = true; todo; todo &= todo - 1, one = false) {
      const int a = __ffs(todo) - 1, wp = (a >> 1) * p.per_cta + w;
      const float* sl = (a & 1) ? reinterpret_cast<const float*>(d8_smem + wp * kRing) : heads_part + wp * kSlot;
      const float2 ml = *reinterpret_cast<const float2*>(sl + kHeads * D + 2 * hh);
      const float4 x = *reinterpret_cast<const float4*>(sl + hh * D + 4 * v);
      const float mn = one ? ml.x : fmaxf(mm, ml.x);
      // (nothing is held before the first, whose mn may be far below zero: 0 * inf would be NaN)
      const float fa = one ? 0.f : ex2_approx(mm - mn), fb = ex2_approx(ml.x - mn) * ml.y;
      mm = mn;
      ll = ll * fa + fb;
      oo = make_float4(oo.x * fa + x.x * fb, oo.y * fa + x.y * fb, oo.z * fa + x.z * fb, oo.w * fa + x.w * fb);
    }
    const float inv = 1.f / ll;
    oo = make_float4(oo.x * inv, oo.y * inv, oo.z * inv, oo.w * inv);
    if (prefix[s] >= c0 && prefix[s + 1] <= c1) {  // all of it in this CTA
      T* op = static_cast<T*>(p.out) + static_cast<int64_t>(s) * p.out_stride + static_cast<int64_t>(head) * D + 4 * v;
      op[0] = Elem<T>::from_f(oo.x);
      op[1] = Elem<T>::from_f(oo.y);
      op[2] = Elem<T>::from_f(oo.z);
      op[3] = Elem<T>::from_f(oo.w);
    } else {
      const int64_t part = prefix[s] > c0 ? 2 * blockIdx.x + 1 : 2 * blockIdx.x;
      reinterpret_cast<float4*>(p.part_o + (part * p.n_q_heads + head) * D)[v] = oo;
      if (v == 0) *reinterpret_cast<float2*>(p.part_ml + (part * p.n_q_heads + head) * 2) = make_float2(mm, ll);
    }
  }
}

// Joins the CTAs' partials of sequence blockIdx.x (heads blockIdx.y * heads_per ..):
// O = sum_c w_c O_c / sum_c w_c, w_c = 2^(m_c - M) l_c, over the CTAs that share
// it, in order.  Four dims of one head to a thread; a sequence that many CTAs
// share (a long one) is read by all the CTA's threads, kLanes partials of a head
// side by side: its weights are made while up to kM8Ahead of a thread's partials
// are on their way (running sums, four at a time: 18.2 us instead of 15.7 for
// 131,072 tokens).  Empty sequences get zeros.  The lengths are read while the
// decode kernel runs (it starts this one after its own wait for them).
//
// Up to kM8Few partials a thread takes all of them for its dims (256 x 1,024 tokens
// when this was chosen: 22.3 us; 37.9 with the other way for all, 24.9 with this way
// for up to 16).
constexpr int kM8Threads = 256, kM8Few = 6, kM8Ahead = 10;
template <typename T, int D>
__global__ void __launch_bounds__(kM8Threads) merge_int8_kernel(const D8Params p, int grid, int heads_per) {
  constexpr int kVec = D / 4, kLanes = kM8Threads / kVec;
  __shared__ float4 s_o[kLanes][kVec];
  __shared__ float s_m[kM8Threads / 32], s_l[kM8Threads / 32], s_w[kD8MaxCtas];
  __shared__ int red[2][kM8Threads / 32];
  const int s = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int64_t room = static_cast<int64_t>(p.max_blocks) * p.tiles_per_block * 16;
  auto tiles_of = [&](int i) {
    return static_cast<int>((min(static_cast<int64_t>(max(p.context_lens[i], 0)), room) + 15) >> 4);
  };
  int before = 0, total = 0;
  for (int i = tid; i < p.n_seqs; i += kM8Threads) {
    const int n = tiles_of(i);
    total += n;
    if (i < s) before += n;
  }
  before = __reduce_add_sync(0xffffffffu, before);
  total = __reduce_add_sync(0xffffffffu, total);
  if (lane == 0) { red[0][warp] = before; red[1][warp] = total; }
  __syncthreads();
  before = total = 0;
#pragma unroll
  for (int w = 0; w < kM8Threads / 32; ++w) { before += red[0][w]; total += red[1][w]; }
  const int mine = tiles_of(s);
  const int per = max((total + grid - 1) / grid, p.min_tiles);
  const int h0 = blockIdx.y * heads_per, h1 = min(p.n_q_heads, h0 + heads_per);
  T* orow = static_cast<T*>(p.out) + static_cast<int64_t>(s) * p.out_stride;
  const int first = mine ? before / per : 0, last = mine ? (before + mine - 1) / per : 0;
  pdl_wait();  // the decode grid's partials are in memory
  if (mine == 0) {
    for (int e = h0 * D + tid; e < h1 * D; e += kM8Threads) orow[e] = Elem<T>::from_f(0.f);
    return;
  }
  if (first == last) return;  // one CTA had it all and wrote it
  struct Acc {
    float m = 0.f, l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    bool any = false;
    __device__ void add(float2 ml, float4 x) {
      const float mn = any ? fmaxf(m, ml.x) : ml.x;
      const float fa = any ? ex2_approx(m - mn) : 0.f, fb = ex2_approx(ml.x - mn) * ml.y;
      m = mn;
      any = true;
      l = l * fa + fb;
      o = make_float4(o.x * fa + x.x * fb, o.y * fa + x.y * fb, o.z * fa + x.z * fb, o.w * fa + x.w * fb);
    }
  };
  auto part_of = [&](int c) { return 2 * static_cast<int64_t>(c) + (before > static_cast<int64_t>(c) * per ? 1 : 0); };
  auto load_o = [&](int64_t part, int h, int v) {
    return reinterpret_cast<const float4*>(p.part_o + (part * p.n_q_heads + h) * D)[v];
  };
  auto load_ml = [&](int64_t part, int h) {
    return *reinterpret_cast<const float2*>(p.part_ml + (part * p.n_q_heads + h) * 2);
  };
  auto store = [&](int h, int v, const Acc& a) {
    T* op = orow + static_cast<int64_t>(h) * D + 4 * v;
    const float inv = 1.f / a.l;
    op[0] = Elem<T>::from_f(a.o.x * inv);
    op[1] = Elem<T>::from_f(a.o.y * inv);
    op[2] = Elem<T>::from_f(a.o.z * inv);
    op[3] = Elem<T>::from_f(a.o.w * inv);
  };
  if (last - first < kM8Few) {
    for (int e = tid; e < (h1 - h0) * kVec; e += kM8Threads) {
      const int h = h0 + e / kVec, v = e % kVec;
      float2 ml[kM8Few];
      float4 x[kM8Few];
#pragma unroll
      for (int k = 0; k < kM8Few; ++k)
        if (first + k <= last) {
          ml[k] = load_ml(part_of(first + k), h);
          x[k] = load_o(part_of(first + k), h, v);
        }
      Acc a;
#pragma unroll
      for (int k = 0; k < kM8Few; ++k)
        if (first + k <= last) a.add(ml[k], x[k]);
      store(h, v, a);
    }
    return;
  }
  const int v = tid % kVec, k0 = tid / kVec, n = last - first + 1;
  for (int h = h0; h < h1; ++h) {
    // the O loads are on their way while the weights are made
    float4 x[kM8Ahead];
#pragma unroll
    for (int i = 0; i < kM8Ahead; ++i)
      if (k0 + i * kLanes < n) x[i] = load_o(part_of(first + k0 + i * kLanes), h, v);
    float top = -INFINITY;
    for (int c = tid; c < n; c += kM8Threads) top = fmaxf(top, load_ml(part_of(first + c), h).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    if (lane == 0) s_m[warp] = top;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kM8Threads / 32; ++w) top = fmaxf(top, s_m[w]);
    float sum = 0.f;
    for (int c = tid; c < n; c += kM8Threads) {
      const float2 ml = load_ml(part_of(first + c), h);
      s_w[c] = ex2_approx(ml.x - top) * ml.y;
      sum += s_w[c];
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_l[warp] = sum;
    __syncthreads();
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](float w, float4 y) {
      o = make_float4(fmaf(w, y.x, o.x), fmaf(w, y.y, o.y), fmaf(w, y.z, o.z), fmaf(w, y.w, o.w));
    };
#pragma unroll
    for (int i = 0; i < kM8Ahead; ++i)
      if (k0 + i * kLanes < n) add(s_w[k0 + i * kLanes], x[i]);
    for (int c = k0 + kM8Ahead * kLanes; c < n; c += kLanes) add(s_w[c], load_o(part_of(first + c), h, v));
    s_o[k0][v] = o;
    __syncthreads();
    if (k0 == 0) {
      Acc all;
      for (int k = 1; k < kLanes; ++k) {
        const float4 y = s_o[k][v];
        o = make_float4(o.x + y.x, o.y + y.y, o.z + y.z, o.w + y.w);
      }
      all.o = o;
#pragma unroll
      for (int w = 0; w < kM8Threads / 32; ++w) all.l += s_l[w];
      store(h, v, all);
    }
    __syncthreads();
  }
}

template <typename T, int D, int NT, int WARPS, int STAGES>
cudaError_t launch_d8(const AttnArgs& a, const CUtensorMap* kmap, const CUtensorMap* vmap, void* workspace, cudaStream_t stream) {
  constexpr int LIMBS = std::is_same<T, float>::value ? 2 : 1;
  auto kern = decode_int8_kernel<T, D, NT, LIMBS, WARPS, STAGES>;
  constexpr int kFixed = 1024 + WARPS * (STAGES * d8_stage<D>() + 8 * NT * (D + 2) * 4);
  constexpr int kMost = kFixed + (2 * kD8MaxSeqs + 1) * 4;
  static_assert(kMost + 1024 <= 232448, "the rings and partials fit the 227 KB of shared memory");
  static std::atomic<int> sm_count[64];  // per device, 0: not asked
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int sms = dev < 64 ? sm_count[dev].load() : 0;
  if (sms == 0) {
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
    if (e != cudaSuccess) return e;
    if (dev < 64) sm_count[dev].store(sms);
  }
  D8Params p{};
  p.k_pool = static_cast<const int8_t*>(a.k_pool);
  p.v_pool = static_cast<const int8_t*>(a.v_pool);
  p.k_scale = a.k_scale;
  p.v_scale = a.v_scale;
  p.bt_stride = a.bt_stride;
  p.max_blocks = a.max_blocks;
  p.num_blocks = a.num_blocks;
  p.tiles_per_block = a.block_size / 16;
  p.n_q_heads = a.n_q_heads;
  p.n_kv_heads = a.n_kv_heads;
  p.group = a.n_q_heads / a.n_kv_heads;
  p.chunks = (p.group + 8 * NT - 1) / (8 * NT);
  p.n_groups = p.n_kv_heads * p.chunks;
  p.per_cta = std::min(p.n_groups, 8);
  p.teams = WARPS / p.per_cta;
  p.min_tiles = 2 * p.teams;
  p.scale_log2 = a.scale * kD8Log2e;
  p.out_stride = a.out_stride;
  p.q_stride = a.q_stride;
  p.err = a.err;
  p.part_ml = static_cast<float*>(workspace);
  p.part_o = p.part_ml + static_cast<size_t>(2) * kD8MaxCtas * p.n_q_heads * 2;
  const int gy = (p.n_groups + p.per_cta - 1) / p.per_cta;
  const int gx = std::max(1, std::min(sms, kD8MaxCtas) / gy);
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = stream;
  const int es = sizeof(T);
  p.q_vec = ((reinterpret_cast<uintptr_t>(a.q) | static_cast<uintptr_t>(a.q_stride * es)) & (4 * es - 1)) == 0;
  for (int s0 = 0; s0 < a.n_seqs; s0 += kD8MaxSeqs) {
    p.n_seqs = std::min(kD8MaxSeqs, a.n_seqs - s0);
    p.out = static_cast<uint8_t*>(a.out) + s0 * a.out_stride * es;
    p.q = static_cast<const uint8_t*>(a.q) + s0 * a.q_stride * es;
    p.block_tables = a.block_tables + s0 * a.bt_stride;
    p.context_lens = a.context_lens + s0;
    cfg.gridDim = dim3(gx, gy);
    cfg.blockDim = dim3(WARPS * 32);
    cfg.dynamicSmemBytes = kFixed + (2 * p.n_seqs + 1) * 4;
    e = cudaLaunchKernelEx(&cfg, kern, *kmap, *vmap, p);
    if (e != cudaSuccess) return e;
    const int splits = std::max(1, std::min(p.n_q_heads, 296 / p.n_seqs));
    const int heads_per = (p.n_q_heads + splits - 1) / splits;
    cfg.gridDim = dim3(p.n_seqs, (p.n_q_heads + heads_per - 1) / heads_per);
    cfg.blockDim = dim3(kM8Threads);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, merge_int8_kernel<T, D>, p, gx, heads_per);
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

template <typename T>
cudaError_t launch_d8_t(const AttnArgs& a, const CUtensorMap* km, const CUtensorMap* vm, void* ws, cudaStream_t stream) {
  // query heads per warp: 8, or 16 where the group has more (V's fragments are
  // then converted once for both halves).  64 sequences of 4,096 tokens with 8 and
  // with 16: 14 / 2 x 64 21.6 and 31.8 us, 32 / 8 x 128 93 and 131; 32 / 2 x 128
  // 46.5 and 44.5, 16 / 1 x 128 in fp32 33.1 and 30.9
  const bool two = a.n_q_heads / a.n_kv_heads > 8;
  constexpr bool f32 = std::is_same<T, float>::value;
  if (a.head_dim == 64)
    return two ? launch_d8<T, 64, 2, 8, 6>(a, km, vm, ws, stream)
               : launch_d8<T, 64, 1, 16, 5>(a, km, vm, ws, stream);
  return two ? launch_d8<T, 128, 2, 8, 4>(a, km, vm, ws, stream)
             : launch_d8<T, 128, 1, f32 ? 8 : 16, f32 ? 4 : 2>(a, km, vm, ws, stream);
}

}  // namespace

size_t decode_int8_workspace_bytes(int n_q_heads, int head_dim) {
  return static_cast<size_t>(2) * kD8MaxCtas * n_q_heads * (head_dim + 2) * 4;
}

cudaError_t launch_decode_int8(const AttnArgs& a, const CUtensorMap* kmap, const CUtensorMap* vmap,
                               void* workspace, cudaStream_t stream) {
  if (a.n_seqs == 0) return cudaSuccess;
  if (a.dtype == PKV_DTYPE_F16) return launch_d8_t<__half>(a, kmap, vmap, workspace, stream);
  if (a.dtype == PKV_DTYPE_BF16) return launch_d8_t<__nv_bfloat16>(a, kmap, vmap, workspace, stream);
  return launch_d8_t<float>(a, kmap, vmap, workspace, stream);
}

}  // namespace pkv
