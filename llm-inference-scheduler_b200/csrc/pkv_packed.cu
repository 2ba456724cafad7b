// pkv_packed.cu -- causal attention with grouped heads over consecutive rows:
// whole prompts packed one behind the other, or chunks behind cached keys that
// were laid out row by row.
//
//   x_ij = scale q_i . k_j,  j <= prior + i,  o_i = sum_j softmax(x_i)_j v_j
//
// in one pass over the keys with a running maximum and sum (fp32).  fp16 and bf16
// rows that TMA can read take the tensor-core tiles (packed_tc_kernel), fp32 rows
// and those at other strides or alignments, or of more than 64 query heads to a
// KV head, the CUDA-core tiles (packed_cores_kernel).
#include <float.h>
#include <limits.h>

#include <atomic>
#include <type_traits>

#include "pkv_common.cuh"
#include "pkv_internal.h"

namespace pkv {

namespace {

// first key row, keys before the first query, and keys of sequence s in all
struct KeySpan {
  int64_t row0;
  int prior, keys;
};
__device__ __forceinline__ KeySpan key_span(const PackedArgs& a, int s, int q_begin, int n_new) {
  KeySpan k;
  if (a.num_prior == nullptr) {
    k.row0 = q_begin;
    k.prior = 0;
    k.keys = n_new;
  } else {
    k.row0 = static_cast<int64_t>(s) * a.key_cap;
    k.prior = max(a.num_prior[s], 0);
    k.keys = static_cast<int>(min(static_cast<int64_t>(k.prior) + n_new, static_cast<int64_t>(a.key_limit)));
  }
  return k;
}

// ---- rows that come out not finite
//
// The tiled kernels multiply a hidden key's V by a probability of zero, which is
// not zero where that V holds an infinity or NaN, and their unnormalised sums pass
// fp32 for values near its end.  A row that comes out not finite is therefore
// computed again by a warp, over its own keys only, unless its own values make it
// so: its sum of probabilities is NaN (hidden scores never enter that), or a V that
// it sees is not finite and none of the hidden ones in its last tiles is (then sums
// that pass fp32 stay infinite in its other columns too).  (Without
// that second rule one NaN in the first V of a prompt of 8,191 tokens had every later
// row computed again: 77 ms.  With it 0.2; and 8.8 where the NaN is hidden from the
// last rows, four at a time, against 45 one by one.)

// four or eight consecutive elements from a 16-byte boundary
template <typename T>
__device__ __forceinline__ void load16_f(const T* p, float* v) {
  const uint4 w = *reinterpret_cast<const uint4*>(p);
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T* e = reinterpret_cast<const T*>(u) + i;
      v[i] = Elem<T>::to_f(*e);
    }
  }
}

// (whole warp) keys from .. to - 1 of one sequence and KV head: the last of them whose
// V is not finite, or the first; `none` if there is none.
template <typename T, int D, bool VEC>
__device__ __forceinline__ int value_not_finite(const PackedArgs& a, int g, int64_t key0, int from, int to, bool last, int none) {
  const int lane = threadIdx.x & 31;
  for (int i = 0; i < to - from; i += 32) {
    const int key = last ? to - 1 - i - lane : from + i + lane;
    bool bad = false;
    if (key >= from && key < to) {
      const T* v = static_cast<const T*>(a.v) + (key0 + key) * a.v_stride + static_cast<int64_t>(g) * D;
      constexpr int kStep = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
#pragma unroll 8
      for (int d = 0; d < D; d += kStep) {
        float f[kStep];
        if constexpr (VEC) load16_f<T>(v + d, f);
        else f[0] = Elem<T>::to_f(v[d]);
#pragma unroll
        for (int e = 0; e < kStep; ++e) bad = bad || !(fabsf(f[e]) < INFINITY);
      }
    }
    const unsigned hit = __ballot_sync(0xffffffffu, bad);
    if (hit) {  // lane 0 has the end that is asked for
      const int l = __ffs(hit) - 1;
      return last ? to - 1 - i - l : from + i + l;
    }
  }
  return none;
}

// Up to kAlone (query row, head) pairs of one KV head by a whole warp, each over its
// own keys 0 .. lim - 1 only: 32 keys at a time, the scores a key to a lane, the
// values D / 32 dims to a lane (VEC: a step's loads ahead of its arithmetic).  Rows with
// lim 0 are not there.  About 64 cycles a row and key (fp16, 64 dims).
constexpr int kAlone = 4;
template <typename T, int D, bool VEC>
__device__ __forceinline__ void packed_rows_alone(const PackedArgs& a, const int64_t (&row)[kAlone], const int (&h)[kAlone],
                                                  const int (&lim)[kAlone], int g, int64_t key0) {
  const int lane = threadIdx.x & 31;
  constexpr int kPer = D / 32, kStep = VEC ? 16 / static_cast<int>(sizeof(T)) : 1;
  constexpr int kAhead = VEC ? 16 : 4;  // values on their way at a time
  const T* kr = static_cast<const T*>(a.k) + key0 * a.k_stride + static_cast<int64_t>(g) * D;
  const T* vr = static_cast<const T*>(a.v) + key0 * a.v_stride + static_cast<int64_t>(g) * D + lane * kPer;
  const T* q[kAlone];
  float acc[kAlone][kPer], m[kAlone], l[kAlone];  // l: this lane's keys
  int most = 0;
#pragma unroll
  for (int r = 0; r < kAlone; ++r) {
    q[r] = static_cast<const T*>(a.q) + row[r] * a.q_stride + static_cast<int64_t>(h[r]) * D;
    m[r] = -FLT_MAX;
    l[r] = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[r][i] = 0.f;
    most = max(most, lim[r]);
  }
  for (int j0 = 0; j0 < most; j0 += 32) {
    const int n = min(32, most - j0);
    struct alignas(VEC ? kPer * sizeof(T) : sizeof(T)) Dims { T e[kPer]; } v[kAhead];
    auto load_v = [&](int at) {
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        // (a key past the last is read as the last, and gets no weight)
        const T* from = vr + static_cast<int64_t>(j0 + min(at + j, n - 1)) * a.v_stride;
        if constexpr (VEC) {
          v[j] = *reinterpret_cast<const Dims*>(from);
        } else {
#pragma unroll
          for (int i = 0; i < kPer; ++i) v[j].e[i] = from[i];
        }
      }
    };
    load_v(0);
    float p[kAlone];
#pragma unroll
    for (int r = 0; r < kAlone; ++r) p[r] = 0.f;
    const T* k = kr + static_cast<int64_t>(j0 + min(lane, n - 1)) * a.k_stride;
#pragma unroll 4
    for (int d = 0; d < D; d += kStep) {
      float kf[kStep], qf[kStep];
      if constexpr (VEC) load16_f<T>(k + d, kf);
      else kf[0] = Elem<T>::to_f(k[d]);
#pragma unroll
      for (int r = 0; r < kAlone; ++r) {
        if constexpr (VEC) load16_f<T>(q[r] + d, qf);
        else qf[0] = Elem<T>::to_f(q[r][d]);
#pragma unroll
        for (int e = 0; e < kStep; ++e) p[r] = fmaf(qf[e], kf[e], p[r]);
      }
    }
#pragma unroll
    for (int r = 0; r < kAlone; ++r) {
      const float s = j0 + lane < lim[r] ? p[r] * a.scale : -INFINITY;
      float mn = fmaxf(m[r], s);
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mn = fmaxf(mn, __shfl_xor_sync(0xffffffffu, mn, o));
      const float c = expf(m[r] - mn);
      p[r] = expf(s - mn);
      m[r] = mn;
      l[r] = l[r] * c + p[r];
#pragma unroll
      for (int i = 0; i < kPer; ++i) acc[r][i] *= c;
    }
#pragma unroll 1
    for (int at = 0; at < n; at += kAhead) {
      if (at > 0) load_v(at);
#pragma unroll
      for (int j = 0; j < kAhead; ++j)
#pragma unroll
        for (int r = 0; r < kAlone; ++r) {
          const float pj = __shfl_sync(0xffffffffu, p[r], (at + j) & 31);
          if (j0 + at + j < lim[r]) {
#pragma unroll
            for (int i = 0; i < kPer; ++i) acc[r][i] = fmaf(pj, Elem<T>::to_f(v[j].e[i]), acc[r][i]);
          }
        }
    }
  }
#pragma unroll
  for (int r = 0; r < kAlone; ++r) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], o);
    if (lim[r] == 0) continue;
    T* out = static_cast<T*>(a.out) + row[r] * a.out_stride + static_cast<int64_t>(h[r]) * D + lane * kPer;
#pragma unroll
    for (int i = 0; i < kPer; ++i) out[i] = Elem<T>::from_f(acc[r][i] / l[r]);
  }
}

// (whole warp) `bad` lanes: a row of head h (all of one KV head) and `lim` keys came
// out not finite with a sum that is.  A row's last key tile ends at most 127 + 127 keys
// behind its last key (the last row of its query tile, the end of a key tile)
template <typename T, int D, bool VEC>
__device__ __noinline__ void redo_rows(const PackedArgs& a, bool bad, int64_t row, int h, int lim, int64_t key0) {
  const int g = __shfl_sync(0xffffffffu, h, 0) / (a.n_q_heads / a.n_kv_heads);
  const int low = __reduce_min_sync(0xffffffffu, bad ? lim : INT_MAX), high = __reduce_max_sync(0xffffffffu, bad ? lim : 0);
  const int end = static_cast<int>(min((static_cast<int64_t>(high) + 254) / 128 * 128, a.n_key_rows - key0));
  const int hidden = value_not_finite<T, D, VEC>(a, g, key0, low, end, true, -1);
  const int seen = value_not_finite<T, D, VEC>(a, g, key0, 0, high, false, INT_MAX);
  unsigned todo = __ballot_sync(0xffffffffu, bad && (lim <= hidden || lim <= seen));
  while (todo) {
    int64_t rows[kAlone];
    int heads[kAlone], lims[kAlone];
#pragma unroll
    for (int r = 0; r < kAlone; ++r) {
      const int b = todo ? __ffs(todo) - 1 : 0;
      rows[r] = __shfl_sync(0xffffffffu, row, b);
      heads[r] = __shfl_sync(0xffffffffu, h, b);
      lims[r] = __shfl_sync(0xffffffffu, lim, b);
      if (todo == 0) lims[r] = 0, rows[r] = rows[0], heads[r] = heads[0];
      todo &= todo - 1;
    }
    packed_rows_alone<T, D, VEC>(a, rows, heads, lims, g, key0);
  }
}

// ---- CUDA-core tiles: 64 queries x 64 keys, fp32 throughout
constexpr int kPkM = 64, kPkN = 64, kPkThreads = 256;

// tile u of the packed rows: sequence i's tiles start at floor(start_i / 64) + i,
// which leaves room for ceil(n_i / 64) of them, so no prefix pass is needed
__device__ __forceinline__ bool find_tile(const PackedArgs& a, int64_t u, int m_rows, int& s, int& tile) {
  int lo = 0, hi = a.n_seqs - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (a.query_start_loc[mid] / m_rows + static_cast<int64_t>(mid) <= u) lo = mid; else hi = mid - 1;
  }
  s = lo;
  const int begin = a.query_start_loc[lo], n = a.query_start_loc[lo + 1] - begin;
  tile = static_cast<int>(u - (begin / m_rows + static_cast<int64_t>(lo)));
  if (begin < 0 || n < 0 || begin + static_cast<int64_t>(n) > a.n_tokens) {
    if (tile == 0 && threadIdx.x == 0) raise_flag(a.err, PKV_FLAG_BAD_QUERY_LAYOUT);
    return false;
  }
  return tile >= 0 && static_cast<int64_t>(tile) * m_rows < n;
}

__device__ __forceinline__ void pk_copy16(void* dst, const void* src, bool on) {  // zeros where not on
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(dst)), "l"(src), "r"(on ? 16 : 0) : "memory");
}

// A thread takes 4 rows x 4 keys of S (keys tx + 16 c) and 4 rows x 4 (or 2 x 4)
// dims of O, two products an instruction (the paired fp32 FMA): 8 16-byte reads
// of shared memory for 32 of them, in both.  fp32 rows on 16-byte boundaries come
// by cp.async, a key tile ahead; other rows element by element.  Bound by those
// reads (55% of the shared-memory pipe's cycles), the FMAs (43%) and, with fewer
// than two CTAs an SM, the latency between them: 37 TFLOP/s for a prompt of 4,096
// tokens (14 / 2 x 64, fp32), 97 us for one of 1,000, 22 for three of 250, 17 and
// 93.  Tiles of 32 or 16 queries were no faster for those (a key tile takes as
// long) and up to 2.2 times slower for long ones.
template <typename T, int D>
__global__ void __launch_bounds__(kPkThreads) packed_cores_kernel(const PackedArgs a, int wide) {
  extern __shared__ __align__(16) float pk_smem[];
  constexpr int kLd = D + 4;                // row pitch of the Q, K and V tiles (16-byte rows, spread banks)
  constexpr int kTile = 64 * kLd;
  float* qs = pk_smem;                      // [64][kLd]
  float* kvs = qs + kTile;                  // [2 buffers][K, V][64][kLd]
  float* ps = kvs + 4 * kTile;              // [64][68] probabilities
  constexpr int kLp = kPkN + 4;
  pdl_wait();
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const unsigned back = gridDim.x - 1 - blockIdx.x, u = back / static_cast<unsigned>(a.n_q_heads);
  const int h = static_cast<int>(back - u * a.n_q_heads), g = h / (a.n_q_heads / a.n_kv_heads);
  int s, tile;
  // the last tiles (the longest of a sequence) first, all heads of one together
  if (!find_tile(a, u, kPkM, s, tile)) return;
  const int q_begin = a.query_start_loc[s], n_new = a.query_start_loc[s + 1] - q_begin;
  const KeySpan span = key_span(a, s, q_begin, n_new);
  const int q0 = tile * kPkM, rows = min(kPkM, n_new - q0);
  const int last = min(span.prior + q0 + rows, span.keys);  // keys any row of the tile sees

  auto load_tile = [&](float* dst, const T* src, int64_t stride, int n) {
    for (int c = tid; c < 64 * (D / 4); c += kPkThreads) {
      const int r = c / (D / 4), d = (c - r * (D / 4)) * 4;
      if constexpr (sizeof(T) == 4) {
        if (wide) {
          pk_copy16(dst + r * kLd + d, src + (r < n ? r * stride + d : 0), r < n);
          continue;
        }
      }
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < n) {
        const T* p = src + r * stride + d;
        f = make_float4(Elem<T>::to_f(p[0]), Elem<T>::to_f(p[1]), Elem<T>::to_f(p[2]), Elem<T>::to_f(p[3]));
      }
      *reinterpret_cast<float4*>(dst + r * kLd + d) = f;
    }
  };
  auto load_kv = [&](int k0) {
    float* buf = kvs + ((k0 / kPkN) & 1) * 2 * kTile;
    const int n = min(kPkN, last - k0);
    if (n > 0) {
      load_tile(buf, static_cast<const T*>(a.k) + (span.row0 + k0) * a.k_stride + static_cast<int64_t>(g) * D, a.k_stride, n);
      load_tile(buf + kTile, static_cast<const T*>(a.v) + (span.row0 + k0) * a.v_stride + static_cast<int64_t>(g) * D, a.v_stride, n);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
  load_tile(qs, static_cast<const T*>(a.q) + static_cast<int64_t>(q_begin + q0) * a.q_stride +
                    static_cast<int64_t>(h) * D, a.q_stride, rows);
  load_kv(0);
  constexpr int kDim = D / 16;  // dims of O per thread and row: 4 tx .. + 3 (D = 128: and 64 on)
  float2 o[4][kDim / 2];
  float m[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < kDim / 2; ++c) o[r][c] = make_float2(0.f, 0.f);
  }
  const float sl2 = a.scale * 1.4426950408889634f;
  for (int k0 = 0; k0 < last; k0 += kPkN) {
    load_kv(k0 + kPkN);
    asm volatile("cp.async.wait_group 1;" ::: "memory");
    __syncthreads();
    const float* ks = kvs + ((k0 / kPkN) & 1) * 2 * kTile;
    const float* vs = ks + kTile;
    const int n = min(kPkN, last - k0);
    float2 x2[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) x2[r][c] = make_float2(0.f, 0.f);
#pragma unroll 4
    for (int d = 0; d < D; d += 4) {
      float4 qa[4], kb[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) qa[r] = *reinterpret_cast<const float4*>(qs + (4 * ty + r) * kLd + d);
#pragma unroll
      for (int c = 0; c < 4; ++c) kb[c] = *reinterpret_cast<const float4*>(ks + (tx + 16 * c) * kLd + d);
#pragma unroll
      for (int r = 0; r < 4; ++r)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
          x2[r][c] = __ffma2_rn(make_float2(qa[r].x, qa[r].y), make_float2(kb[c].x, kb[c].y), x2[r][c]);
          x2[r][c] = __ffma2_rn(make_float2(qa[r].z, qa[r].w), make_float2(kb[c].z, kb[c].w), x2[r][c]);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int lim = span.prior + q0 + 4 * ty + r + 1 - k0;  // keys of this tile the row sees
      float mx = -INFINITY, x[4];
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[c] = tx + 16 * c < min(lim, n) ? (x2[r][c].x + x2[r][c].y) * sl2 : -INFINITY;
        mx = fmaxf(mx, x[c]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[r], mx);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float f = exp2f(m[r] - base);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = exp2f(x[c] - base);
        sum += p;
        ps[(4 * ty + r) * kLp + tx + 16 * c] = p;
      }
      m[r] = mn;
      l[r] = l[r] * f + sum;  // this thread's keys; joined at the end
#pragma unroll
      for (int c = 0; c < kDim / 2; ++c) o[r][c] = __fmul2_rn(o[r][c], make_float2(f, f));
    }
    __syncwarp();  // a warp's two row groups write and read only their own rows of ps
#pragma unroll 2
    for (int j = 0; j < kPkN; j += 4) {
      float4 pv[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) pv[r] = *reinterpret_cast<const float4*>(ps + (4 * ty + r) * kLp + j);
#pragma unroll
      for (int jj = 0; jj < 4; ++jj)
#pragma unroll
        for (int c = 0; c < kDim / 4; ++c) {
          const float4 v = *reinterpret_cast<const float4*>(vs + (j + jj) * kLd + 64 * c + 4 * tx);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = jj == 0 ? pv[r].x : jj == 1 ? pv[r].y : jj == 2 ? pv[r].z : pv[r].w;
            o[r][2 * c] = __ffma2_rn(make_float2(p, p), make_float2(v.x, v.y), o[r][2 * c]);
            o[r][2 * c + 1] = __ffma2_rn(make_float2(p, p), make_float2(v.z, v.w), o[r][2 * c + 1]);
          }
        }
    }
    __syncthreads();  // the buffer is filled again next
  }
  // (not before: the next launch's CTAs would share the SMs of these, two to one
  // and none to another)
  pdl_trigger();
  bool fine[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = 4 * ty + r;
#pragma unroll
    for (int w = 8; w > 0; w >>= 1) l[r] += __shfl_xor_sync(0xffffffffu, l[r], w);
    const float inv = 1.f / l[r];
    bool ok = true;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(q_begin + q0 + row) * a.out_stride +
             static_cast<int64_t>(h) * D;
#pragma unroll
    for (int c = 0; c < kDim / 4; ++c) {
      const float v[4] = {o[r][2 * c].x * inv, o[r][2 * c].y * inv, o[r][2 * c + 1].x * inv, o[r][2 * c + 1].y * inv};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        ok = ok && fabsf(v[i]) < INFINITY;
        if (row < rows) out[64 * c + 4 * tx + i] = Elem<T>::from_f(v[i]);
      }
    }
    fine[r] = ok || row >= rows || !(l[r] < INFINITY);
  }
  // rows 4 ty + r of the warp's two half-warps: lane 4 half + r takes its row's part
  unsigned bad = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const unsigned b = __ballot_sync(0xffffffffu, !fine[r]);
    bad |= (b & 0xffffu ? 1u << r : 0u) | (b >> 16 ? 16u << r : 0u);
  }
  if (bad == 0) return;  // (warp-uniform)
  __syncwarp();
  const int lane = tid & 31, my_row = 4 * (tid >> 5) * 2 + (lane & 7);
  const int my_lim = min(span.prior + q0 + my_row + 1, span.keys);
  const int64_t row0 = static_cast<int64_t>(q_begin) + q0 + my_row;
  if constexpr (sizeof(T) == 4) {
    if (wide) return redo_rows<T, D, true>(a, (bad >> lane) & 1, row0, h, my_lim, span.row0);
  }
  redo_rows<T, D, false>(a, (bad >> lane) & 1, row0, h, my_lim, span.row0);
}

template <typename T, int D>
cudaError_t launch_cores(const PackedArgs& a, cudaStream_t stream) {
  constexpr int smem = (5 * 64 * (D + 4) + 64 * 68) * 4;
  static std::atomic<bool> ready[64];  // per device
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e == cudaSuccess && (dev >= 64 || !ready[dev].load())) {
    e = cudaFuncSetAttribute(packed_cores_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e == cudaSuccess && dev < 64) ready[dev].store(true);
  }
  if (e != cudaSuccess) return e;
  const int64_t tiles = a.n_tokens / kPkM + static_cast<int64_t>(a.n_seqs);
  cudaLaunchConfig_t cfg = {};
  if (tiles * a.n_q_heads > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cfg.gridDim = dim3(static_cast<unsigned>(tiles * a.n_q_heads));
  cfg.blockDim = dim3(kPkThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  const int es = sizeof(T);
  const int wide = es == 4 && ((reinterpret_cast<uintptr_t>(a.q) | reinterpret_cast<uintptr_t>(a.k) | reinterpret_cast<uintptr_t>(a.v) |
                                static_cast<uintptr_t>((a.q_stride | a.k_stride | a.v_stride) * es)) & 15) == 0;
  return cudaLaunchKernelEx(&cfg, packed_cores_kernel<T, D>, a, wide);
}


// ---- tensor-core tiles (fp16 / bf16)
//
// Tile rows are (token, query head of one KV head's group) pairs, token-major:
// 128 / G tokens of all G heads (18 tokens x 7 heads = 126 rows for 14 / 2
// heads).  One K / V tile then serves the whole group, a prompt of a few tokens
// fills a tile that would hold 128 rows of one head, and the causal diagonal
// cuts only the last tokens' worth of a key tile.  A CTA takes items of two such
// tiles (A and B) of one KV head, which share every K / V tile it loads.
// 12 warps: two warpgroups of softmax (one thread per row of tile A / B: S from
// tensor memory, running maximum and sum in registers, P back to tensor memory),
// a producer (TMA of Q, K, V), an issuer for S, one for O, and the scheduler.
//   S = Q K^T  (M 128, N 128 keys, K = D, both operands in shared memory)
//   O += P V   (M 128, N = D, K 128 keys; P from tensor memory)
// O is rescaled only when the running maximum grows by more than 2^8.
//
// Roundings.  S, the maximum, the row sum and O are fp32.  P goes into the second
// product in q's type, since both operands of an MMA have one (fp16: 2^-11 of a
// probability, bf16: 2^-8), and a third of the exponentials are polynomials good to
// 7.5e-5, below that; the row sum takes P before its rounding.  Outputs are then off
// by 1.3 times the output's own rounding (fp16 2.5e-4, bf16 2.0e-3 against 2.0e-4 and
// 1.6e-3 for fp32 probabilities).  P in two parts would be two MMAs for one.
//
// Steps A(0), B(0), A(1), B(1), .. (query tile, key tile) go through a ring of S
// buffers in tensor memory, which O leaves 384 columns (D = 64) or 256 of: three
// buffers of 128 keys, or four of 64.  P of a step overwrites its own S, so a
// buffer is free again when its PV is done, while the softmaxes work on the
// others.  (D = 64 with P in columns of its own and one S buffer a tile: 189 us
// against 183 for four prompts of up to 8,191 tokens; key tiles of 64: 216.
// D = 128 with two buffers of 128 keys: 252 us against 238 for twelve prompts of
// up to 2,048.)
// One issuer for S and one for O, both in step order, so A and B alternate: an
// issuer per tile let both fall into step, and the instructions between two
// batches of MMAs (waits, indices) take a warp that shares its scheduler with two
// softmax warps about 700 cycles, in which one issuer for both would leave the
// tensor pipe idle (1,780 cycles a step at D = 64).
//
// A chunk of few rows behind many cached keys would leave most SMs idle, or one of
// them busy long after the others.  Where the caller brings room for partials,
// items much longer than an SM's share of all key tiles are cut over their keys
// into segments of that length, items of their own; each leaves its normalised O
// with its maximum and sum, and the one that finishes last joins them in segment
// order.  16 rows behind 32,768 keys (14 heads / 2 x 64): 226 us unsplit, 42 split
// (38 by now); 512 behind 8,192: 95, 63 (53); 16 chunks of about 500 of which two
// lie behind some 3,400 keys: 79.7, 68.0 (58).  All with the laying out of the rows.
// Segments of half the share, of 1,024 keys at least or up to 32 an item were no
// faster.
//
// What bounds it: at 64 dims the exponentials, one for every 256 FLOP of MMA (a
// third of them are polynomials on the FMA pipe), at 128 dims the S -> P -> O chain
// of short items.  One prompt of 16,384 tokens: 933 TFLOP/s (14 / 2 x 64), 1,308
// (32 / 8 x 128); four of up to 8,191 tokens, 14 / 2 x 64: 167 us, 727 TFLOP/s;
// twelve of up to 2,048, 32 / 8 x 128: 222 us, 822 TFLOP/s.  No unit is full there
// (issue slots 59% and 48%, exponentials 56% and 36%, tensor pipe 38% and 49% of the
// launch): items' starts, diagonals and ends cost what long prompts do not show.
//
// Items are handed out while the kernel runs: a CTA starts with its own block
// index and then takes the indices of blocks that have not started
// (clusterlaunchcontrol.try_cancel), each once the item before has issued its last
// loads: four key tiles of work hide the latency, and no CTA holds an item that
// another could start (two
// items ahead, as two slots allow: four prompts of 4,096 tokens, 8 / 8 x 64, 164 us
// against 115; of up to 8,191, 14 / 2 x 64, 180 against 164).  So tensor memory, barriers and the
// item order are set up once per SM.  Indices run from the sequences with
// the most keys to those with the fewest, the last tokens of each first.
constexpr int kTcM = 128, kTcThreads = 384;
constexpr int kTcProducerWarp = 8, kTcQkWarp = 9, kTcSchedWarp = 10;  // warp 11: O
constexpr int kTcRegsSoftmax = 224, kTcRegsOther = 56;
constexpr int kTcRegSplit = 256 * kTcRegsSoftmax + 128 * kTcRegsOther;
constexpr int kTcMaxSorted = 384;   // sequences ordered by their keys (more: taken as they come)
constexpr int kTcItemInts = 12;
constexpr int kTcMaxSegs = 16;      // segments of an item
constexpr int kTcSegKeys = 1536;    // least keys of a segment
constexpr int kTcSplitPerSm = 4;    // split calls of up to this many items an SM
constexpr uint32_t kTcTmemCols = 512;
// log2 of the cycles that a wait takes at most (9 seconds): the other warps wait while
// one computes up to 32 rows on its own (redo_rows), some 2,000 cycles a key
constexpr int kTcWait = 34;

template <int D> struct TcShape {
  static constexpr int kN = D == 64 ? 128 : 64;         // keys per tile
  static constexpr int kStages = 4;                     // of K and of V
  static constexpr int kBufs = D == 64 ? 3 : 4;         // S buffers
  static constexpr int kHalves = D / 64;                // 64 dims are a 128-byte swizzled row
  static constexpr int kQHalf = 128 * 128, kQTile = kHalves * kQHalf;
  static constexpr int kKHalf = kN * 128, kKTile = kHalves * kKHalf;  // K and V
  static constexpr int kOffQ = 0;
  static constexpr int kOffK = 2 * kQTile;
  static constexpr int kOffV = kOffK + kStages * kKTile;
  static constexpr int kOffBar = kOffV + kStages * kKTile;
  // q_full, q_empty, K and V full / empty [stages], S full [2 tiles][bufs], P full and S free [bufs],
  // o_done [2 tiles][bufs], item_full, item_empty [2], clc, loaded
  static constexpr int kBars = 2 + 4 * kStages + 6 * kBufs + 4 + 1 + 1;
  static constexpr int kOffClc = (kOffBar + kBars * 8 + 15) / 16 * 16;
  static constexpr int kOffItem = kOffClc + 16;
  static constexpr int kOffTmem = kOffItem + 2 * kTcItemInts * 4;
  static constexpr int kOffOrder = kOffTmem + 16;        // sorted sequences, item prefix, items and key tiles of each
  static constexpr int kOffOut = (kOffOrder + (4 * kTcMaxSorted + 1) * 4 + 15) / 16 * 16;  // 2 KB per softmax warp
  static constexpr int kBytes = 1024 + kOffOut + 8 * 2048;
  static constexpr uint32_t kColO = kBufs * kN;          // O_A, O_B behind the S buffers
};
static_assert(TcShape<64>::kBytes <= 232448 && TcShape<128>::kBytes <= 232448, "tiles fit the shared memory of an SM");

struct TcParams {
  PackedArgs a;
  int group, tokens;   // query heads per KV head, tokens per tile
  int sorted;
  int n_sms;
  float scale_log2;
};

// high word of every shared-memory descriptor here: 1024 bytes between groups of 8
// rows, descriptor version 1, 128-byte swizzle (smem_desc)
constexpr uint32_t kSmemDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// tc_mma_f16 / tc_mma_f16_ts with descriptors given by their low words
template <uint32_t HI>
__device__ __forceinline__ void tc_mma_ss(uint32_t d_tmem, uint32_t alo, uint32_t blo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
      "mov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(alo), "r"(blo), "r"(idesc), "r"(accumulate), "n"(HI)
      : "memory");
}
template <uint32_t HI>
__device__ __forceinline__ void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint32_t blo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
      "mov.b64 b, {%2, %5};\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(blo), "r"(idesc), "r"(accumulate), "n"(HI)
      : "memory");
}
__device__ __forceinline__ void clc_try_cancel(void* result, uint64_t* bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(
                   smem_u32(result)),
               "r"(smem_u32(bar))
               : "memory");
}
// the cancelled block's x index, or -1
__device__ __forceinline__ int clc_index(const void* result) {
  uint32_t x = 0, ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b128 r;\n\t"
      "ld.shared.b128 r, [%2];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.u32 %1, 1, 0, p;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid::x.b32.b128 %0, r;\n\t}"
      : "+r"(x), "=r"(ok)
      : "r"(smem_u32(result))
      : "memory");
  return ok ? static_cast<int>(x) : -1;
}

// the largest of three, NaN if one is
__device__ __forceinline__ float fmax3_nan(float a, float b, float c) {
  float d;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// an item: two tiles of one (sequence, KV head), or a segment of their keys
struct TcItem {
  int s, g, tok0, q_begin, n_new, prior, keys;
  int row0;      // first key row
  int j0, j1;    // key tiles
  int seg, segs; // which of how many segments
  int idx;       // index of this one (segment q of the same item: idx + (seg - q) n_kv_heads)
};

// SPLIT: the caller brought room for partials (without it the code for them cost
// the others 4%)
template <typename T, int D, bool SPLIT>
__global__ void __launch_bounds__(kTcThreads, 1)
    packed_tc_kernel(const __grid_constant__ CUtensorMap qmap, const __grid_constant__ CUtensorMap kmap,
                     const __grid_constant__ CUtensorMap vmap, const TcParams p) {
  using Sh = TcShape<D>;
  constexpr int kStages = Sh::kStages, kHalves = Sh::kHalves, kBufs = Sh::kBufs, kN = Sh::kN;
  extern __shared__ uint8_t tc_smem[];
  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = __shfl_sync(0xffffffffu, tid >> 5, 0);  // uniform for the compiler too
  const uint32_t raw = smem_u32(tc_smem);
  uint8_t* base = tc_smem + ((1024u - (raw & 1023u)) & 1023u);
  const uint32_t sbase = smem_u32(base);
  uint64_t* q_full = reinterpret_cast<uint64_t*>(base + Sh::kOffBar);
  uint64_t* q_empty = q_full + 1;
  uint64_t* k_full = q_empty + 1;
  uint64_t* k_empty = k_full + kStages;
  uint64_t* v_full = k_empty + kStages;
  uint64_t* v_empty = v_full + kStages;
  uint64_t* s_full = v_empty + kStages;
  uint64_t* p_full = s_full + 2 * kBufs;
  uint64_t* s_free = p_full + kBufs;
  uint64_t* o_done = s_free + kBufs;
  uint64_t* item_full = o_done + 2 * kBufs;
  uint64_t* item_empty = item_full + 2;
  uint64_t* clc_bar = item_empty + 2;
  uint64_t* loaded = clc_bar + 1;  // an item's last K / V tile is on its way
  int* items = reinterpret_cast<int*>(base + Sh::kOffItem);
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(base + Sh::kOffTmem);
  int* order = reinterpret_cast<int*>(base + Sh::kOffOrder);
  int* first_item = order + kTcMaxSorted;
  int* n_items = first_item + kTcMaxSorted + 1;
  int* last_tiles = n_items + kTcMaxSorted;
  const PackedArgs& a = p.a;
  const int G = p.group, TT = p.tokens, B = a.n_seqs;

  if (warp == 0 && elect_one()) {
    mbar_init(q_full, 1);
    mbar_init(q_empty, 1);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(&k_full[i], 1);
      mbar_init(&k_empty[i], 1);
      mbar_init(&v_full[i], 1);
      mbar_init(&v_empty[i], 1);
    }
    for (int i = 0; i < 2 * kBufs; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&o_done[i], 1);
    }
    for (int i = 0; i < kBufs; ++i) {
      mbar_init(&p_full[i], 128);
      mbar_init(&s_free[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&item_full[i], 1);
      mbar_init(&item_empty[i], 11);  // 8 softmax warps, producer, two issuers
    }
    mbar_init(clc_bar, 1);
    mbar_init(loaded, 1);
    fence_barrier_init();
  }
  if (warp == kTcQkWarp) tmem_alloc(tmem_slot, kTcTmemCols);
  if (warp == kTcProducerWarp && elect_one()) {
    prefetch_tensormap(&qmap);
    prefetch_tensormap(&kmap);
    prefetch_tensormap(&vmap);
  }
  if (tid == 0) pdl_trigger();
  pdl_wait();  // the starts, q, k and v may come from the kernel before this one
  const int per_item = 2 * TT;
  __shared__ int seg_len;   // key tiles of a segment, if items are split
  // segments of the items of a sequence of so many key tiles
  auto segs_of = [&](int tiles, int len) { return tiles <= max(len + len / 4, 3 * kTcSegKeys / 2 / kN) ? 1 : min(kTcMaxSegs, (tiles + len - 1) / len); };
  if (blockIdx.x == 0)
    for (int t = tid; t < B; t += kTcThreads) {
      const int b = a.query_start_loc[t], n = a.query_start_loc[t + 1] - b;
      if (b < 0 || n < 0 || b + static_cast<int64_t>(n) > a.n_tokens) raise_flag(a.err, PKV_FLAG_BAD_QUERY_LAYOUT);
    }
  if (p.sorted) {
    // sequences by decreasing number of keys (ties by index), then the items before each
    int* keys = first_item;
    int mine = 0;
    if (tid < B) {
      mine = a.query_start_loc[tid + 1] - a.query_start_loc[tid] + (a.num_prior ? max(a.num_prior[tid], 0) : 0);
      keys[tid] = mine;
    }
    __syncthreads();
    int rank = 0;
    if (tid < B)
      for (int u = 0; u < B; ++u) rank += keys[u] > mine || (keys[u] == mine && u < tid);
    __syncthreads();
    if (tid < B) {
      const int len = max(a.query_start_loc[tid + 1] - a.query_start_loc[tid], 0);
      order[rank] = tid;
      n_items[rank] = (min(len, a.n_tokens) + per_item - 1) / per_item;
      if (SPLIT) last_tiles[rank] = (key_span(a, tid, 0, len).keys + kN - 1) / kN;
    }
    __syncthreads();
    if (warp == 0) {
      if (SPLIT) {
        // an SM's share of the key tiles of all items (a sequence's taken as
        // between those of its first and last) is a segment's length: there are
        // at most two SMs' worth more segments than items
        float work = 0.f, n = 0.f;
        int most = 0;
        for (int i = lane; i < B; i += 32) {
          n += static_cast<float>(n_items[i]);
          work += n_items[i] * (last_tiles[i] - 0.5f * n_items[i] * per_item / kN);
          most = max(most, last_tiles[i]);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          work += __shfl_xor_sync(0xffffffffu, work, o);
          n += __shfl_xor_sync(0xffffffffu, n, o);
          most = max(most, __shfl_xor_sync(0xffffffffu, most, o));
        }
        int len = max(kTcSegKeys / kN, static_cast<int>(fminf(work * a.n_kv_heads / p.n_sms + 1.f, 1e9f)));
        float split = 0.f;
        for (int i = lane; i < B; i += 32) split += static_cast<float>(n_items[i]) * segs_of(last_tiles[i], len);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) split += __shfl_xor_sync(0xffffffffu, split, o);
        // none if they pass the room all the same (lengths that are flagged); and
        // items that find an SM each anyway are split only where that shortens the
        // longest (2,048 rows behind 16,384 keys: 114 items, 192 us; in halves, 210)
        if (split * a.n_kv_heads > static_cast<float>(gridDim.x) ||
            (n * a.n_kv_heads <= p.n_sms && ceilf(split * a.n_kv_heads / p.n_sms) >= 0.9f * segs_of(most, len)))
          len = INT_MAX / 2;
        if (lane == 0) seg_len = len;
        __syncwarp();
      }
      int run = 0;
      for (int b0 = 0; b0 < B; b0 += 32) {
        const int i = b0 + lane;
        const int n = i < B ? n_items[i] * (SPLIT ? segs_of(last_tiles[i], seg_len) : 1) : 0;
        int x = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
          const int y = __shfl_up_sync(0xffffffffu, x, o);
          if (lane >= o) x += y;
        }
        if (i < B) first_item[i] = run + x - n;
        run += __shfl_sync(0xffffffffu, x, 31);
      }
      if (lane == 0) first_item[B] = run;
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tbase = __shfl_sync(0xffffffffu, *tmem_slot, 0);

  // the item of block index idx; false if there is none
  auto find_item = [&](int idx, TcItem& it) -> bool {
    const int u = idx / a.n_kv_heads;
    it.g = idx - u * a.n_kv_heads;
    it.idx = idx;
    it.seg = 0;
    it.segs = 1;
    it.j0 = 0;
    it.j1 = INT_MAX;
    int tile;
    [[maybe_unused]] int segs = 1, last = 0;
    if (p.sorted) {
      int lo = 0, hi = B - 1;
      if (u >= first_item[B]) return false;
      while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (first_item[m] <= u) lo = m; else hi = m - 1;
      }
      it.s = order[lo];
      tile = first_item[lo + 1] - 1 - u;  // last tokens first
      if (SPLIT) {
        last = last_tiles[lo];
        segs = segs_of(last, seg_len);
        it.seg = tile % segs;
        tile /= segs;
      }
      it.q_begin = a.query_start_loc[it.s];
      it.n_new = a.query_start_loc[it.s + 1] - it.q_begin;
    } else {
      int lo = 0, hi = B - 1;
      while (lo < hi) {
        const int m = (lo + hi + 1) >> 1;
        if (a.query_start_loc[m] / per_item + static_cast<int64_t>(m) <= u) lo = m; else hi = m - 1;
      }
      it.s = lo;
      it.q_begin = a.query_start_loc[lo];
      it.n_new = a.query_start_loc[lo + 1] - it.q_begin;
      const int k = static_cast<int>(u - (it.q_begin / per_item + static_cast<int64_t>(lo)));
      tile = (it.n_new + per_item - 1) / per_item - 1 - k;
    }
    if (it.q_begin < 0 || it.n_new < 0 || it.q_begin + static_cast<int64_t>(it.n_new) > a.n_tokens) return false;  // flagged above
    if (tile < 0 || tile >= (it.n_new + per_item - 1) / per_item) return false;
    it.tok0 = tile * per_item;
    const KeySpan k = key_span(a, it.s, it.q_begin, it.n_new);
    it.prior = k.prior;
    it.keys = k.keys;
    it.row0 = static_cast<int>(k.row0);
    if (segs > 1) {
      // the sequence's segments are equally long; an item uses those that its keys reach
      const int len = (last + segs - 1) / segs;
      const int tiles = (min(it.prior + min(it.tok0 + per_item, it.n_new), it.keys) + kN - 1) / kN;
      it.j0 = it.seg * len;
      it.j1 = it.j0 + len;
      it.segs = (tiles + len - 1) / len;
      if (it.seg >= it.segs) return false;
    }
    return true;
  };
  // item `k` (counted per CTA) as the scheduler published it; tok0 < 0: no more
  auto take_item = [&](int k, TcItem& it) -> bool {
    const int sl = k & 1;
    bool ok = mbar_wait<kTcWait>(&item_full[sl], (k >> 1) & 1);
    ok = __all_sync(0xffffffffu, ok);
    const int* w = items + sl * kTcItemInts;
    it.s = w[0], it.g = w[1], it.tok0 = w[2], it.q_begin = w[3], it.n_new = w[4], it.prior = w[5], it.keys = w[6], it.row0 = w[7];
    if constexpr (SPLIT) it.j0 = w[8], it.j1 = w[9], it.seg = w[10] & 255, it.segs = w[10] >> 8, it.idx = w[11];
    __syncwarp();
    if (lane == 0) mbar_arrive(&item_empty[sl]);
    if (!ok && lane == 0) raise_flag(a.err, PKV_FLAG_PIPELINE_TIMEOUT);
    return ok && it.tok0 >= 0;
  };
  // keys visible to tile x's last row, key tiles
  auto tile_keys = [&](const TcItem& it, int x) {
    const int t0 = it.tok0 + x * TT;
    const int n = min(max(it.n_new - t0, 0), TT);
    return n > 0 ? min(it.prior + t0 + n, it.keys) : 0;
  };
  // key tiles of tile x in this item (segment)
  auto item_tiles = [&](const TcItem& it, int x) {
    const int n = (tile_keys(it, x) + kN - 1) / kN;
    return SPLIT ? max(0, min(n, it.j1) - it.j0) : n;
  };

  if (warp >= 8) {
    setmaxnreg_dec<kTcRegsOther>();
    if (warp == kTcSchedWarp) {
      // ======================= scheduler (one lane) =======================
      if (lane == 0) {
        int idx = blockIdx.x;
        bool more = true;
        uint32_t clc_phase = 0;
        for (int k = 0;; ++k) {
          TcItem it;
          bool have = false;
          // taken late, so that a CTA with a long item leaves the next one to others
          if (k >= 1 && more && !mbar_wait<kTcWait>(loaded, (k - 1) & 1)) {
            raise_flag(a.err, PKV_FLAG_PIPELINE_TIMEOUT);
            more = false;
          }
          while (more) {
            if (idx >= 0) have = find_item(idx, it);
            if (have) break;
            // the next block that has not started, if there is one
            mbar_arrive_expect_tx(clc_bar, 16);
            clc_try_cancel(base + Sh::kOffClc, clc_bar);
            if (!mbar_wait<kTcWait>(clc_bar, clc_phase)) {
              raise_flag(a.err, PKV_FLAG_PIPELINE_TIMEOUT);
              more = false;
              break;
            }
            clc_phase ^= 1;
            idx = clc_index(base + Sh::kOffClc);
            fence_proxy_async_smem();  // the response was read before the next one is written
            if (idx < 0) more = false;
          }
          idx = -1;
          const int sl = k & 1;
          if (k >= 2 && !mbar_wait<kTcWait>(&item_empty[sl], ((k >> 1) & 1) ^ 1)) {
            raise_flag(a.err, PKV_FLAG_PIPELINE_TIMEOUT);
            have = false;
          }
          int* w = items + sl * kTcItemInts;
          w[0] = it.s, w[1] = it.g, w[2] = have ? it.tok0 : -1, w[3] = it.q_begin, w[4] = it.n_new, w[5] = it.prior, w[6] = it.keys,
          w[7] = it.row0;
          if constexpr (SPLIT) w[8] = it.j0, w[9] = it.j1, w[10] = it.seg | (it.segs << 8), w[11] = it.idx;
          mbar_arrive(&item_full[sl]);
          if (!have) break;
        }
      }
      __syncwarp();
    } else if (warp == kTcProducerWarp) {
      // ======================= producer =======================
      int c = 0;  // K / V tiles loaded so far
      TcItem it;
      for (int k = 0; take_item(k, it); ++k) {
        const int n_tiles = max(item_tiles(it, 0), item_tiles(it, 1));
        if (k >= 1 && !__all_sync(0xffffffffu, mbar_wait<kTcWait>(q_empty, (k - 1) & 1))) {
          if (lane == 0) raise_flag(a.err, PKV_FLAG_PIPELINE_TIMEOUT);
          break;
        }
        const bool two = it.tok0 + TT < it.n_new;
        if (elect_one()) {
          mbar_arrive_expect_tx(q_full, (two ? 2 : 1) * kHalves * G * TT * 128);
          for (int x = 0; x < (two ? 2 : 1); ++x)
#pragma unroll
            for (int h = 0; h < kHalves; ++h)
              tma_load_3d(base + Sh::kOffQ + x * Sh::kQTile + h * Sh::kQHalf, &qmap, q_full, h * 64, it.g * G,
                          it.q_begin + it.tok0 + x * TT);
        }
        __syncwarp();
        bool dead = false;
        for (int j = 0; j < n_tiles; ++j, ++c) {
          const int st = c % kStages;
          // K is free again once S of its tile is done, V once its PV is: each has a ring of its own
#pragma unroll
          for (int kv = 0; kv < 2; ++kv) {
            uint64_t* full = kv ? &v_full[st] : &k_full[st];
            if (!__all_sync(0xffffffffu, mbar_wait<kTcWait>(kv ? &v_empty[st] : &k_empty[st], ((c / kStages) & 1) ^ 1))) {
              if (lane == 0) raise_flag(a.err, PKV_FLAG_PIPELINE_TIMEOUT);
              dead = true;
              break;
            }
            if (elect_one()) {
              mbar_arrive_expect_tx(full, Sh::kKTile);
#pragma unroll
              for (int h = 0; h < kHalves; ++h)
                tma_load_3d(base + (kv ? Sh::kOffV : Sh::kOffK) + st * Sh::kKTile + h * Sh::kKHalf, kv ? &vmap : &kmap, full, h * 64, it.g,
                            it.row0 + ((SPLIT ? it.j0 : 0) + j) * kN);
            }
            __syncwarp();
          }
          if (dead) break;
        }
        if (dead) break;
        if (lane == 0) mbar_arrive(loaded);
      }
    } else {
      // ======================= MMA issuers (warp 9: S, warp 11: O) =======================
      // Descriptors are a constant high word and a low word that advances by
      // constants, ring indices are counted, not divided, and what comes from
      // shared memory is broadcast, so that the compiler knows the loops to be
      // uniform and keeps the MMAs' operands in uniform registers.
      constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
      auto wait_all = [&](uint64_t* bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait<kTcWait>(bar, parity)); };
      int st = 0, buf = 0;                 // K / V stage, S buffer
      uint32_t st_ph = 0, buf_ph = 0;      // their phases
      int turn[2] = {0, 0};                // the tile's next barrier of its ring
      int nt0 = 0, nt1 = 0;                // key tiles of A and B
      bool dead = false;
      auto open_item = [&](int k) {
        TcItem it;
        const bool ok = __all_sync(0xffffffffu, take_item(k, it));
        nt0 = __shfl_sync(0xffffffffu, item_tiles(it, 0), 0);
        nt1 = __shfl_sync(0xffffffffu, item_tiles(it, 1), 0);
        return ok;
      };
      // past a step of tile x
      auto next_step = [&](int x) {
        if (++turn[x] == kBufs) turn[x] = 0;
        if (++buf == kBufs) {
          buf = 0;
          buf_ph ^= 1;
        }
      };
      auto next_stage = [&]() {
        if (++st == kStages) {
          st = 0;
          st_ph ^= 1;
        }
      };
      if (warp == kTcQkWarp) {
        constexpr uint32_t idesc = mma_idesc_f16(fmt, 0, 0, kN, kTcM);
        const uint32_t q_lo = ((sbase + Sh::kOffQ) >> 4) | (1u << 16), k_lo = ((sbase + Sh::kOffK) >> 4) | (1u << 16);
        for (int k = 0; !dead && open_item(k); ++k) {
          if (!wait_all(q_full, k & 1)) { dead = true; break; }
          const int n_tiles = max(nt0, nt1);
          for (int j = 0; j < n_tiles && !dead; ++j) {
            if (!wait_all(&k_full[st], st_ph)) { dead = true; break; }
            const uint32_t blo = k_lo + st * (Sh::kKTile >> 4);
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if (j >= (x ? nt1 : nt0)) continue;
              if (!wait_all(&s_free[buf], buf_ph ^ 1)) { dead = true; break; }  // its last P has been read
              const uint32_t t_s = tbase + buf * kN;
              // S signals a ring of barriers of its own tile: the other tile's softmax
              // may be items ahead, where it would take an old phase for its own
              uint64_t* sf = s_full + x * kBufs + turn[x];
              const bool last = x == 1 || j >= nt1;
              if (elect_one()) {
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < 4 * kHalves; ++kk)
                  tc_mma_ss<kSmemDescHi>(t_s, q_lo + x * (Sh::kQTile >> 4) + (kk >> 2) * (Sh::kQHalf >> 4) + (kk & 3) * 2,
                                         blo + (kk >> 2) * (Sh::kKHalf >> 4) + (kk & 3) * 2, idesc, kk > 0 ? 1u : 0u);
                tc_commit(sf);
                if (last) tc_commit(&k_empty[st]);
                if (last && j + 1 == n_tiles) tc_commit(q_empty);
              }
              __syncwarp();
              next_step(x);
            }
            next_stage();
          }
        }
      } else {
        constexpr uint32_t idesc = mma_idesc_f16(fmt, 0, 1, D, kTcM);
        // V is the MN-major operand: 8 keys every 1024 bytes, the second 64 dims (D = 128) a half tile on
        const uint32_t v_lo = ((sbase + Sh::kOffV) >> 4) | (static_cast<uint32_t>(kHalves == 2 ? Sh::kKHalf >> 4 : 1) << 16);
        for (int k = 0; !dead && open_item(k); ++k) {
          const int n_tiles = max(nt0, nt1);
          for (int j = 0; j < n_tiles && !dead; ++j) {
            if (!wait_all(&v_full[st], st_ph)) { dead = true; break; }
            const uint32_t blo = v_lo + st * (Sh::kKTile >> 4);
            const uint32_t keep = j > 0 ? 1u : 0u;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
              if (j >= (x ? nt1 : nt0)) continue;
              if (!wait_all(&p_full[buf], buf_ph)) { dead = true; break; }
              const uint32_t t_o = tbase + Sh::kColO + x * D, t_p = tbase + buf * kN;
              if (elect_one()) {
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < kN / 16; ++kk) tc_mma_ts<kSmemDescHi>(t_o, t_p + kk * 8, blo + kk * 128, idesc, kk > 0 ? 1u : keep);
                tc_commit(&s_free[buf]);
                tc_commit(o_done + x * kBufs + turn[x]);
                if (x == 1 || j >= nt1) tc_commit(&v_empty[st]);
              }
              __syncwarp();
              next_step(x);
            }
            next_stage();
          }
        }
      }
      if (dead && lane == 0) raise_flag(a.err, PKV_FLAG_PIPELINE_TIMEOUT);
    }
  } else {
    setmaxnreg_inc<kTcRegsSoftmax>();
    // ======================= softmax and epilogue (thread = row of tile x) =======================
    const int x = warp >> 2, r = tid & 127;
    const uint32_t lane_off = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_o = tbase + Sh::kColO + x * D + lane_off;
    const int rtok = r / G, rhead = r - rtok * G;
    const float sl2 = p.scale_log2;
    int cx = 0;   // PVs of this tile so far
    int n0 = 0;   // steps of both tiles so far
    bool dead = false;
    TcItem it;
    unsigned again;  // lanes whose row may have to be computed again
    int k = 0;
    do {
    again = 0;
    for (; take_item(k, it); ++k) {
      const int kvx = tile_keys(it, x), ntx = item_tiles(it, x), nto = item_tiles(it, 1 - x);
      // PV number i of this item and tile has completed.  PVs signal a ring of
      // barriers: a wait tells a phase from the one before it only, and the S
      // that the caller has seen vouches for the PV a ring's length back.
      auto wait_pv = [&](int i) {
        const int w = cx + i;
        if (!dead && !mbar_wait<kTcWait>(&o_done[x * kBufs + w % kBufs], (w / kBufs) & 1)) dead = true;
      };
      const int tok = it.tok0 + x * TT + rtok;
      const bool row_valid = rtok < TT && tok < it.n_new;
      // rows without a token are not stored, so they need no mask (one of them
      // would send its warp through the masking code at every step)
      const int lim = row_valid ? min(it.prior + tok + 1, kvx) : INT_MAX;
      float m_used = -INFINITY, l = 0.f;
      bool odd = false;  // a NaN or +infinity among the visible scores: the row is NaN
      for (int j = 0; j < ntx; ++j) {
        // the step's number (A(j) and B(j) alternate while both tiles have key tiles), its S buffer
        const int n = n0 + (x == 0 ? (nto > 0 ? 2 * j : j) : (j < nto ? 2 * j + 1 : nto + j));
        const int b = n % kBufs;
        const uint32_t t_s = tbase + b * kN + lane_off;
        if (!dead && !mbar_wait<kTcWait>(&s_full[x * kBufs + (cx + j) % kBufs], ((cx + j) / kBufs) & 1)) dead = true;
        __syncwarp();
        tc_fence_after();
        uint32_t sr[kN / 32][32];
#pragma unroll
        for (int c4 = 0; c4 < kN / 32; ++c4) tmem_ld32(t_s + c4 * 32, sr[c4]);
        tmem_wait_ld_regs(sr[0]);
#pragma unroll
        for (int c4 = 1; c4 < kN / 32; ++c4) reg_after_wait(sr[c4]);
        const int kbase = ((SPLIT ? it.j0 : 0) + j) * kN;
        if (kbase + kN > lim) {
#pragma unroll
          for (int c = 0; c < kN; ++c)
            if (kbase + c >= lim) sr[c >> 5][c & 31] = __float_as_uint(-INFINITY);
        }
        float m8[8];
#pragma unroll
        for (int q = 0; q < 8; ++q) m8[q] = fmax3_nan(__uint_as_float(sr[0][q]), __uint_as_float(sr[0][q + 8]), -INFINITY);
#pragma unroll
        for (int c = 16; c < kN; c += 16) {
#pragma unroll
          for (int q = 0; q < 8; ++q)
            m8[q] = fmax3_nan(m8[q], __uint_as_float(sr[c >> 5][(c & 31) + q]), __uint_as_float(sr[(c + 8) >> 5][((c + 8) & 31) + q]));
        }
        const float mt = fmax3_nan(fmax3_nan(m8[0], m8[1], m8[2]), fmax3_nan(m8[3], m8[4], m8[5]), fmax3_nan(m8[6], m8[7], -INFINITY)) * sl2;
        odd = odd || !(mt < INFINITY);  // (the polynomials below would swallow a NaN)
        float factor = 1.f;
        if (mt > m_used + 8.f) {
          factor = exp2f(m_used - mt);
          m_used = mt;
          l *= factor;
        }
        const bool rescale = __any_sync(0xffffffffu, factor != 1.f) && j > 0;
        const float nm = (m_used == -INFINITY) ? 0.f : -m_used;
        float2 ls[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
        const float2 sl2v = make_float2(sl2, sl2), nmv = make_float2(nm, nm);
#pragma unroll
        for (int half = 0; half < kN / 64; ++half) {
          uint32_t pk[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            const int c2 = half * 32 + i, c = 2 * c2;
            const float2 xs = __ffma2_rn(make_float2(__uint_as_float(sr[c >> 5][c & 31]), __uint_as_float(sr[(c + 1) >> 5][(c + 1) & 31])),
                                         sl2v, nmv);
            const float2 pp = c2 % 3 == 2 ? exp2_poly3x2(xs) : make_float2(ex2_approx(xs.x), ex2_approx(xs.y));
            ls[i & 1] = __fadd2_rn(ls[i & 1], pp);
            pk[i] = pack2<T>(pp.x, pp.y);
          }
          if (half == 0 && rescale) {  // after the PV before this step
            wait_pv(j - 1);
            __syncwarp();
            tc_fence_after();
#pragma unroll
            for (int c2 = 0; c2 < D / 32; ++c2) {
              uint32_t orr[32];
              tmem_ld32(t_o + c2 * 32, orr);
              tmem_wait_ld_regs(orr);
#pragma unroll
              for (int c = 0; c < 32; ++c) orr[c] = __float_as_uint(__uint_as_float(orr[c]) * factor);
              tmem_st32(t_o + c2 * 32, orr);
            }
          }
          tmem_st32(t_s + half * 32, pk);
        }
        l += (ls[0].x + ls[1].x) + (ls[0].y + ls[1].y);
        tmem_wait_st();
        tc_fence_before();
        mbar_arrive(&p_full[b]);
      }
      if (odd) l = NAN;
      else if (m_used == -INFINITY) l = 0.f;  // nothing seen, or scores of -infinity alone
      // ---- epilogue: O / l -> out
      bool fine = true;
      const int64_t row = static_cast<int64_t>(it.q_begin) + tok;
      const int head = it.g * G + rhead;
      // 32 columns at a time through the warp's 2 KB: a store then covers 64
      // bytes of each of 8 rows (each thread storing its own row, 16 bytes
      // here and there, took 3,300 cycles an item at D = 64, 5,500 at 128)
      const int64_t off = row * a.out_stride + static_cast<int64_t>(head) * D;
      const unsigned rows_ok = __ballot_sync(0xffffffffu, row_valid);
      uint8_t* mine = base + Sh::kOffOut + warp * 2048;
      int64_t roff[4];
#pragma unroll
      for (int r8 = 0; r8 < 4; ++r8) roff[r8] = __shfl_sync(0xffffffffu, off, r8 * 8 + (lane >> 2));
      auto store32 = [&](int c2, const float* f) {
#pragma unroll
        for (int c8 = 0; c8 < 4; ++c8)
          *reinterpret_cast<uint4*>(mine + lane * 64 + ((c8 ^ ((lane >> 1) & 3)) << 4)) =
              make_uint4(pack2<T>(f[8 * c8], f[8 * c8 + 1]), pack2<T>(f[8 * c8 + 2], f[8 * c8 + 3]),
                         pack2<T>(f[8 * c8 + 4], f[8 * c8 + 5]), pack2<T>(f[8 * c8 + 6], f[8 * c8 + 7]));
        __syncwarp();
#pragma unroll
        for (int r8 = 0; r8 < 4; ++r8) {
          const int rr = r8 * 8 + (lane >> 2), c8 = lane & 3;
          const uint4 v = *reinterpret_cast<const uint4*>(mine + rr * 64 + ((c8 ^ ((rr >> 1) & 3)) << 4));
          if ((rows_ok >> rr) & 1) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + roff[r8] + c2 * 32 + c8 * 8) = v;
        }
        __syncwarp();
      };
      // partials of segment q: four columns of a tile's 128 rows side by side
      auto part_slot = [&](int q) { return static_cast<int64_t>(it.idx + (it.seg - q) * a.n_kv_heads) * 2 + x; };
      const bool whole = !SPLIT || it.segs == 1;
      if (ntx > 0) {
        wait_pv(ntx - 1);
        __syncwarp();
        tc_fence_after();
        const float inv = l > 0.f ? 1.f / l : NAN;  // (0: scores of -infinity alone, or a segment without a say)
        float fsum = 0.f;
#pragma unroll
        for (int c2 = 0; c2 < D / 32; ++c2) {
          uint32_t o[32];
          tmem_ld32(t_o + c2 * 32, o);
          tmem_wait_ld_regs(o);
          float f[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            fsum += fabsf(__uint_as_float(o[i]));
            f[i] = __uint_as_float(o[i]) * inv;
          }
          if (whole) {
            store32(c2, f);
          } else {
            float4* to = reinterpret_cast<float4*>(a.part_o) + (part_slot(it.seg) * (D / 4) + c2 * 8) * 128 + r;
#pragma unroll
            for (int i = 0; i < 8; ++i) to[i * 128] = make_float4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]);
          }
        }
        tc_fence_before();  // O is read before the next item's PV (ordered by p_full)
        if (whole) fine = !row_valid || !(l > 0.f && l < INFINITY) || fsum < INFINITY;
      }
      if (!whole) {
        // each warp on its own: its rows of all segments are in memory once their
        // warps have counted
        a.part_ml[part_slot(it.seg) * 128 + r] = make_float2(m_used, ntx > 0 ? l : 0.f);
        __threadfence();
        __syncwarp();
        int seen = 0;
        if (lane == 0) seen = atomicAdd(a.part_count + (it.idx + it.seg * a.n_kv_heads) * 8 + warp, 1);
        if (__shfl_sync(0xffffffffu, seen, 0) == it.segs - 1) {
          __threadfence();
          // several segments' loads at a time: each is a trip to L2
          float top = -INFINITY, sum = 0.f, w[kTcMaxSegs];
          float2 ml[kTcMaxSegs];
#pragma unroll 4
          for (int q = 0; q < kTcMaxSegs; ++q) {
            if (q < it.segs) ml[q] = __ldcg(a.part_ml + part_slot(q) * 128 + r);
          }
          for (int q = 0; q < it.segs; ++q)
            if (ml[q].y != 0.f) top = fmaxf(top, ml[q].x);  // (0: the row saw nothing there)
          for (int q = 0; q < it.segs; ++q) {
            w[q] = ml[q].y != 0.f ? ex2_approx(ml[q].x - top) * ml[q].y : 0.f;
            sum += w[q];
          }
          const float inv = sum > 0.f ? 1.f / sum : NAN;  // (0: scores of -infinity alone)
          float fsum = 0.f;
          for (int c2 = 0; c2 < D / 32; ++c2) {
            float f[32];
#pragma unroll
            for (int i = 0; i < 32; ++i) f[i] = 0.f;
            for (int q = 0; q < it.segs; q += 2) {
              const float w0 = w[q] * inv, w1 = q + 1 < it.segs ? w[q + 1] * inv : 0.f;
              const float4* from0 = reinterpret_cast<const float4*>(a.part_o) + (part_slot(q) * (D / 4) + c2 * 8) * 128 + r;
              const float4* from1 = from0 - (q + 1 < it.segs ? a.n_kv_heads * 2 * (D / 4) * 128 : 0);
              float4 v0[8], v1[8];
#pragma unroll
              for (int i = 0; i < 8; ++i) v0[i] = __ldcg(from0 + i * 128);
#pragma unroll
              for (int i = 0; i < 8; ++i) v1[i] = __ldcg(from1 + i * 128);
              // (without a weight its O may not have been written)
#pragma unroll
              for (int i = 0; i < 8; ++i) {
                if (w0 != 0.f) {
                  f[4 * i] = fmaf(w0, v0[i].x, f[4 * i]);
                  f[4 * i + 1] = fmaf(w0, v0[i].y, f[4 * i + 1]);
                  f[4 * i + 2] = fmaf(w0, v0[i].z, f[4 * i + 2]);
                  f[4 * i + 3] = fmaf(w0, v0[i].w, f[4 * i + 3]);
                }
                if (w1 != 0.f) {
                  f[4 * i] = fmaf(w1, v1[i].x, f[4 * i]);
                  f[4 * i + 1] = fmaf(w1, v1[i].y, f[4 * i + 1]);
                  f[4 * i + 2] = fmaf(w1, v1[i].z, f[4 * i + 2]);
                  f[4 * i + 3] = fmaf(w1, v1[i].w, f[4 * i + 3]);
                }
              }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) fsum += fabsf(f[i]);
            __syncwarp();
            store32(c2, f);
          }
          fine = !row_valid || !(sum > 0.f && sum < INFINITY) || fsum < INFINITY;
        }
      }
      cx += ntx;
      n0 += ntx + nto;
      // rows that a key they must not see may have spoiled: out of the loop over items
      // and back into it (with the call inside, the whole loop was 5% slower)
      again = __ballot_sync(0xffffffffu, !fine);
      if (again) {
        reinterpret_cast<int4*>(mine)[lane] = make_int4(static_cast<int>(row), head, lim, it.row0);
        ++k;
        break;
      }
    }
    if (again) {
      const int4 me = reinterpret_cast<const int4*>(base + Sh::kOffOut + warp * 2048)[lane];
      redo_rows<T, D, true>(a, (again >> lane) & 1, me.x, me.y, me.z, me.w);
    }
    } while (again);
    if (dead && r == 0) raise_flag(a.err, PKV_FLAG_PIPELINE_TIMEOUT);
  }
  tc_fence_before();
  __syncthreads();
  if (warp == kTcQkWarp) {
    tc_fence_after();
    tmem_dealloc(tbase, kTcTmemCols);
  }
}

bool tc_supported(const PackedArgs& a) {
  auto al = [](const void* q, int64_t stride) { return ((reinterpret_cast<uintptr_t>(q) | static_cast<uintptr_t>(stride * 2)) & 15) == 0; };
  return a.dtype != PKV_DTYPE_F32 && a.n_q_heads / a.n_kv_heads <= 64 && al(a.q, a.q_stride) && al(a.k, a.k_stride) &&
         al(a.v, a.v_stride) && al(a.out, a.out_stride);
}

int64_t tc_items(int n_seqs, int n_tokens, int n_q_heads, int n_kv_heads) {
  const int tokens = kTcM / (n_q_heads / n_kv_heads);
  return (n_tokens / (2 * tokens) + static_cast<int64_t>(n_seqs)) * n_kv_heads;
}

template <typename T, int D, bool SPLIT>
cudaError_t launch_tc(const PackedArgs& a, cudaStream_t stream) {
  auto kern = packed_tc_kernel<T, D, SPLIT>;
  static std::atomic<int> ready[64];  // per device: 0 not asked, SMs: ready, -1 the register split does not fit
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int state = dev < 64 ? ready[dev].load() : 0;
  if (state == 0) {
    cudaFuncAttributes fa;
    e = cudaFuncGetAttributes(&fa, kern);
    if (e != cudaSuccess) return e;
    state = -1;
    if (fa.numRegs * kTcThreads >= kTcRegSplit) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, TcShape<D>::kBytes);
      if (e == cudaSuccess) e = cudaDeviceGetAttribute(&state, cudaDevAttrMultiProcessorCount, dev);
      if (e != cudaSuccess) return e;
    }
    if (dev < 64) ready[dev].store(state);
  }
  if (state < 0) return launch_cores<T, D>(a, stream);
  TcParams p{};
  p.a = a;
  p.group = a.n_q_heads / a.n_kv_heads;
  p.tokens = kTcM / p.group;
  p.sorted = a.n_seqs <= kTcMaxSorted;
  p.n_sms = state;
  p.scale_log2 = a.scale * 1.4426950408889634f;
  CUtensorMap qm, km, vm;
  int rc = encode_rows_tensormap(&qm, a.q, a.q_stride, a.n_tokens, a.n_q_heads, D, a.dtype, p.group, p.tokens);
  if (rc == 0) rc = encode_rows_tensormap(&km, a.k, a.k_stride, a.n_key_rows, a.n_kv_heads, D, a.dtype, 1, TcShape<D>::kN);
  if (rc == 0) rc = encode_rows_tensormap(&vm, a.v, a.v_stride, a.n_key_rows, a.n_kv_heads, D, a.dtype, 1, TcShape<D>::kN);
  if (rc != 0) return cudaErrorNotSupported;
  int64_t items = tc_items(a.n_seqs, a.n_tokens, a.n_q_heads, a.n_kv_heads);
  if (items > 0x7fffffff) return cudaErrorInvalidConfiguration;
  if (SPLIT) items = a.n_parts;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(items));
  cfg.blockDim = dim3(kTcThreads);
  cfg.dynamicSmemBytes = TcShape<D>::kBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kern, qm, km, vm, p);
}

}  // namespace

// The room for partials: a slot for every item and two for each of 148 SMs
// besides; none if no item can be long enough.  Calls with more than
// kTcSplitPerSm items an SM are not split (they fill the GPU, and their partials
// would fill memory).
int packed_split_parts(int n_seqs, int n_tokens, int n_q_heads, int n_kv_heads, int64_t key_limit, int dtype) {
  if (dtype == PKV_DTYPE_F32 || n_seqs > kTcMaxSorted || n_q_heads / n_kv_heads > 64) return 0;
  if (key_limit <= 3 * kTcSegKeys / 2) return 0;
  const int64_t items = tc_items(n_seqs, n_tokens, n_q_heads, n_kv_heads);
  return items > 148 * kTcSplitPerSm ? 0 : static_cast<int>(items + 2 * 148);
}
cudaError_t launch_packed_attention(const PackedArgs& a, cudaStream_t stream) {
  if (a.n_tokens == 0 || a.n_seqs == 0) return cudaSuccess;
  auto go = [&](auto tag) {
    using T = decltype(tag);
    if constexpr (sizeof(T) == 2) {
      if (tc_supported(a)) {
        if (a.n_parts > 0) return a.head_dim == 64 ? launch_tc<T, 64, true>(a, stream) : launch_tc<T, 128, true>(a, stream);
        return a.head_dim == 64 ? launch_tc<T, 64, false>(a, stream) : launch_tc<T, 128, false>(a, stream);
      }
    }
    return a.head_dim == 64 ? launch_cores<T, 64>(a, stream) : launch_cores<T, 128>(a, stream);
  };
  if (a.dtype == PKV_DTYPE_F16) return go(__half{});
  if (a.dtype == PKV_DTYPE_BF16) return go(__nv_bfloat16{});
  return go(float{});
}

}  // namespace pkv
