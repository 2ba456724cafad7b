// pkv_int8.cu -- int8 pools with one power-of-two scale per (block, KV head):
// the quantising append, the fetch of rows as values, and the pass that lays a
// step's visible keys and values out for the chunked prefill.
//
// The reference keeps 32-bit pools (mini_engine/paged/block_manager.py:37) and
// names a compact cache as its next step (mini_engine/quant.py); the append
// replaces the scatter of append_and_fetch (block_manager.py:121-131) and the
// fetch its gather (block_manager.py:136-141).
//
// Format.  Element x of row (block b, offset o, head h) is stored as the integer
// q = rne(x / s) with s = s[b][h] the smallest power of two 2^e, e >= -120, for
// which absmax <= 127 s over the block's rows of that head.  With a power of two
// x / s and q s are exact, so a value is off by at most s / 2 (absmax / 127 at
// most), dequantising to fp16 / bf16 / fp32 is exact (7 bits), and when a later
// token needs a larger scale the held integers become rne(q * s_old / s_new),
// an exact product rounded once; the roundings of a block that grows k times add
// up to less than one step (1/2 + 1/4 + ...), which no other ratio gives.
// Infinities are stored as +-127 and do not enter absmax; NaN is stored as 0.
//
// Work split of the append and the fetch: one warp per (sequence, touched block,
// K or V, head or, where there are warps enough for the GPU without, several
// heads in turn), so one warp owns a scale and the rows under it and nothing is
// atomic.  The host does not know how many blocks each sequence touches, but
// floor(n / b) + 2 bounds it, so sequence i's units start at
// floor(start_i / b) + 2 i and a warp finds its sequence by a search on the
// start positions: no prefix pass, no scratch.  Bound by the bytes of the
// rows for prompts (64 of 200 to 2,000 tokens, 8 x 128 in bf16, appended and
// fetched: 460 MB in 105 us, 67% of the copy rate), by launch and round trips for
// decode steps (256 single tokens, 2 x 64: 3.9 us, 7.4 with the fetch).
#include <type_traits>

#include "pkv_common.cuh"
#include "pkv_internal.h"

namespace pkv {

namespace {

constexpr int kI8Warps = 4;
constexpr int kI8Regs = 8;  // 16-byte loads a lane keeps

// the block scale for rows of largest finite magnitude amax
__device__ __forceinline__ float int8_block_scale(float amax) {
  const uint32_t b = __float_as_uint(amax);
  // 1.f * 2^E holds amax <= 127 * 2^(E-6) iff 1.f <= 127/64
  int e = static_cast<int>(b >> 23) - 127 - ((b & 0x7fffffu) <= 0x7e0000u ? 6 : 5);
  e = max(e, -120);  // zeros and subnormals too
  return __uint_as_float(static_cast<uint32_t>(e + 127) << 23);
}

__device__ __forceinline__ int int8_round(float x, float inv) {
  return min(127, max(-127, __float2int_rn(x * inv)));  // NaN -> 0, infinities saturate
}
__device__ __forceinline__ uint32_t pack_bytes(int a, int b, int c, int d) {
  return (a & 255) | ((b & 255) << 8) | ((c & 255) << 16) | (static_cast<uint32_t>(d) << 24);
}

// four values of at most 127.5 in size as bytes, rounded to nearest even: the low
// byte of 1.5 * 2^23 + x * inv (x * inv is exact, the sum rounds once)
__device__ __forceinline__ uint32_t pack_scaled(const float* v, float2 inv) {
  const float2 big = make_float2(12582912.f, 12582912.f);
  const float2 a = __ffma2_rn(make_float2(v[0], v[1]), inv, big), b = __ffma2_rn(make_float2(v[2], v[3]), inv, big);
  return __byte_perm(__byte_perm(__float_as_uint(a.x), __float_as_uint(a.y), 0x0040),
                     __byte_perm(__float_as_uint(b.x), __float_as_uint(b.y), 0x0040), 0x5410);
}

// four consecutive elements; `vec` says whether they may be loaded as one word
template <typename T>
__device__ __forceinline__ void load4_any(const T* p, bool vec, float* v) {
  if (vec) {
    load4_f<T>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = Elem<T>::to_f(p[i]);
  }
}
template <typename T>
__device__ __forceinline__ void store4_any(T* p, bool vec, const float* v) {
  if (vec) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
    } else {
      *reinterpret_cast<uint2*>(p) = make_uint2(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]));
    }
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = Elem<T>::from_f(v[i]);
  }
}
// signed bytes as floats, exactly and without conversion instructions: x + 128 as
// the low byte of 2^23 + 128 + x
__device__ __forceinline__ void bytes_to_f(uint32_t w, float* v) {
  w ^= 0x80808080u;
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540 + i)) - 8388736.f;
}

// 16 bytes as floats
template <typename T>
__device__ __forceinline__ void unpack16(const uint4& w, float* v) {
  const uint32_t u[4] = {w.x, w.y, w.z, w.w};
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __uint_as_float(u[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      if constexpr (std::is_same<T, __half>::value) {
        const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&u[i]));
        v[2 * i] = f.x, v[2 * i + 1] = f.y;
      } else {
        v[2 * i] = __uint_as_float(u[i] << 16), v[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u);
      }
    }
  }
}

// the sequence and touched-block number of unit u (see the header comment)
struct Unit {
  int s, j;        // sequence, number of the touched block
  int row0, n;     // first packed row of the sequence, rows of the sequence
  int ctx;         // tokens of the sequence after the call
};
// (whole warp) the last sequence whose units start at or before u: 32 positions a
// round, so two dependent loads for up to 1,024 sequences where halving takes ten
__device__ __forceinline__ bool find_unit(const int32_t* start_loc, const int32_t* context_lens,
                                          int n_seqs, int n_rows, int bs, int64_t u, Unit& w) {
  const int lane = threadIdx.x & 31;
  int lo = 0, n = n_seqs;  // the answer is in [lo, lo + n)
  while (n > 1) {
    const int step = (n + 31) / 32, m = lo + lane * step;
    const bool before = lane * step < n && start_loc[m] / bs + 2 * static_cast<int64_t>(m) <= u;
    const unsigned hits = __ballot_sync(0xffffffffu, before) | 1u;  // (lane 0: a bad first start goes to sequence lo)
    const int k = 31 - __clz(hits);
    n = min(step, n - k * step);
    lo += k * step;
  }
  w.s = lo;
  w.row0 = start_loc[lo];
  w.j = static_cast<int>(u - (w.row0 / bs + 2 * static_cast<int64_t>(lo)));
  w.n = start_loc[lo + 1] - w.row0;
  w.ctx = context_lens[lo];
  return w.row0 >= 0 && w.n > 0 && w.j >= 0 && w.row0 + static_cast<int64_t>(w.n) <= n_rows;
}

template <typename T>
__global__ void __launch_bounds__(kI8Warps * 32) append_int8_kernel(const Int8RowsArgs a) {
  pdl_trigger();
  pdl_wait();  // the metadata and the rows may come from the kernel before this one
  const int lane = threadIdx.x & 31;
  const int64_t wid = static_cast<int64_t>(blockIdx.x) * kI8Warps + (threadIdx.x >> 5);
  const int per_half = (a.n_kv_heads + a.heads_per_warp - 1) / a.heads_per_warp, per_unit = 2 * per_half;
  const int64_t u = wid / per_unit;
  const int rem = static_cast<int>(wid - u * per_unit);
  const bool isv = rem >= per_half;
  const int h0 = (isv ? rem - per_half : rem) * a.heads_per_warp, h1 = min(a.n_kv_heads, h0 + a.heads_per_warp);
  const int bs = a.block_size, D = a.head_dim;
  if (u >= a.n_units) return;
  Unit w;
  if (!find_unit(a.start_loc, a.context_lens, a.n_seqs, a.n_rows, bs, u, w)) {
    if (w.j == 0 && rem == 0 && lane == 0 &&
        (w.row0 < 0 || w.n < 0 || w.row0 + static_cast<int64_t>(w.n) > a.n_rows))
      raise_flag(a.err, PKV_FLAG_BAD_QUERY_LAYOUT);
    return;
  }
  if (w.ctx == 0) return;  // a padding or unserved sequence: nothing is written
  const int prior = w.ctx - w.n;
  if (prior < 0) {
    if (w.j == 0 && rem == 0 && lane == 0) raise_flag(a.err, PKV_FLAG_BAD_QUERY_LAYOUT);
    return;
  }
  const int jb = prior / bs + w.j;  // table column
  const int64_t blk0 = static_cast<int64_t>(jb) * bs;
  if (blk0 >= w.ctx) return;
  if (jb >= a.max_blocks) {
    if (rem == 0 && lane == 0) raise_flag(a.err, PKV_FLAG_CONTEXT_EXCEEDS_TABLE);
    return;
  }
  const int id = a.block_tables[static_cast<int64_t>(w.s) * a.bt_stride + jb];
  if (id < 0 || id >= a.num_blocks) {
    if (rem == 0 && lane == 0) raise_flag(a.err, PKV_FLAG_BLOCK_OUT_OF_RANGE);
    return;
  }
  const int held = max(0, prior - static_cast<int>(blk0));                // rows the block keeps
  const int end = min(bs, static_cast<int>(w.ctx - blk0));                // rows after the call
  const int src0 = w.row0 + static_cast<int>(blk0) + held - prior;        // packed row of row `held`
  const int64_t stride = isv ? a.v_stride : a.k_stride;
  const bool vec = isv ? a.v_vec : a.k_vec;
  const int64_t pitch = static_cast<int64_t>(a.n_kv_heads) * D;
  for (int h = h0; h < h1; ++h) {
  const T* src = static_cast<const T*>(isv ? a.v : a.k) + src0 * stride + static_cast<int64_t>(h) * D;
  int8_t* dst = static_cast<int8_t*>(isv ? a.v_pool : a.k_pool) +
                (static_cast<int64_t>(id) * bs * a.n_kv_heads + h) * D;
  float* scale = (isv ? a.v_scale : a.k_scale) + static_cast<int64_t>(id) * a.n_kv_heads + h;

  // units of four consecutive elements: cpr to a row
  const int cpr = D / 4, total = (end - held) * cpr;
  // new rows that one load of 16 bytes a lane, at most kI8Regs times, can bring:
  // they stay in registers between absmax and rounding (4 KB: 16 rows of 128 dims or
  // 32 of 64 in 16 bits, 16 of 64 in fp32); larger blocks are read twice
  constexpr int kPer = 16 / sizeof(T), kLog = sizeof(T) == 2 ? 3 : 2;
  const int chunks = total * 4 / kPer, row_log = (D == 64 ? 6 : 7) - kLog;  // 2^row_log chunks to a row
  bool once = (isv ? a.v_vec16 : a.k_vec16) && chunks <= 32 * kI8Regs;
  uint4 raw[kI8Regs];
  float amax = 0.f;
  // a load of the warp covers 32 >> row_log rows
  const int lane_row = lane >> row_log, lane_col = (lane & ((1 << row_log) - 1)) << kLog;
  if (once) {
    const T* from = src + lane_row * stride + lane_col;
    const int64_t step = (32 >> row_log) * stride;
#pragma unroll
    for (int i = 0; i < kI8Regs; ++i) {
      raw[i] = make_uint4(0u, 0u, 0u, 0u);
      if (i * 32 + lane < chunks) raw[i] = *reinterpret_cast<const uint4*>(from);
      from += step;
    }
    // the largest magnitude as an integer: of the bit patterns without their
    // signs (two 16-bit ones at a time), which order as the values do, with
    // infinities and NaN above all
    uint32_t top = 0u;
#pragma unroll
    for (int i = 0; i < kI8Regs; ++i) {
      constexpr uint32_t kMask = sizeof(T) == 4 ? 0x7fffffffu : 0x7fff7fffu;
      const uint32_t x = raw[i].x & kMask, y = raw[i].y & kMask, z = raw[i].z & kMask, w4 = raw[i].w & kMask;
      if constexpr (sizeof(T) == 4) {
        top = max(max(top, max(x, y)), max(z, w4));
      } else {
        top = __vimax3_u16x2(__vimax3_u16x2(top, x, y), z, w4);
      }
    }
    if constexpr (sizeof(T) == 4) {
      amax = __uint_as_float(top);
    } else {
      const uint32_t m = max(top & 0xffffu, top >> 16);
      if constexpr (std::is_same<T, __half>::value) amax = __half2float(__ushort_as_half(static_cast<unsigned short>(m)));
      else amax = __uint_as_float(m << 16);
    }
    // rows with infinities or NaN take the other path
    once = __all_sync(0xffffffffu, amax < INFINITY);
  }
  if (!once) {
    amax = 0.f;
    for (int c = lane; c < total; c += 32) {
      const int r = c / cpr, d = (c - r * cpr) * 4;
      float v[4];
      load4_any<T>(src + r * stride + d, vec, v);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float m = fabsf(v[i]);
        amax = fmaxf(amax, m < INFINITY ? m : 0.f);
      }
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
  float sc = int8_block_scale(amax);
  if (held > 0) {
    const float old = *scale;
    sc = fmaxf(sc, old);
    if (sc != old) {  // the held rows on the larger scale
      const float ratio = old * (1.f / sc);
      for (int c = lane; c < held * cpr; c += 32) {
        const int r = c / cpr, d = (c - r * cpr) * 4;
        uint32_t* p = reinterpret_cast<uint32_t*>(dst + r * pitch + d);
        float v[4];
        bytes_to_f(*p, v);
        *p = pack_bytes(int8_round(v[0], ratio), int8_round(v[1], ratio), int8_round(v[2], ratio),
                        int8_round(v[3], ratio));
      }
    }
  }
  const float inv = 1.f / sc;  // exact: a power of two
  if (once) {
    const float2 inv2 = make_float2(inv, inv);
    int8_t* to = dst + (held + lane_row) * pitch + lane_col;
    const int64_t step = (32 >> row_log) * pitch;
#pragma unroll
    for (int i = 0; i < kI8Regs; ++i, to += step) {
      if (i * 32 + lane >= chunks) continue;
      float v[kPer];
      unpack16<T>(raw[i], v);
      if constexpr (kPer == 8) {
        *reinterpret_cast<uint2*>(to) = make_uint2(pack_scaled(v, inv2), pack_scaled(v + 4, inv2));
      } else {
        *reinterpret_cast<uint32_t*>(to) = pack_scaled(v, inv2);
      }
    }
  } else {
    for (int c = lane; c < total; c += 32) {
      const int r = c / cpr, d = (c - r * cpr) * 4;
      float v[4];
      load4_any<T>(src + r * stride + d, vec, v);
      *reinterpret_cast<uint32_t*>(dst + (held + r) * pitch + d) =
          pack_bytes(int8_round(v[0], inv), int8_round(v[1], inv), int8_round(v[2], inv), int8_round(v[3], inv));
    }
  }
  __syncwarp();
  if (lane == 0) *scale = sc;
  }
}

template <typename T>
__global__ void __launch_bounds__(kI8Warps * 32) fetch_int8_kernel(const Int8RowsArgs a) {
  pdl_trigger();
  pdl_wait();
  const int lane = threadIdx.x & 31;
  const int64_t wid = static_cast<int64_t>(blockIdx.x) * kI8Warps + (threadIdx.x >> 5);
  const int per_half = (a.n_kv_heads + a.heads_per_warp - 1) / a.heads_per_warp, per_unit = 2 * per_half;
  const int64_t u = wid / per_unit;
  const int rem = static_cast<int>(wid - u * per_unit);
  const bool isv = rem >= per_half;
  const int h0 = (isv ? rem - per_half : rem) * a.heads_per_warp, h1 = min(a.n_kv_heads, h0 + a.heads_per_warp);
  const int bs = a.block_size, D = a.head_dim;
  if (u >= a.n_units) return;
  Unit w;
  if (!find_unit(a.start_loc, a.context_lens, a.n_seqs, a.n_rows, bs, u, w)) {
    if (w.j == 0 && rem == 0 && lane == 0 &&
        (w.row0 < 0 || w.n < 0 || w.row0 + static_cast<int64_t>(w.n) > a.n_rows))
      raise_flag(a.err, PKV_FLAG_BAD_QUERY_LAYOUT);
    return;
  }
  if (w.ctx == 0) {  // an unserved sequence: zero rows, bs of them a unit
    T* dst = static_cast<T*>(const_cast<void*>(isv ? a.v : a.k));
    const int r1 = static_cast<int>(min(static_cast<int64_t>(w.n), (w.j + static_cast<int64_t>(1)) * bs));
    for (int64_t r = static_cast<int64_t>(w.j) * bs; r < r1; ++r)
      for (int e = h0 * D + lane; e < h1 * D; e += 32) dst[(w.row0 + r) * (isv ? a.v_stride : a.k_stride) + e] = Elem<T>::from_f(0.f);
    return;
  }
  const int from = w.ctx - w.n;  // first position fetched
  if (from < 0) {
    if (w.j == 0 && rem == 0 && lane == 0) raise_flag(a.err, PKV_FLAG_BAD_QUERY_LAYOUT);
    return;
  }
  const int jb = from / bs + w.j;
  const int64_t blk0 = static_cast<int64_t>(jb) * bs;
  if (blk0 >= w.ctx) return;
  if (jb >= a.max_blocks) {
    if (rem == 0 && lane == 0) raise_flag(a.err, PKV_FLAG_CONTEXT_EXCEEDS_TABLE);
    return;
  }
  const int id = a.block_tables[static_cast<int64_t>(w.s) * a.bt_stride + jb];
  if (id < 0 || id >= a.num_blocks) {
    if (rem == 0 && lane == 0) raise_flag(a.err, PKV_FLAG_BLOCK_OUT_OF_RANGE);
    return;
  }
  const int r0 = max(0, from - static_cast<int>(blk0));
  const int r1 = min(bs, static_cast<int>(w.ctx - blk0));
  const int64_t out0 = w.row0 + (blk0 + r0 - from);
  const int64_t stride = isv ? a.v_stride : a.k_stride;
  const bool vec = isv ? a.v_vec : a.k_vec;
  const int64_t pitch = static_cast<int64_t>(a.n_kv_heads) * D;
  for (int h = h0; h < h1; ++h) {
    T* dst = static_cast<T*>(const_cast<void*>(isv ? a.v : a.k)) + out0 * stride + static_cast<int64_t>(h) * D;
    const int8_t* src = static_cast<const int8_t*>(isv ? a.v_pool : a.k_pool) +
                        (static_cast<int64_t>(id) * bs * a.n_kv_heads + h) * D + r0 * pitch;
    const float sc = (isv ? a.v_scale : a.k_scale)[static_cast<int64_t>(id) * a.n_kv_heads + h];
    if (isv ? a.v_vec16 : a.k_vec16) {
      // a 16-byte store a lane, so that a store of the warp fills whole sectors
      // (two a lane, 32 bytes apart, wrote every sector twice); eight loads ahead
      constexpr int kPer = 16 / sizeof(T);
      const int row_log = (D == 64 ? 6 : 7) - (sizeof(T) == 2 ? 3 : 2), total = (r1 - r0) << row_log;
      const int row = lane >> row_log, col = (lane & ((1 << row_log) - 1)) * kPer;
      const int8_t* from = src + row * pitch + col;
      T* to = dst + row * stride + col;
      const int64_t from_step = (32 >> row_log) * pitch, to_step = (32 >> row_log) * stride;
      for (int c0 = lane; c0 < total; c0 += 256) {
        uint2 w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k, from += from_step)
          if (c0 + 32 * k < total) {
            if constexpr (sizeof(T) == 2) w[k] = *reinterpret_cast<const uint2*>(from);
            else w[k].x = *reinterpret_cast<const uint32_t*>(from);
          }
#pragma unroll
        for (int k = 0; k < 8; ++k, to += to_step) {
          if (c0 + 32 * k >= total) continue;
          float v[8];
          bytes_to_f(w[k].x, v);
          if constexpr (sizeof(T) == 2) {
            bytes_to_f(w[k].y, v + 4);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] *= sc;
            *reinterpret_cast<uint4*>(to) =
                make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
          } else {
            *reinterpret_cast<float4*>(to) = make_float4(v[0] * sc, v[1] * sc, v[2] * sc, v[3] * sc);
          }
        }
      }
      continue;
    }
    const int cpr = D / 4, total = (r1 - r0) * cpr;
    for (int c = lane; c < total; c += 32) {
      const int r = c / cpr, d = (c - r * cpr) * 4;
      float v[4];
      bytes_to_f(*reinterpret_cast<const uint32_t*>(src + r * pitch + d), v);
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] *= sc;
      store4_any<T>(dst + r * stride + d, vec, v);
    }
  }
}

// The visible rows of sequence blockIdx.y as values, all heads, K and V, row j
// into row s * cap + j of k_out / v_out [n_seqs * cap][n_kv_heads][D], so that a
// sequence's keys are consecutive rows.  Rows past its last key are zeros up to
// the next multiple of 128 (the attention kernel's key tile): a tile holds no
// stale bytes.  All rows of a sequence that is not served are zeros, and so is what the
// attention makes of them.  A warp takes up to kLayLoads stores a lane of a 16-row group's K or V at
// a time, all its loads ahead of them.
// Also clears the counters of the attention behind it.  Bound by the bytes for
// long ones (64-bit divisions for every unit and a head index by division for
// every load had made 32 sequences of 4,064 keys, 8 x 128, 109 us slower), by four
// dependent round trips for short ones.
constexpr int kLayThreads = 256, kLayLoads = 8;
template <typename T>
__global__ void __launch_bounds__(kLayThreads) lay_out_int8_kernel(const Int8LayArgs a) {
  pdl_trigger();
  pdl_wait();  // the append before it writes the pools; an earlier layer may still read the scratch
  const int s = blockIdx.y, bs = a.block_size, lane = threadIdx.x & 31;
  for (int64_t i = (static_cast<int64_t>(blockIdx.y) * gridDim.x + blockIdx.x) * kLayThreads + threadIdx.x; i < a.n_zero;
       i += static_cast<int64_t>(gridDim.x) * gridDim.y * kLayThreads)
    a.zero[i] = 0;
  const int new_rows = a.query_start_loc[s + 1] - a.query_start_loc[s];
  const bool served = a.context_lens == nullptr || a.context_lens[s] > 0;
  int64_t keys = static_cast<int64_t>(max(a.num_prior[s], 0)) + max(new_rows, 0);
  if (keys > static_cast<int64_t>(a.max_blocks) * bs) {
    if (blockIdx.x == 0 && threadIdx.x == 0) raise_flag(a.err, PKV_FLAG_CONTEXT_EXCEEDS_TABLE);
    keys = static_cast<int64_t>(a.max_blocks) * bs;
  }
  constexpr int kPer = 16 / sizeof(T);               // elements of a 16-byte store
  const int pitch = a.n_kv_heads * a.head_dim;       // elements of a row
  const int chunks = 16 * pitch / kPer;              // stores of a group, K or V
  const unsigned parts = (chunks + 32 * kLayLoads - 1) / (32 * kLayLoads);  // warps of a group, K or V
  // 16-row groups x K, V x parts, of 4 KB each: 2^31 of them would be 8 TB
  const unsigned n_work = static_cast<unsigned>((keys + 127) / 128) * 16 * parts;
  const int per_head = (a.head_dim == 64 ? 64 : 128) / kPer;               // stores of a row of a head
  const int head_step = 32 / per_head % a.n_kv_heads;                      // heads that 32 stores go on by
  for (unsigned w = blockIdx.x * (kLayThreads / 32) + (threadIdx.x >> 5); w < n_work; w += gridDim.x * (kLayThreads / 32)) {
    const unsigned wp = parts == 1 ? w : w / parts;
    const int part = static_cast<int>(w - wp * parts);
    const bool isv = wp & 1;
    const int row0 = static_cast<int>(wp >> 1) * 16;
    int id = -1;
    if (row0 < keys && served) {
      id = a.block_tables[static_cast<int64_t>(s) * a.bt_stride + row0 / bs];
      if (id < 0 || id >= a.num_blocks) {
        if (lane == 0) raise_flag(a.err, PKV_FLAG_BLOCK_OUT_OF_RANGE);
        id = -1;
      }
    }
    const int left = id < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(16), keys - row0));
    const int valid = left * (pitch / kPer);  // stores of rows that are keys
    // 16 rows x pitch are consecutive on both sides
    const int8_t* src = static_cast<const int8_t*>(isv ? a.v_pool : a.k_pool) +
                        (static_cast<int64_t>(id < 0 ? 0 : id) * bs + row0 % bs) * pitch;
    T* dst = static_cast<T*>(isv ? a.v_out : a.k_out) + (static_cast<int64_t>(s) * a.cap + row0) * pitch;
    const float* scale = (isv ? a.v_scale : a.k_scale) + static_cast<int64_t>(id < 0 ? 0 : id) * a.n_kv_heads;
    int head = (part * kLayLoads * 32 + lane) / per_head % a.n_kv_heads;
    uint2 u[kLayLoads];
    float sc[kLayLoads];
#pragma unroll
    for (int k = 0; k < kLayLoads; ++k) {
      const int c = (part * kLayLoads + k) * 32 + lane;
      u[k] = make_uint2(0u, 0u);
      sc[k] = 0.f;
      if (c < valid) {
        if constexpr (sizeof(T) == 2) u[k] = *reinterpret_cast<const uint2*>(src + static_cast<int64_t>(c) * kPer);
        else u[k].x = *reinterpret_cast<const uint32_t*>(src + static_cast<int64_t>(c) * kPer);
        sc[k] = scale[head];
      }
      head += head_step;
      if (head >= a.n_kv_heads) head -= a.n_kv_heads;
    }
#pragma unroll
    for (int k = 0; k < kLayLoads; ++k) {
      const int c = (part * kLayLoads + k) * 32 + lane;
      if (c >= chunks) continue;
      float v[8];
      bytes_to_f(u[k].x, v);
      T* to = dst + static_cast<int64_t>(c) * kPer;
      if constexpr (sizeof(T) == 4) {
        *reinterpret_cast<float4*>(to) = make_float4(v[0] * sc[k], v[1] * sc[k], v[2] * sc[k], v[3] * sc[k]);
      } else {
        bytes_to_f(u[k].y, v + 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] *= sc[k];
        *reinterpret_cast<uint4*>(to) =
            make_uint4(pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3]), pack2<T>(v[4], v[5]), pack2<T>(v[6], v[7]));
      }
    }
  }
}

template <typename K>
cudaError_t launch_rows(K f16, K bf16, K f32, Int8RowsArgs a, cudaStream_t stream) {
  // one head a warp while that leaves the SMs' warp slots short, up to four beyond
  // (append of 64 prompts of 1,000 tokens, 8 x 128: 83.1 us with one, 68.4 with
  // four; of 256 single tokens, 2 x 64: 3.9 and 4.8)
  const int64_t each = a.n_units * 2 * a.n_kv_heads;
  a.heads_per_warp = each < 32768 ? 1 : each < 65536 ? 2 : 4;
  if (a.heads_per_warp > a.n_kv_heads) a.heads_per_warp = a.n_kv_heads;
  const int64_t warps = a.n_units * 2 * ((a.n_kv_heads + a.heads_per_warp - 1) / a.heads_per_warp);
  const int64_t grid = (warps + kI8Warps - 1) / kI8Warps;
  if (grid == 0) return cudaSuccess;
  if (grid > 0x7fffffff) return cudaErrorInvalidConfiguration;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(kI8Warps * 32);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  K kern = a.dtype == PKV_DTYPE_F16 ? f16 : a.dtype == PKV_DTYPE_BF16 ? bf16 : f32;
  return cudaLaunchKernelEx(&cfg, kern, a);
}

// may `bytes` of these rows, from a multiple of that, be one access?
bool rows_vec(const void* p, int64_t stride, int esize, int bytes) {
  return ((reinterpret_cast<uintptr_t>(p) | static_cast<uintptr_t>(stride * esize)) & (bytes - 1)) == 0;
}

void fill_rows(Int8RowsArgs& a) {
  const int es = a.dtype == PKV_DTYPE_F32 ? 4 : 2;
  a.k_vec = rows_vec(a.k, a.k_stride, es, 4 * es);
  a.v_vec = rows_vec(a.v, a.v_stride, es, 4 * es);
  a.k_vec16 = rows_vec(a.k, a.k_stride, es, 16);
  a.v_vec16 = rows_vec(a.v, a.v_stride, es, 16);
  a.n_units = a.n_rows / a.block_size + 2 * static_cast<int64_t>(a.n_seqs);
}

}  // namespace

cudaError_t launch_append_int8(Int8RowsArgs a, cudaStream_t stream) {
  fill_rows(a);
  return launch_rows(append_int8_kernel<__half>, append_int8_kernel<__nv_bfloat16>,
                     append_int8_kernel<float>, a, stream);
}

cudaError_t launch_fetch_int8(Int8RowsArgs a, cudaStream_t stream) {
  fill_rows(a);
  return launch_rows(fetch_int8_kernel<__half>, fetch_int8_kernel<__nv_bfloat16>,
                     fetch_int8_kernel<float>, a, stream);
}

cudaError_t launch_lay_out_int8(const Int8LayArgs& a, int dtype, cudaStream_t stream) {
  cudaLaunchConfig_t cfg = {};
  // a warp for every unit of work of the longest possible sequence, up to what
  // fills the GPU; the kernel's loop takes the rest
  const int kv_bytes = 16 * a.n_kv_heads * a.head_dim * (dtype == PKV_DTYPE_F32 ? 4 : 2);
  const int64_t parts = (kv_bytes + 512 * kLayLoads - 1) / (512 * kLayLoads);
  const int64_t want = (static_cast<int64_t>(a.cap) / 16 * 2 * parts + kLayThreads / 32 - 1) / (kLayThreads / 32);
  const int64_t most = (2048 + a.n_seqs - 1) / a.n_seqs;
  cfg.gridDim = dim3(static_cast<unsigned>(want < most ? want : most), a.n_seqs);
  cfg.blockDim = dim3(kLayThreads);
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  if (dtype == PKV_DTYPE_F16) return cudaLaunchKernelEx(&cfg, lay_out_int8_kernel<__half>, a);
  if (dtype == PKV_DTYPE_BF16) return cudaLaunchKernelEx(&cfg, lay_out_int8_kernel<__nv_bfloat16>, a);
  return cudaLaunchKernelEx(&cfg, lay_out_int8_kernel<float>, a);
}

}  // namespace pkv
