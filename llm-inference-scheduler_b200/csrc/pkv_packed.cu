// pkv_packed.cu -- causal attention with grouped heads over consecutive rows:
// whole prompts packed one behind the other, or chunks behind cached keys that
// were laid out row by row.
#include <float.h>

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

// One (query row, head) by a whole warp, keys 0 .. lim - 1 only: the row's own
// arithmetic, untouched by any key it must not see.  The tiled kernels multiply
// masked keys by a probability of zero, which is not zero where such a key's V
// holds an infinity or NaN; a row that comes out not finite is computed again
// here (and stays so if its own keys make it so).
template <typename T, int D>
__device__ __noinline__ void packed_row_alone(const PackedArgs& a, int64_t row, int h, int64_t key0, int lim) {
  const int lane = threadIdx.x & 31, g = h / (a.n_q_heads / a.n_kv_heads);
  constexpr int kPer = D / 32;
  const T* q = static_cast<const T*>(a.q) + row * a.q_stride + static_cast<int64_t>(h) * D;
  float qv[kPer], acc[kPer];
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    qv[i] = Elem<T>::to_f(q[lane + 32 * i]);
    acc[i] = 0.f;
  }
  float m = -FLT_MAX, l = 0.f;
  for (int j = 0; j < lim; ++j) {
    const T* k = static_cast<const T*>(a.k) + (key0 + j) * a.k_stride + static_cast<int64_t>(g) * D;
    const T* v = static_cast<const T*>(a.v) + (key0 + j) * a.v_stride + static_cast<int64_t>(g) * D;
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < kPer; ++i) s = fmaf(qv[i], Elem<T>::to_f(k[lane + 32 * i]), s);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    s *= a.scale;
    const float mn = fmaxf(m, s), c = expf(m - mn), p = expf(s - mn);
    m = mn;
    l = l * c + p;
#pragma unroll
    for (int i = 0; i < kPer; ++i) acc[i] = acc[i] * c + p * Elem<T>::to_f(v[lane + 32 * i]);
  }
  T* out = static_cast<T*>(a.out) + row * a.out_stride + static_cast<int64_t>(h) * D;
#pragma unroll
  for (int i = 0; i < kPer; ++i) out[lane + 32 * i] = Elem<T>::from_f(acc[i] / l);
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

template <typename T, int D>
__global__ void __launch_bounds__(kPkThreads) packed_cores_kernel(const PackedArgs a) {
  extern __shared__ float pk_smem[];
  constexpr int kLd = D + 4;                // row pitch of the Q, K and V tiles (16-byte rows, spread banks)
  float* qs = pk_smem;                      // [64][kLd]
  float* ks = qs + kPkM * kLd;              // [64][kLd]
  float* vs = ks + kPkN * kLd;              // [64][kLd]
  float* ps = vs + kPkN * kLd;              // [64][68] probabilities
  constexpr int kLp = kPkN + 4;
  pdl_trigger();
  pdl_wait();
  const int tid = threadIdx.x, ty = tid >> 4, tx = tid & 15;
  const int h = blockIdx.y, g = h / (a.n_q_heads / a.n_kv_heads);
  int s, tile;
  // the last tiles (the longest of a sequence) first
  if (!find_tile(a, static_cast<int64_t>(gridDim.x) - 1 - blockIdx.x, kPkM, s, tile)) return;
  const int q_begin = a.query_start_loc[s], n_new = a.query_start_loc[s + 1] - q_begin;
  const KeySpan span = key_span(a, s, q_begin, n_new);
  const int q0 = tile * kPkM, rows = min(kPkM, n_new - q0);
  const int last = min(span.prior + q0 + rows, span.keys);  // keys any row of the tile sees

  auto load_tile = [&](float* dst, const T* src, int64_t stride, int n) {
    for (int c = tid; c < 64 * (D / 4); c += kPkThreads) {
      const int r = c / (D / 4), d = (c - r * (D / 4)) * 4;
      float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
      if (r < n) {
        const T* p = src + r * stride + d;
        f = make_float4(Elem<T>::to_f(p[0]), Elem<T>::to_f(p[1]), Elem<T>::to_f(p[2]), Elem<T>::to_f(p[3]));
      }
      *reinterpret_cast<float4*>(dst + r * kLd + d) = f;
    }
  };
  load_tile(qs, static_cast<const T*>(a.q) + static_cast<int64_t>(q_begin + q0) * a.q_stride +
                    static_cast<int64_t>(h) * D, a.q_stride, rows);
  // this thread: rows 4 ty .. 4 ty + 3; keys tx + 16 c; dims tx + 16 c
  constexpr int kDim = D / 16;
  float o[4][kDim], m[4], l[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    m[r] = -INFINITY;
    l[r] = 0.f;
#pragma unroll
    for (int c = 0; c < kDim; ++c) o[r][c] = 0.f;
  }
  const float sl2 = a.scale * 1.4426950408889634f;
  for (int k0 = 0; k0 < last; k0 += kPkN) {
    __syncthreads();
    const int n = min(kPkN, last - k0);
    load_tile(ks, static_cast<const T*>(a.k) + (span.row0 + k0) * a.k_stride + static_cast<int64_t>(g) * D,
              a.k_stride, n);
    load_tile(vs, static_cast<const T*>(a.v) + (span.row0 + k0) * a.v_stride + static_cast<int64_t>(g) * D,
              a.v_stride, n);
    __syncthreads();
    float x[4][4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int c = 0; c < 4; ++c) x[r][c] = 0.f;
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
          x[r][c] = fmaf(qa[r].x, kb[c].x, x[r][c]);
          x[r][c] = fmaf(qa[r].y, kb[c].y, x[r][c]);
          x[r][c] = fmaf(qa[r].z, kb[c].z, x[r][c]);
          x[r][c] = fmaf(qa[r].w, kb[c].w, x[r][c]);
        }
    }
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int lim = span.prior + q0 + 4 * ty + r + 1 - k0;  // keys of this tile the row sees
      float mx = -INFINITY;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        x[r][c] = tx + 16 * c < min(lim, n) ? x[r][c] * sl2 : -INFINITY;
        mx = fmaxf(mx, x[r][c]);
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, w));
      const float mn = fmaxf(m[r], mx);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float f = exp2f(m[r] - base);
      float sum = 0.f;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const float p = exp2f(x[r][c] - base);
        sum += p;
        ps[(4 * ty + r) * kLp + tx + 16 * c] = p;
      }
#pragma unroll
      for (int w = 8; w > 0; w >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, w);
      m[r] = mn;
      l[r] = l[r] * f + sum;
#pragma unroll
      for (int c = 0; c < kDim; ++c) o[r][c] *= f;
    }
    __syncwarp();  // a warp's two row groups write and read only their own rows of ps
#pragma unroll 4
    for (int j = 0; j < kPkN; ++j) {
      float pv[4];
#pragma unroll
      for (int r = 0; r < 4; ++r) pv[r] = ps[(4 * ty + r) * kLp + j];
#pragma unroll
      for (int c = 0; c < kDim; ++c) {
        const float v = vs[j * kLd + tx + 16 * c];
#pragma unroll
        for (int r = 0; r < 4; ++r) o[r][c] = fmaf(pv[r], v, o[r][c]);
      }
    }
  }
  bool fine[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int row = 4 * ty + r;
    const float inv = 1.f / l[r];
    bool ok = true;
    T* out = static_cast<T*>(a.out) + static_cast<int64_t>(q_begin + q0 + row) * a.out_stride +
             static_cast<int64_t>(h) * D;
#pragma unroll
    for (int c = 0; c < kDim; ++c) {
      ok = ok && fabsf(o[r][c] * inv) < INFINITY;
      if (row < rows) out[tx + 16 * c] = Elem<T>::from_f(o[r][c] * inv);
    }
    fine[r] = ok || row >= rows;
  }
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const unsigned bad = __ballot_sync(0xffffffffu, !fine[r]);
#pragma unroll
    for (int half = 0; half < 2; ++half)
      if (bad & (0xffffu << (16 * half))) {  // warp-uniform: row 4 ty + r of this half-warp
        const int row = 4 * ((tid >> 5) * 2 + half) + r;
        __syncwarp();
        packed_row_alone<T, D>(a, static_cast<int64_t>(q_begin) + q0 + row, h, span.row0,
                               min(span.prior + q0 + row + 1, span.keys));
      }
  }
}

template <typename T, int D>
cudaError_t launch_cores(const PackedArgs& a, cudaStream_t stream) {
  constexpr int smem = (3 * 64 * (D + 4) + 64 * 68) * 4;
  cudaError_t e = cudaFuncSetAttribute(packed_cores_kernel<T, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return e;
  const int64_t tiles = a.n_tokens / kPkM + static_cast<int64_t>(a.n_seqs);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(tiles), a.n_q_heads);
  cfg.blockDim = dim3(kPkThreads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, packed_cores_kernel<T, D>, a);
}

}  // namespace

cudaError_t launch_packed_attention(const PackedArgs& a, cudaStream_t stream) {
  if (a.n_tokens == 0 || a.n_seqs == 0) return cudaSuccess;
  auto go = [&](auto tag) {
    using T = decltype(tag);
    return a.head_dim == 64 ? launch_cores<T, 64>(a, stream) : launch_cores<T, 128>(a, stream);
  };
  if (a.dtype == PKV_DTYPE_F16) return go(__half{});
  if (a.dtype == PKV_DTYPE_BF16) return go(__nv_bfloat16{});
  return go(float{});
}

}  // namespace pkv
