// pkv_step_tables.cu -- block tables, slot map, positions and lengths of a step,
// built on the GPU from the request lengths.
//
// The reference builds them on the host, one sequence at a time
// (mini_engine/scheduler.py:79-156 grows the tables, mini_engine/paged/
// block_manager.py:121-131 derives the slots), and so does
// PagedKVCache.step_arrays.  Here request i with p_i cached and n_i new tokens
// gets, over blocks of b tokens,
//
//   have_i = ceil(p_i / b),  need_i = ceil((p_i + n_i) / b) - have_i,
//   off_i  = need_0 + .. + need_{i-1},   served_i = off_i + need_i <= F,
//   table[i][have_i + j] = free[F - 1 - (off_i + j)]        (LIFO, request order)
//   pos(t) = p_i + (t - start_i),  slot(t) = table[i][pos / b] * b + pos % b.
//
// A new block begins with one of the step's own tokens (its first slot is
// position have_i * b >= p_i), so the thread that computes that token's slot
// also writes the table entry, and no thread waits for another's entry.
//
// One launch.  Every CTA scans the lengths itself (two loads and a shared-memory
// scan of (tokens, blocks) pairs, so no CTA waits for another), then takes its
// share of the requests and of the tokens, four consecutive tokens to a thread:
// one binary search, then 16-byte stores.  The free count is read by all CTAs
// and the new count goes to another word, so no CTA can see it change.
//
// What bounds it: the launch and three dependent round trips (lengths, the free
// list or table entry, the store) for decode steps; the 16 bytes a token of
// slots and positions for prompts (280,000 tokens: 4.5 MB).  256 decode requests
// take 6.1 us in a graph; a call from Python takes 20, most of it on the host.
#include <atomic>

#include "pkv_common.cuh"
#include "pkv_internal.h"

namespace pkv {

namespace {

constexpr int kStThreads = 512;
constexpr int kStTok = 4;  // consecutive tokens per thread
constexpr unsigned kStSat = 0x7fffffffu;

// sums of lengths saturate: a batch whose lengths add up past 2^31 - 1 is
// refused as a whole, not wrapped around
__device__ __forceinline__ unsigned sat_add(unsigned a, unsigned b) { return min(a + b, kStSat); }

__global__ void __launch_bounds__(kStThreads) step_tables_kernel(const StepTablesArgs a) {
  extern __shared__ unsigned st_smem[];
  const int B = a.n_seqs, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned* start = st_smem;         // [B + 1] first token of each request
  unsigned* first = start + B + 1;   // [B + 1] first new block of each request
  int* prior = reinterpret_cast<int*>(first + B + 1);  // [B] cached tokens, -1: lengths not valid
  __shared__ unsigned wsum[2][kStThreads / 32];
  __shared__ unsigned s_taken;
  const int64_t room = static_cast<int64_t>(a.max_blocks) * a.block_size;
  const int bs = a.block_size;
  int n_free = *a.n_free;
  if (n_free < 0 || n_free > a.free_capacity) {
    if (blockIdx.x == 0 && tid == 0) raise_flag(a.err, PKV_FLAG_BLOCK_OUT_OF_RANGE);
    n_free = n_free < 0 ? 0 : a.free_capacity;
  }
  auto blocks_of = [&](int n) { return static_cast<unsigned>((static_cast<int64_t>(n) + bs - 1) / bs); };

  // lengths once from memory: the tokens (start) and new blocks (first) of each
  // request, none if its lengths are not valid, then their prefixes
  const int per = (B + kStThreads - 1) / kStThreads;
  const int lo = min(B, tid * per), hi = min(B, lo + per);
  unsigned tn = 0, tb = 0;
  for (int i = lo; i < hi; ++i) {
    const int p = __ldg(a.num_prior + i), n = __ldg(a.num_new + i);
    const bool ok = p >= 0 && n >= 0 && static_cast<int64_t>(p) + n <= room;
    const unsigned blocks = ok ? blocks_of(p + n) - blocks_of(p) : 0u;
    prior[i] = ok ? p : -1;
    start[i] = ok ? n : 0;
    first[i] = blocks;
    tn = sat_add(tn, start[i]);
    tb = sat_add(tb, blocks);
  }
  unsigned xn = tn, xb = tb;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const unsigned yn = __shfl_up_sync(0xffffffffu, xn, o), yb = __shfl_up_sync(0xffffffffu, xb, o);
    if (lane >= o) { xn = sat_add(xn, yn); xb = sat_add(xb, yb); }
  }
  if (lane == 31) { wsum[0][warp] = xn; wsum[1][warp] = xb; }
  if (tid == 0) s_taken = 0;
  __syncthreads();
  unsigned bn = 0, bb = 0;
#pragma unroll
  for (int w = 0; w < kStThreads / 32; ++w)
    if (w < warp) { bn = sat_add(bn, wsum[0][w]); bb = sat_add(bb, wsum[1][w]); }
  // exclusive prefix of this thread's first request (the lane before it)
  const unsigned en = __shfl_up_sync(0xffffffffu, xn, 1), eb = __shfl_up_sync(0xffffffffu, xb, 1);
  unsigned rn = lane ? sat_add(bn, en) : bn, rb = lane ? sat_add(bb, eb) : bb;
  for (int i = lo; i < hi; ++i) {
    const unsigned n = start[i], blocks = first[i];
    start[i] = rn;
    first[i] = rb;
    rn = sat_add(rn, n);
    rb = sat_add(rb, blocks);
  }
  if (hi == B && lo < B) { start[B] = rn; first[B] = rb; }
  if (B == 0 && tid == 0) start[0] = first[0] = 0;
  __syncthreads();
  const unsigned total = start[B];
  // a request is served if its blocks and its tokens fit
  auto served = [&](int i) {
    return first[i + 1] <= static_cast<unsigned>(n_free) &&
           start[i + 1] <= static_cast<unsigned>(a.n_tokens);
  };

  // ---- the requests' outputs, dealt over the grid
  for (int i = blockIdx.x * kStThreads + tid; i < B; i += gridDim.x * kStThreads) {
    const bool ok = prior[i] >= 0;
    const bool srv = ok && served(i);
    a.context_lens[i] = srv ? prior[i] + static_cast<int>(start[i + 1] - start[i]) : 0;
    a.query_start_loc[i] = static_cast<int>(start[i]);
    if (!ok) {
      const int rp = a.num_prior[i], rn2 = a.num_new[i];
      raise_flag(a.err, (rp < 0 || rn2 < 0) ? PKV_FLAG_BAD_QUERY_LAYOUT : PKV_FLAG_CONTEXT_EXCEEDS_TABLE);
    } else if (!srv) {
      raise_flag(a.err, start[i + 1] > static_cast<unsigned>(a.n_tokens) ? PKV_FLAG_BAD_QUERY_LAYOUT
                                                                         : PKV_FLAG_OUT_OF_BLOCKS);
    }
  }
  if (blockIdx.x == 0) {
    // blocks taken: the last served request's end
    unsigned t = 0;
    for (int i = lo; i < hi; ++i)
      if (served(i)) t = max(t, first[i + 1]);
    t = __reduce_max_sync(0xffffffffu, t);
    if (lane == 0) atomicMax(&s_taken, t);
    __syncthreads();
    if (tid == 0) {
      *a.n_free_out = n_free - static_cast<int>(s_taken);
      a.query_start_loc[B] = static_cast<int>(total);
    }
  }

  // ---- the tokens' slots and positions
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kStThreads * kStTok;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * kStThreads + tid) * kStTok; t0 < a.n_tokens;
       t0 += stride) {
    int64_t slot[kStTok], pos[kStTok];
    int s = 0;
    if (t0 < total) {  // last request with start <= t0
      int l = 0, h = B - 1;
      while (l < h) {
        const int m = (l + h + 1) >> 1;
        if (start[m] <= static_cast<unsigned>(t0)) l = m; else h = m - 1;
      }
      s = l;
    }
    int p = 0, have = 0, cur = -1, col = -1, blk = 0;
    bool srv = false;
#pragma unroll
    for (int k = 0; k < kStTok; ++k) {
      const int64_t t = t0 + k;
      slot[k] = -1;
      pos[k] = 0;
      if (t >= total || t >= a.n_tokens) continue;
      while (start[s + 1] <= static_cast<unsigned>(t)) ++s;  // empty requests are passed over
      if (s != cur) {
        cur = s;
        p = prior[s];
        have = static_cast<int>(blocks_of(p));
        srv = served(s);
        col = -1;
      }
      const int ps = p + static_cast<int>(t - start[s]);
      pos[k] = ps;
      if (!srv) continue;
      const int c = ps / bs, off = ps - c * bs;
      int32_t* entry = a.block_tables + static_cast<int64_t>(s) * a.bt_stride + c;
      if (c != col) {
        col = c;
        if (c >= have) {
          blk = __ldg(a.free_blocks + (n_free - 1 - static_cast<int>(first[s]) - (c - have)));
          if (off == 0) *entry = blk;  // this token opens the block
        } else {
          blk = *entry;
        }
      }
      slot[k] = static_cast<int64_t>(blk) * bs + off;
    }
    if (t0 + kStTok <= a.n_tokens && a.vec_ok) {
      longlong2* so = reinterpret_cast<longlong2*>(a.slot_mapping + t0);
      longlong2* po = reinterpret_cast<longlong2*>(a.positions + t0);
#pragma unroll
      for (int k = 0; k < kStTok; k += 2) {
        so[k / 2] = make_longlong2(slot[k], slot[k + 1]);
        po[k / 2] = make_longlong2(pos[k], pos[k + 1]);
      }
    } else {
#pragma unroll
      for (int k = 0; k < kStTok; ++k)
        if (t0 + k < a.n_tokens) {
          a.slot_mapping[t0 + k] = slot[k];
          a.positions[t0 + k] = pos[k];
        }
    }
  }
}

}  // namespace

cudaError_t launch_step_tables(StepTablesArgs a, cudaStream_t stream) {
  static std::atomic<int> sm_count[64];  // per device, 0: not asked
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return e;
  int sms = dev < 64 ? sm_count[dev].load() : 0;
  if (sms == 0) {
    e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev);
    if (e == cudaSuccess)
      e = cudaFuncSetAttribute(step_tables_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                               static_cast<int>((3 * kStepTablesMaxSeqs + 2) * sizeof(unsigned)));
    if (e != cudaSuccess) return e;
    if (dev < 64) sm_count[dev].store(sms);
  }
  const size_t smem = (3 * static_cast<size_t>(a.n_seqs) + 2) * sizeof(unsigned);
  a.vec_ok = ((reinterpret_cast<uintptr_t>(a.slot_mapping) | reinterpret_cast<uintptr_t>(a.positions)) & 15) == 0;
  const int64_t want = (static_cast<int64_t>(a.n_tokens) + kStThreads * kStTok - 1) / (kStThreads * kStTok);
  const int grid = static_cast<int>(want < 1 ? 1 : want > sms ? sms : want);
  step_tables_kernel<<<grid, kStThreads, smem, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace pkv
