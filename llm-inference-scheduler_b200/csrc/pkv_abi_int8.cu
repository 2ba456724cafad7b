// pkv_abi_int8.cu -- extern "C" entry points of the step tables, the int8 pools
// and the packed-prompt attention (include/pagedkv.h): host checks, then one
// launcher each.  Nothing here allocates or synchronises.
#include "pkv_common.cuh"
#include "pkv_internal.h"

using namespace pkv;

namespace {

inline bool known_dtype(int dt) { return dt == PKV_DTYPE_F32 || dt == PKV_DTYPE_F16 || dt == PKV_DTYPE_BF16; }
inline int size_of(int dt) { return dt == PKV_DTYPE_F32 ? 4 : 2; }
inline int status(cudaError_t e) { return e == cudaSuccess ? PKV_OK : static_cast<int>(e); }
inline bool aligned(const void* p, uintptr_t m) { return (reinterpret_cast<uintptr_t>(p) & (m - 1)) == 0; }

// pools, scales and tables that every int8 entry takes
int check_int8(const void* k_pool, const void* v_pool, const float* k_scale, const float* v_scale,
               int num_blocks, const int32_t* tables, int64_t bt_stride, int max_blocks,
               int n_kv_heads, int head_dim, int block_size, int dtype) {
  if (!k_pool || !v_pool || !k_scale || !v_scale || !tables) return PKV_ERR_NULL_POINTER;
  if (!known_dtype(dtype)) return PKV_ERR_BAD_DTYPE;
  if (num_blocks <= 0 || max_blocks <= 0 || n_kv_heads <= 0 || bt_stride < max_blocks) return PKV_ERR_BAD_SHAPE;
  if (head_dim <= 0 || block_size <= 0) return PKV_ERR_BAD_SHAPE;
  if (static_cast<int64_t>(num_blocks) * block_size > 0x7fffffff ||
      static_cast<int64_t>(max_blocks) * block_size > 0x7fffffff)
    return PKV_ERR_BAD_SHAPE;
  if ((head_dim != 64 && head_dim != 128) || block_size % 16 != 0) return PKV_ERR_UNSUPPORTED;
  if (!aligned(k_pool, 16) || !aligned(v_pool, 16)) return PKV_ERR_MISALIGNED;
  return PKV_OK;
}

}  // namespace

extern "C" {

int pkv_build_step_tables(int32_t* block_tables, int64_t block_table_stride, int max_blocks_per_seq,
                          const int32_t* free_blocks, int n_free_blocks, const int32_t* n_free,
                          int32_t* n_free_out, const int32_t* num_prior, const int32_t* num_new,
                          int n_seqs, int block_size, int32_t* context_lens,
                          int32_t* query_start_loc, int64_t* slot_mapping, int64_t* positions,
                          int n_tokens, int* err_flags, pkv_stream_t stream) {
  if (n_seqs < 0 || n_tokens < 0 || n_free_blocks < 0 || block_size <= 0) return PKV_ERR_BAD_SHAPE;
  if (!n_free || !n_free_out || !query_start_loc) return PKV_ERR_NULL_POINTER;
  if (n_seqs > 0) {
    if (!block_tables || !num_prior || !num_new || !context_lens) return PKV_ERR_NULL_POINTER;
    if (max_blocks_per_seq <= 0 || block_table_stride < max_blocks_per_seq ||
        static_cast<int64_t>(max_blocks_per_seq) * block_size > 0x7fffffff)
      return PKV_ERR_BAD_SHAPE;
    if (n_seqs > kStepTablesMaxSeqs) return PKV_ERR_UNSUPPORTED;
  }
  if (n_free_blocks > 0 && !free_blocks) return PKV_ERR_NULL_POINTER;
  if (n_tokens > 0 && (!slot_mapping || !positions)) return PKV_ERR_NULL_POINTER;
  // every CTA reads the inputs while others write: no output may lie over an input
  const struct { const void* p; size_t bytes; } ins[] = {
      {n_free, 4}, {num_prior, 4 * static_cast<size_t>(n_seqs)}, {num_new, 4 * static_cast<size_t>(n_seqs)},
      {free_blocks, 4 * static_cast<size_t>(n_free_blocks)}}, outs[] = {
      {n_free_out, 4}, {context_lens, 4 * static_cast<size_t>(n_seqs)}, {query_start_loc, 4 * (static_cast<size_t>(n_seqs) + 1)},
      {slot_mapping, 8 * static_cast<size_t>(n_tokens)}, {positions, 8 * static_cast<size_t>(n_tokens)}};
  for (const auto& o : outs)
    for (const auto& i : ins) {
      const uintptr_t x = reinterpret_cast<uintptr_t>(o.p), y = reinterpret_cast<uintptr_t>(i.p);
      if (x < y + i.bytes && y < x + o.bytes) return PKV_ERR_UNSUPPORTED;
    }
  StepTablesArgs a{};
  a.block_tables = block_tables;
  a.bt_stride = block_table_stride;
  a.max_blocks = max_blocks_per_seq;
  a.free_blocks = free_blocks;
  a.free_capacity = n_free_blocks;
  a.n_free = n_free;
  a.n_free_out = n_free_out;
  a.num_prior = num_prior;
  a.num_new = num_new;
  a.n_seqs = n_seqs;
  a.block_size = block_size;
  a.context_lens = context_lens;
  a.query_start_loc = query_start_loc;
  a.slot_mapping = slot_mapping;
  a.positions = positions;
  a.n_tokens = n_tokens;
  a.err = err_flags;
  return status(launch_step_tables(a, static_cast<cudaStream_t>(stream)));
}

static int int8_rows(bool append, const void* k, int64_t k_stride, const void* v, int64_t v_stride,
                     void* k_pool, void* v_pool, float* k_scale, float* v_scale, int num_blocks,
                     const int32_t* tables, int64_t bt_stride, int max_blocks,
                     const int32_t* context_lens, const int32_t* start_loc, int n_seqs, int n_rows,
                     int n_kv_heads, int head_dim, int block_size, int dtype, int* err,
                     pkv_stream_t stream) {
  if (n_seqs < 0 || n_rows < 0) return PKV_ERR_BAD_SHAPE;
  if (n_seqs == 0 || n_rows == 0) return PKV_OK;
  int rc = check_int8(k_pool, v_pool, k_scale, v_scale, num_blocks, tables, bt_stride, max_blocks,
                      n_kv_heads, head_dim, block_size, dtype);
  if (rc != PKV_OK) return rc;
  if (!k || !v || !context_lens || !start_loc) return PKV_ERR_NULL_POINTER;
  const int64_t row = static_cast<int64_t>(n_kv_heads) * head_dim;
  if (k_stride < row || v_stride < row) return PKV_ERR_BAD_SHAPE;
  if (!aligned(k, size_of(dtype)) || !aligned(v, size_of(dtype))) return PKV_ERR_MISALIGNED;
  Int8RowsArgs a{};
  a.k = k;
  a.v = v;
  a.k_stride = k_stride;
  a.v_stride = v_stride;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  a.block_tables = tables;
  a.bt_stride = bt_stride;
  a.max_blocks = max_blocks;
  a.context_lens = context_lens;
  a.start_loc = start_loc;
  a.n_seqs = n_seqs;
  a.n_rows = n_rows;
  a.num_blocks = num_blocks;
  a.block_size = block_size;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.dtype = dtype;
  a.err = err;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  return status(append ? launch_append_int8(a, st) : launch_fetch_int8(a, st));
}

int pkv_reshape_and_cache_int8(const void* k, const void* v, int64_t k_row_stride,
                               int64_t v_row_stride, void* k_pool, void* v_pool, float* k_scale,
                               float* v_scale, int num_blocks, const int32_t* block_tables,
                               int64_t block_table_stride, int max_blocks_per_seq,
                               const int32_t* context_lens, const int32_t* query_start_loc,
                               int n_seqs, int n_tokens, int n_kv_heads, int head_dim,
                               int block_size, int dtype, int* err_flags, pkv_stream_t stream) {
  return int8_rows(true, k, k_row_stride, v, v_row_stride, k_pool, v_pool, k_scale, v_scale,
                   num_blocks, block_tables, block_table_stride, max_blocks_per_seq, context_lens,
                   query_start_loc, n_seqs, n_tokens, n_kv_heads, head_dim, block_size, dtype,
                   err_flags, stream);
}

int pkv_fetch_int8(void* k_out, void* v_out, int64_t k_row_stride, int64_t v_row_stride,
                   const void* k_pool, const void* v_pool, const float* k_scale,
                   const float* v_scale, int num_blocks, const int32_t* block_tables,
                   int64_t block_table_stride, int max_blocks_per_seq,
                   const int32_t* context_lens, const int32_t* row_start_loc, int n_seqs,
                   int n_rows, int n_kv_heads, int head_dim, int block_size, int dtype,
                   int* err_flags, pkv_stream_t stream) {
  return int8_rows(false, k_out, k_row_stride, v_out, v_row_stride, const_cast<void*>(k_pool),
                   const_cast<void*>(v_pool), const_cast<float*>(k_scale),
                   const_cast<float*>(v_scale), num_blocks, block_tables, block_table_stride,
                   max_blocks_per_seq, context_lens, row_start_loc, n_seqs, n_rows, n_kv_heads,
                   head_dim, block_size, dtype, err_flags, stream);
}

size_t pkv_decode_int8_workspace_bytes(int n_q_heads, int head_dim) {
  if (n_q_heads <= 0 || head_dim <= 0) return 0;
  return decode_int8_workspace_bytes(n_q_heads, head_dim);
}

int pkv_paged_decode_attention_int8(void* out, int64_t out_row_stride, const void* q,
                                    int64_t q_row_stride, const void* k_pool, const void* v_pool,
                                    const float* k_scale, const float* v_scale, int num_blocks,
                                    const int32_t* block_tables, int64_t block_table_stride,
                                    int max_blocks_per_seq, const int32_t* context_lens,
                                    int n_seqs, int n_q_heads, int n_kv_heads, int head_dim,
                                    int block_size, float scale, int dtype, void* workspace,
                                    size_t workspace_bytes, int* err_flags, pkv_stream_t stream) {
  if (n_seqs < 0) return PKV_ERR_BAD_SHAPE;
  if (n_seqs == 0) return PKV_OK;
  int rc = check_int8(k_pool, v_pool, k_scale, v_scale, num_blocks, block_tables, block_table_stride,
                      max_blocks_per_seq, n_kv_heads, head_dim, block_size, dtype);
  if (rc != PKV_OK) return rc;
  if (!out || !q || !context_lens || !workspace) return PKV_ERR_NULL_POINTER;
  if (n_q_heads <= 0 || n_q_heads % n_kv_heads != 0) return PKV_ERR_BAD_SHAPE;
  const int64_t row = static_cast<int64_t>(n_q_heads) * head_dim;
  if (q_row_stride < row || out_row_stride < row) return PKV_ERR_BAD_SHAPE;
  // the tiles of a launch are counted in 32 bits
  if (static_cast<int64_t>(n_seqs < 1024 ? n_seqs : 1024) * max_blocks_per_seq * (block_size / 16) > 0x7fffffff)
    return PKV_ERR_BAD_SHAPE;
  if (workspace_bytes < decode_int8_workspace_bytes(n_q_heads, head_dim)) return PKV_ERR_WORKSPACE_TOO_SMALL;
  if (!aligned(workspace, 16) || !aligned(q, size_of(dtype)) || !aligned(out, size_of(dtype)))
    return PKV_ERR_MISALIGNED;
  AttnArgs a{};
  a.out = out;
  a.out_stride = out_row_stride;
  a.q = q;
  a.q_stride = q_row_stride;
  a.k_pool = k_pool;
  a.v_pool = v_pool;
  a.num_blocks = num_blocks;
  a.block_tables = block_tables;
  a.bt_stride = block_table_stride;
  a.max_blocks = max_blocks_per_seq;
  a.context_lens = context_lens;
  a.n_seqs = n_seqs;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.scale = scale;
  a.dtype = dtype;
  a.err = err_flags;
  a.k_scale = k_scale;
  a.v_scale = v_scale;
  CUtensorMap km, vm;
  rc = pool_tensormap(&km, k_pool, num_blocks, block_size, n_kv_heads, head_dim, kPoolInt8);
  if (rc == 0) rc = pool_tensormap(&vm, v_pool, num_blocks, block_size, n_kv_heads, head_dim, kPoolInt8);
  if (rc != 0) return rc;
  return status(launch_decode_int8(a, &km, &vm, workspace, static_cast<cudaStream_t>(stream)));
}

// rows per sequence of the laid-out keys: whole key tiles
static int64_t lay_cap(int max_blocks, int block_size) {
  return (static_cast<int64_t>(max_blocks) * block_size + 127) / 128 * 128;
}

// the scratch: K and V rows, then counters, O and (m, l) of the segments
namespace {
struct PrefillScratch {
  size_t kv, counts, o, ml, total;  // bytes of K (and of V), offsets, size
  int parts;
};
PrefillScratch prefill_scratch(int n_seqs, int n_tokens, int max_blocks, int hq, int hkv, int d, int bs, int dtype) {
  auto up = [](size_t n) { return (n + 255) / 256 * 256; };
  PrefillScratch s;
  s.kv = static_cast<size_t>(n_seqs) * lay_cap(max_blocks, bs) * hkv * d * size_of(dtype);
  s.parts = packed_split_parts(n_seqs, n_tokens, hq, hkv, static_cast<int64_t>(max_blocks) * bs, dtype);
  s.counts = up(2 * s.kv);
  s.o = s.counts + up(static_cast<size_t>(s.parts) * 32);
  s.ml = s.o + static_cast<size_t>(s.parts) * 2 * 128 * d * 4;
  s.total = s.ml + static_cast<size_t>(s.parts) * 2 * 128 * 8;
  return s;
}
}  // namespace

size_t pkv_prefill_int8_scratch_bytes(int n_seqs, int n_tokens, int max_blocks_per_seq, int n_q_heads,
                                      int n_kv_heads, int head_dim, int block_size, int dtype) {
  if (n_seqs <= 0 || n_tokens < 0 || max_blocks_per_seq <= 0 || n_kv_heads <= 0 || n_q_heads < n_kv_heads ||
      head_dim <= 0 || block_size <= 0 || !known_dtype(dtype) || n_q_heads / n_kv_heads > 65535)
    return 0;
  return prefill_scratch(n_seqs, n_tokens, max_blocks_per_seq, n_q_heads, n_kv_heads, head_dim, block_size, dtype).total;
}

int pkv_paged_prefill_attention_int8_served(
    void* out, int64_t out_row_stride, const void* q, int64_t q_row_stride, const void* k_pool,
    const void* v_pool, const float* k_scale, const float* v_scale, int num_blocks,
    const int32_t* block_tables, int64_t block_table_stride, int max_blocks_per_seq,
    const int32_t* query_start_loc, const int32_t* num_prior, const int32_t* context_lens, int n_seqs,
    int n_tokens, int n_q_heads, int n_kv_heads, int head_dim, int block_size, float scale, int dtype,
    void* scratch, size_t scratch_bytes, int* err_flags, pkv_stream_t stream) {
  if (n_seqs < 0 || n_tokens < 0) return PKV_ERR_BAD_SHAPE;
  if (n_seqs == 0 || n_tokens == 0) return PKV_OK;
  int rc = check_int8(k_pool, v_pool, k_scale, v_scale, num_blocks, block_tables, block_table_stride,
                      max_blocks_per_seq, n_kv_heads, head_dim, block_size, dtype);
  if (rc != PKV_OK) return rc;
  if (!out || !q || !query_start_loc || !num_prior || !scratch) return PKV_ERR_NULL_POINTER;
  if (n_q_heads <= 0 || n_q_heads % n_kv_heads != 0 || !(scale > 0.f)) return PKV_ERR_BAD_SHAPE;
  const int64_t row = static_cast<int64_t>(n_q_heads) * head_dim;
  if (q_row_stride < row || out_row_stride < row) return PKV_ERR_BAD_SHAPE;
  const int64_t cap = lay_cap(max_blocks_per_seq, block_size);
  if (n_seqs > 65535 || cap * n_seqs > 0x7fffffff) return PKV_ERR_BAD_SHAPE;
  const PrefillScratch sc = prefill_scratch(n_seqs, n_tokens, max_blocks_per_seq, n_q_heads, n_kv_heads,
                                            head_dim, block_size, dtype);
  if (scratch_bytes < sc.total) return PKV_ERR_WORKSPACE_TOO_SMALL;
  if (!aligned(scratch, 256) || !aligned(q, size_of(dtype)) || !aligned(out, size_of(dtype)))
    return PKV_ERR_MISALIGNED;
  if (out == q) return PKV_ERR_UNSUPPORTED;  // a row may be read again after its first store
  Int8LayArgs y{};
  y.k_pool = k_pool;
  y.v_pool = v_pool;
  y.k_scale = k_scale;
  y.v_scale = v_scale;
  y.block_tables = block_tables;
  y.bt_stride = block_table_stride;
  y.max_blocks = max_blocks_per_seq;
  y.query_start_loc = query_start_loc;
  y.num_prior = num_prior;
  y.context_lens = context_lens;
  y.n_seqs = n_seqs;
  y.num_blocks = num_blocks;
  y.block_size = block_size;
  y.n_kv_heads = n_kv_heads;
  y.head_dim = head_dim;
  y.k_out = scratch;
  uint8_t* room = static_cast<uint8_t*>(scratch);
  y.v_out = room + sc.kv;
  y.zero = reinterpret_cast<int*>(room + sc.counts);
  y.n_zero = 8 * sc.parts;
  y.cap = static_cast<int>(cap);
  y.err = err_flags;
  const cudaStream_t st = static_cast<cudaStream_t>(stream);
  cudaError_t e = launch_lay_out_int8(y, dtype, st);
  if (e != cudaSuccess) return status(e);
  PackedArgs a{};
  a.out = out;
  a.q = q;
  a.k = y.k_out;
  a.v = y.v_out;
  a.out_stride = out_row_stride;
  a.q_stride = q_row_stride;
  a.k_stride = a.v_stride = static_cast<int64_t>(n_kv_heads) * head_dim;
  a.query_start_loc = query_start_loc;
  a.num_prior = num_prior;
  a.key_cap = static_cast<int>(cap);
  a.n_key_rows = static_cast<int>(cap * n_seqs);
  a.n_parts = sc.parts;
  a.part_count = sc.parts ? y.zero : nullptr;
  a.part_o = reinterpret_cast<float*>(room + sc.o);
  a.part_ml = reinterpret_cast<float2*>(room + sc.ml);
  a.key_limit = max_blocks_per_seq * block_size;
  a.n_seqs = n_seqs;
  a.n_tokens = n_tokens;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.scale = scale;
  a.dtype = dtype;
  a.err = err_flags;
  return status(launch_packed_attention(a, st));
}

int pkv_paged_prefill_attention_int8(void* out, int64_t out_row_stride, const void* q,
                                     int64_t q_row_stride, const void* k_pool, const void* v_pool,
                                     const float* k_scale, const float* v_scale, int num_blocks,
                                     const int32_t* block_tables, int64_t block_table_stride,
                                     int max_blocks_per_seq, const int32_t* query_start_loc,
                                     const int32_t* num_prior, int n_seqs, int n_tokens,
                                     int n_q_heads, int n_kv_heads, int head_dim, int block_size,
                                     float scale, int dtype, void* scratch, size_t scratch_bytes,
                                     int* err_flags, pkv_stream_t stream) {
  return pkv_paged_prefill_attention_int8_served(
      out, out_row_stride, q, q_row_stride, k_pool, v_pool, k_scale, v_scale, num_blocks, block_tables,
      block_table_stride, max_blocks_per_seq, query_start_loc, num_prior, nullptr, n_seqs, n_tokens, n_q_heads,
      n_kv_heads, head_dim, block_size, scale, dtype, scratch, scratch_bytes, err_flags, stream);
}

int pkv_packed_prompt_attention(void* out, int64_t out_row_stride, const void* q,
                                int64_t q_row_stride, const void* k, int64_t k_row_stride,
                                const void* v, int64_t v_row_stride, const int32_t* query_start_loc,
                                int n_seqs, int n_tokens, int n_q_heads, int n_kv_heads,
                                int head_dim, float scale, int dtype, int* err_flags,
                                pkv_stream_t stream) {
  if (n_seqs < 0 || n_tokens < 0) return PKV_ERR_BAD_SHAPE;
  if (n_seqs == 0 || n_tokens == 0) return PKV_OK;
  if (!out || !q || !k || !v || !query_start_loc) return PKV_ERR_NULL_POINTER;
  if (!known_dtype(dtype)) return PKV_ERR_BAD_DTYPE;
  if (n_q_heads <= 0 || n_kv_heads <= 0 || n_q_heads % n_kv_heads != 0 || head_dim <= 0 || !(scale > 0.f))
    return PKV_ERR_BAD_SHAPE;
  const int64_t qrow = static_cast<int64_t>(n_q_heads) * head_dim, krow = static_cast<int64_t>(n_kv_heads) * head_dim;
  if (q_row_stride < qrow || out_row_stride < qrow || k_row_stride < krow || v_row_stride < krow)
    return PKV_ERR_BAD_SHAPE;
  if (n_q_heads > 65535 || n_tokens > 0x7fffffff - 1024) return PKV_ERR_BAD_SHAPE;
  if (head_dim != 64 && head_dim != 128) return PKV_ERR_UNSUPPORTED;
  const int es = size_of(dtype);
  if (!aligned(out, es) || !aligned(q, es) || !aligned(k, es) || !aligned(v, es)) return PKV_ERR_MISALIGNED;
  if (out == q || out == k || out == v) return PKV_ERR_UNSUPPORTED;  // rows are read again after a first store
  PackedArgs a{};
  a.out = out;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out_stride = out_row_stride;
  a.q_stride = q_row_stride;
  a.k_stride = k_row_stride;
  a.v_stride = v_row_stride;
  a.query_start_loc = query_start_loc;
  a.n_key_rows = n_tokens;
  a.n_seqs = n_seqs;
  a.n_tokens = n_tokens;
  a.n_q_heads = n_q_heads;
  a.n_kv_heads = n_kv_heads;
  a.head_dim = head_dim;
  a.scale = scale;
  a.dtype = dtype;
  a.err = err_flags;
  return status(launch_packed_attention(a, static_cast<cudaStream_t>(stream)));
}

}  // extern "C"
