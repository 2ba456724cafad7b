// pkv_internal.h -- host-side launchers shared between the kernel files and
// the C ABI (pkv_abi.cu).  Argument validation happens in pkv_abi.cu; these
// functions assume valid shapes and only launch.
#pragma once

#include <cuda.h>
#include <cuda_runtime.h>
#include <stdint.h>

namespace pkv {

// pool format code (internal; not an ABI dtype) of fp8 e4m3 pools, for
// encode_pool_tensormap / pool_tensormap
constexpr int kPoolFp8 = 100;
// ... and of int8 pools (16-row boxes whatever the block size)
constexpr int kPoolInt8 = 101;

struct RopeArgs {
  void* q_out;
  int64_t q_out_stride;  // elements between token rows
  const void* qkv;
  int64_t qkv_stride;
  const int64_t* positions;
  const void* cos_t;
  const void* sin_t;
  int max_pos;
  void* k_pool;
  void* v_pool;
  const int64_t* slots;
  int n_tokens, num_blocks, block_size, n_q_heads, n_kv_heads, head_dim, dtype;
  int* err;
  // fp8 e4m3 pools: per-(slot, KV head) scales written with the bytes (NULL: 16/32-bit pools)
  float* k_scale = nullptr;
  float* v_scale = nullptr;
};
cudaError_t launch_rope_reshape_and_cache(const RopeArgs& a, cudaStream_t stream);

struct AttnArgs {
  void* out;
  int64_t out_stride;  // elements between token rows of out
  const void* q;
  int64_t q_stride;    // elements between token rows of q
  const void* k_pool;
  const void* v_pool;
  int num_blocks;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  // decode: context_lens != nullptr, one query row per sequence
  const int32_t* context_lens;
  // prefill: query_start_loc / num_prior
  const int32_t* query_start_loc;
  const int32_t* num_prior;
  int n_seqs;
  int n_tokens;
  int max_query_len;
  int n_q_heads;
  int n_kv_heads;
  int head_dim;
  int block_size;
  float scale;
  int dtype;
  int* err;
  // decode only: the new token of each sequence, written by the decode
  // kernel at position context_lens[s] - 1 before it is read (NULL = none)
  const void* k_new = nullptr;
  const void* v_new = nullptr;
  int64_t k_new_stride = 0;  // elements between rows
  int64_t v_new_stride = 0;
  // fp8 e4m3 pools: one fp32 scale per (slot, KV head); NULL = 16/32-bit pools
  // of `dtype` (q, out and the dequantised arithmetic stay in `dtype`)
  const float* k_scale = nullptr;
  const float* v_scale = nullptr;
  // decode: the step's schedule built by pkv_decode_schedule (NULL = none)
  const void* schedule = nullptr;
  // decode (tensor-core path): a device word the kernel waits on, bounded,
  // until it is nonzero before reading q / k_new / v_new (NULL = none)
  const int* input_ready = nullptr;
  // decode: one layer of a multi-layer call with a workspace per layer (NULL:
  // a single-layer call, its merge launched behind it)
  const struct LayerChain* chain = nullptr;
};

// Layers of one multi-layer decode call, each with its own split-K
// workspace: the decode kernels of layers after the first wait for their
// predecessor only at their end (defer_wait), and one merge launch after the
// last layer's decode covers every layer.
struct LayerChain {
  int defer_wait;            // this layer's decode kernel
  int merge;                 // launch the merge of all n_layers after this decode
  int n_layers;
  void* out0;                // layer 0's output rows
  int64_t out_layer_stride;  // elements between layers' outputs
  void* ws0;                 // layer 0's workspace
  int64_t ws_layer_stride;   // bytes between layers' workspaces
};
cudaError_t launch_reshape_and_cache_fp8(const void* k, const void* v, int64_t k_stride,
                                         int64_t v_stride, void* k_pool, void* v_pool,
                                         float* k_scale, float* v_scale, const int64_t* slots,
                                         int n_tokens, int num_blocks, int block_size,
                                         int n_kv_heads, int head_dim, int src_dtype, int* err,
                                         cudaStream_t stream);

cudaError_t launch_reshape_and_cache(const void* k, const void* v, int64_t k_stride,
                                     int64_t v_stride, void* k_pool, void* v_pool,
                                     const int64_t* slots, int n_tokens, int num_blocks,
                                     int block_size, int n_kv_heads, int head_dim, int esize,
                                     int* err, cudaStream_t stream);

cudaError_t launch_append_at_context_end_fp8(const void* k, const void* v, int64_t k_stride,
                                             int64_t v_stride, void* k_pool, void* v_pool,
                                             float* k_scale, float* v_scale, const int32_t* tables,
                                             int64_t bt_stride, int max_blocks,
                                             const int32_t* context_lens, int n_seqs,
                                             int num_blocks, int block_size, int n_kv_heads,
                                             int head_dim, int src_dtype, int* err,
                                             cudaStream_t stream);
cudaError_t launch_append_at_context_end(const void* k, const void* v, int64_t k_stride,
                                         int64_t v_stride, void* k_pool, void* v_pool,
                                         const int32_t* tables, int64_t bt_stride, int max_blocks,
                                         const int32_t* context_lens, int n_seqs, int num_blocks,
                                         int block_size, int n_kv_heads, int head_dim, int esize,
                                         int* err, cudaStream_t stream);

size_t decode_schedule_bytes(int n_seqs, int max_blocks);
cudaError_t launch_decode_schedule(void* schedule, const AttnArgs& a, cudaStream_t stream);
cudaError_t launch_copy_blocks_peer(void* dst_k, void* dst_v, int64_t dst_layer_stride,
                                    int dst_num_blocks, const void* src_k, const void* src_v,
                                    int64_t src_layer_stride, int src_num_blocks, int n_layers,
                                    const int32_t* pairs, int n_pairs, int64_t block_bytes, int* err,
                                    cudaStream_t stream);
cudaError_t launch_copy_blocks(void* k_pools, void* v_pools, int64_t layer_stride, int n_layers,
                               const int32_t* pairs, int n_pairs, int num_blocks,
                               int64_t block_bytes, int* err, cudaStream_t stream);

// CUDA-core attention for any dtype / head_dim <= 256 / block_size; decode
// (context_lens set) or chunked prefill (query_start_loc + num_prior set).
cudaError_t launch_generic_attention(const AttnArgs& a, cudaStream_t stream);

// Decode fast path: TMA + mbarrier pipeline, tensor-core math, stream-K
// split with fused combine.  Requires fp16/bf16, head_dim 64, block 16,
// n_kv_heads in {1,2,4}, q heads per kv head <= 8.
bool decode_fast_supported(const AttnArgs& a);
bool decode_fast_supported_shape(const AttnArgs& a);
size_t decode_workspace_bytes(int n_seqs, int n_q_heads, int head_dim);
cudaError_t launch_decode_fast(const AttnArgs& a, const CUtensorMap* kmap, const CUtensorMap* vmap,
                               void* workspace, cudaStream_t stream);

// TMA descriptor for a pool [num_blocks*block_size][n_kv_heads][head_dim]
// with one (head_dim x 1 head x block_size tokens) box, 128-byte swizzle.
// Returns 0 or a CUresult.
int encode_pool_tensormap(CUtensorMap* map, const void* pool, int num_blocks, int block_size,
                          int n_kv_heads, int head_dim, int dtype);

// Chunked prefill on tcgen05 tensor cores: fp16/bf16, head_dim 64, block 16,
// 16-byte aligned q / out rows.
bool prefill_fast_supported(const AttnArgs& a);
bool prefill_fp8_tc_supported(const AttnArgs& a);
size_t prefill_fp8_scratch_bytes(int n_seqs, int max_blocks, int n_kv_heads, int head_dim);
cudaError_t launch_dequant_blocks(const AttnArgs& a, void* scratch, cudaStream_t stream,
                                  void** k_out, void** v_out, int32_t** table_out);
cudaError_t launch_prefill_fast(const AttnArgs& a, const CUtensorMap* qmap, const CUtensorMap* kmap,
                                const CUtensorMap* vmap, cudaStream_t stream);
// TMA descriptor for q viewed as [n_tokens][n_q_heads][head_dim] (row stride
// q_stride elements) with one (head_dim x 1 head x 128 tokens) box, 128-byte
// swizzle.  Returns 0 or PKV_ERR_DRIVER.
int encode_q_tensormap(CUtensorMap* map, const void* q, int64_t q_stride, int n_tokens,
                       int n_q_heads, int head_dim, int dtype);

// ---- step tables (pkv_step_tables.cu)
constexpr int kStepTablesMaxSeqs = 16384;
struct StepTablesArgs {
  int32_t* block_tables;  // [n_seqs][bt_stride], new entries written
  int64_t bt_stride;
  int max_blocks;
  const int32_t* free_blocks;  // [free_capacity], taken from the end
  int free_capacity;
  const int32_t* n_free;
  int32_t* n_free_out;
  const int32_t* num_prior;
  const int32_t* num_new;
  int n_seqs, block_size;
  int32_t* context_lens;
  int32_t* query_start_loc;  // [n_seqs + 1]
  int64_t* slot_mapping;     // [n_tokens]
  int64_t* positions;        // [n_tokens]
  int n_tokens;
  int* err;
  int vec_ok;  // slot_mapping and positions take 16-byte stores (set by the launcher)
};
cudaError_t launch_step_tables(StepTablesArgs a, cudaStream_t stream);

// ---- int8 pools with a scale per (block, KV head) (pkv_int8.cu, pkv_decode_int8.cu)
struct Int8RowsArgs {
  const void* k;  // append: the new rows; fetch: the output rows
  const void* v;
  int64_t k_stride, v_stride;  // elements between rows
  void* k_pool;
  void* v_pool;
  float* k_scale;
  float* v_scale;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* context_lens;
  const int32_t* start_loc;  // [n_seqs + 1]: the last start_loc[i + 1] - start_loc[i] rows of context i
  int n_seqs, n_rows, num_blocks, block_size, n_kv_heads, head_dim, dtype;
  int* err;
  int k_vec, v_vec, k_vec16, v_vec16;  // set by the launcher: accesses of 4 elements, of 16 bytes
  int heads_per_warp;                     // likewise
  int64_t n_units;
};
cudaError_t launch_append_int8(Int8RowsArgs a, cudaStream_t stream);
cudaError_t launch_fetch_int8(Int8RowsArgs a, cudaStream_t stream);
struct Int8LayArgs {
  const void* k_pool;
  const void* v_pool;
  const float* k_scale;
  const float* v_scale;
  const int32_t* block_tables;
  int64_t bt_stride;
  int max_blocks;
  const int32_t* query_start_loc;
  const int32_t* num_prior;
  const int32_t* context_lens;  // NULL, or 0 for a sequence that is not served: its rows are zeros
  int n_seqs, num_blocks, block_size, n_kv_heads, head_dim;
  void* k_out;
  void* v_out;
  int cap;  // rows per sequence in k_out / v_out, a multiple of 128
  int* zero;  // words to clear for the attention behind this pass
  int n_zero;
  int* err;
};
cudaError_t launch_lay_out_int8(const Int8LayArgs& a, int dtype, cudaStream_t stream);
// AttnArgs with k_scale / v_scale per (block, KV head); decode form
size_t decode_int8_workspace_bytes(int n_q_heads, int head_dim);
cudaError_t launch_decode_int8(const AttnArgs& a, const CUtensorMap* kmap, const CUtensorMap* vmap,
                               void* workspace, cudaStream_t stream);

// ---- causal attention over consecutive rows (pkv_packed.cu)
struct PackedArgs {
  void* out;
  const void* q;
  const void* k;
  const void* v;
  int64_t out_stride, q_stride, k_stride, v_stride;  // elements between token rows
  const int32_t* query_start_loc;
  // NULL: the keys of sequence s are its own rows query_start_loc[s] .. (a
  // whole prompt).  Otherwise they are rows s * key_cap .. of k / v, num_prior[s]
  // of them before the first query.
  const int32_t* num_prior;
  int key_cap;
  int key_limit;   // keys a sequence's table can hold
  int n_key_rows;  // rows of k / v
  // splitting of long items over their keys: zeroed counters (8 a segment) and
  // partials for n_parts segments (packed_split_parts; 0: none)
  int* part_count = nullptr;
  float* part_o = nullptr;   // 16-byte aligned
  float2* part_ml = nullptr;
  int n_parts = 0;
  int n_seqs, n_tokens, n_q_heads, n_kv_heads, head_dim;
  float scale;
  int dtype;
  int* err;
};
cudaError_t launch_packed_attention(const PackedArgs& a, cudaStream_t stream);
// segments that a chunk call of these sizes may be split into (0: it is not)
int packed_split_parts(int n_seqs, int n_tokens, int n_q_heads, int n_kv_heads, int64_t key_limit, int dtype);

// TMA descriptor for rows [n_rows][n_heads][head_dim] of 16-bit values (row stride
// in elements) with a box of 64 dims x box_heads x box_rows, 128-byte swizzle.
// Returns 0 or PKV_ERR_DRIVER.
int encode_rows_tensormap(CUtensorMap* map, const void* rows, int64_t row_stride, int n_rows,
                          int n_heads, int head_dim, int dtype, int box_heads, int box_rows);

// Argument checks, TMA-descriptor cache and kernel selection of pkv_abi.cu,
// reused by the allocation-free decode entry point.
int validate_attention_args(const void* out, int64_t out_stride, const void* q, int64_t q_stride,
                            const void* k_pool, const void* v_pool, int num_blocks,
                            const int32_t* tables, int64_t bt_stride, int max_blocks,
                            int n_q_heads, int n_kv_heads, int head_dim, int block_size, int dtype);
int pool_tensormap(CUtensorMap* out, const void* pool, int num_blocks, int block_size,
                   int n_kv_heads, int head_dim, int dtype);
int decode_impl_setting();

}  // namespace pkv
