// Internal launcher interface shared by the C-ABI layer (abi.cu) and the
// kernel translation units.  Every launcher enqueues work on `stream` and
// returns a pkv::Status; none of them synchronizes.
#pragma once

#include <cuda_runtime.h>

#include <atomic>
#include <cstddef>
#include <cstdint>
#include <string>

namespace pkv {

// Per-device error word (abi.cu).  Kernels record the first bad-input or
// timeout event here instead of trapping.
int* device_error_word();

// Raises a kernel's dynamic shared memory limit, once per device: `done` is a
// flag word of that kernel, one bit per device (abi.cu).
void allow_shared_memory(const void* kernel, int bytes, std::atomic<uint64_t>& done);

// Thread-local message for the last failing call (abi.cu).
void set_error(const std::string& msg);

// ---- quantize.cu ----------------------------------------------------------
// skip (nullable): blocks with a nonzero byte are neither read nor written.
int launch_quantize(const void* kv, int dtype, int8_t* q, float* scale, int64_t num_blocks,
                    int block_size, int num_kv_heads, int head_dim, const uint8_t* skip,
                    cudaStream_t stream);

// ---- attn_stats.cu ------------------------------------------------------------
size_t attention_stats_workspace_size(int64_t num_blocks, int block_size, int num_kv_heads);
int launch_attention_stats(const void* k, int dtype, const float* q, float* attn,
                           int64_t num_blocks, int block_size, int num_kv_heads, float sm_scale,
                           void* workspace, size_t workspace_bytes, cudaStream_t stream);

// ---- compose.cu -------------------------------------------------------------
int launch_mark_blocks(const int64_t* ids, int64_t n, int64_t id_offset, int64_t num_blocks,
                       uint8_t* mask, cudaStream_t stream);
int launch_compact_tables(const int32_t* block_tables, const int32_t* seq_lens,
                          const uint8_t* evicted, int32_t* tables_out, int32_t* lens_out,
                          int num_seqs, int max_blocks_per_seq, int block_size,
                          int64_t num_blocks, cudaStream_t stream);

int launch_write_to_cache(const void* key, const void* value, int dtype, int8_t* kv_cache,
                          float* scale_cache, const int64_t* slot_mapping, int64_t num_tokens,
                          int64_t num_blocks, int block_size, int num_kv_heads, int head_dim,
                          void* workspace, size_t workspace_bytes, cudaStream_t stream);
size_t write_to_cache_workspace_size(int64_t num_tokens, int num_kv_heads);

// ---- rotary.cu ------------------------------------------------------------
struct QkNormRopeArgs {
  const void* q;
  const void* k;
  void* q_out;
  void* k_out;
  int dtype;  // 0 fp32, 1 fp16, 2 bf16
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride;  // elements
  const int64_t* positions;
  const float* table;  // [table_rows, rot]: cos | sin
  const void* q_weight;  // nullable with k_weight: no norm
  const void* k_weight;
  bool weight_f32;
  int64_t tokens, table_rows;
  int heads, kv_heads, dim, rot;
  float eps;
  bool interleaved;
};
int launch_qk_norm_rope(const QkNormRopeArgs& a, cudaStream_t stream);

struct AppendKvArgs {
  const void* key;
  const void* value;
  int dtype;
  int64_t k_token_stride, k_head_stride, v_token_stride, v_head_stride;  // elements
  int8_t* cache;
  float* scales;
  const int64_t* slots;
  const int64_t* positions;  // nullable: no rotation
  const float* table;
  int64_t tokens, blocks, table_rows;
  int block_size, kv_heads, dim, rot;
  bool interleaved;
};
size_t append_kv_workspace_size(int64_t tokens, int64_t blocks);
int launch_append_kv(const AppendKvArgs& a, void* workspace, size_t workspace_bytes,
                     cudaStream_t stream);

// ---- prefill.cu -----------------------------------------------------------
struct PrefillArgs {
  const void* q;
  const void* k;
  const void* v;
  void* out;
  float* lse;  // nullable
  int dtype;   // 1 fp16, 2 bf16
  const int32_t* cu_q;
  const int32_t* cu_k;
  int num_seqs, heads, kv_heads, dim;
  int64_t total_q, total_k;
  int64_t q_token_stride, q_head_stride, k_token_stride, k_head_stride, v_token_stride,
      v_head_stride;  // elements, multiples of 8
  float sm_scale;
  bool causal;
};
// The workspace is nullable: without it O is summed over all keys at once.
size_t prefill_workspace_size(const PrefillArgs& a);
int launch_prefill(const PrefillArgs& a, void* workspace, size_t workspace_bytes,
                   cudaStream_t stream);

// ---- eviction.cu ----------------------------------------------------------
int launch_eviction_scores(const float* recency, const float* frequency, const float* attn,
                           const uint8_t* valid, float* scores, int64_t num_blocks,
                           int block_size, float w_r, float w_f, float w_a,
                           cudaStream_t stream);

size_t select_workspace_size(int64_t n, int64_t k);
// Sorts (orderable(score) << 32 | id) keys; emits the first k ids (out_ids)
// and/or the first k keys with `id_offset` added to the id (out_keys).
int launch_select(const float* scores, const uint64_t* keys_in, int64_t n, int64_t k,
                  int64_t id_offset, int64_t* out_ids, uint64_t* out_keys, void* workspace,
                  size_t workspace_bytes, cudaStream_t stream);

// Single-launch cluster path (eviction_cluster.cu) for n <= 16,384: scores
// from the statistics (scores_in == nullptr) or given scores; writes the k
// selected ids.  Returns kUnsupported without launching when it cannot run.
int launch_cluster_select(const float* rec, const float* freq, const float* attn,
                          const uint8_t* valid, const float* scores_in, float* scores_out,
                          int64_t n, int bs, float wr, float wf, float wa, int64_t k,
                          int64_t* out_ids, cudaStream_t stream);
int cluster_select_max_blocks();
// True when the current device can schedule the selection cluster.
bool cluster_select_available();
// Workspace bytes for pkv_eviction_select: 0 when the cluster path runs.
size_t scores_select_workspace_size(int64_t n, int64_t k);

size_t fused_select_workspace_size(int64_t n, int64_t k);
int launch_scores_select(const float* recency, const float* frequency, const float* attn,
                         const uint8_t* valid, float* scores, int64_t num_blocks,
                         int block_size, float w_r, float w_f, float w_a, int64_t k,
                         int64_t* out_ids, void* workspace, size_t workspace_bytes,
                         cudaStream_t stream);

// ---- decode.cu ------------------------------------------------------------
struct DecodeArgs {
  const float* q;
  const int8_t* k_cache;
  const float* k_scale;
  const int8_t* v_cache;
  const float* v_scale;
  const int32_t* block_tables;
  const int32_t* seq_lens;
  float* out;
  int num_seqs, num_heads, num_kv_heads, head_dim, block_size;
  int64_t num_blocks;
  int max_blocks_per_seq;
  float sm_scale;
};

size_t decode_workspace_size(const DecodeArgs& a);
// Kernels one launch_decode call issues for these arguments.
int decode_kernel_launches(const DecodeArgs& a);
int launch_decode(const DecodeArgs& a, void* workspace, size_t workspace_bytes,
                  cudaStream_t stream);

// Decode as partials: the split kernel alone, every split's (acc, m in log2
// units, l) at slot (seq * max_splits + split) * num_heads + head of ws_acc
// [slots][head_dim] and ws_ml [slots]; a sequence has ceil(pages /
// pages_per_split) splits, its other slots are not written.  `a.out` is unused.
// The plan is false for shapes that only the generic kernel takes; those are not
// launched so.
bool decode_partials_plan(const DecodeArgs& a, int* max_splits, int* pages_per_split);
int launch_decode_partials(const DecodeArgs& a, float* ws_acc, float2* ws_ml, cudaStream_t stream);

// ---- prefix.cu ------------------------------------------------------------
struct SharedPrefixArgs {
  DecodeArgs own;  // queries, caches, each sequence's own pages, output
  const int32_t* prefix_table;
  const int32_t* prefix_len;
  int prefix_width;
};
size_t shared_prefix_workspace_size(const SharedPrefixArgs& a);
int launch_shared_prefix(const SharedPrefixArgs& a, void* workspace, size_t workspace_bytes,
                         cudaStream_t stream);

// ---- chunk.cu --------------------------------------------------------------
// Words of the tables' pages that become zero beside a call's plan (sums null: none).
struct ZeroArgs {
  const int32_t* tables = nullptr;
  const int32_t* lens = nullptr;
  unsigned long long* sums = nullptr;  // [num_blocks, block_size]
  int64_t num_blocks = 0;
  int seqs = 0, block_size = 0, width = 0;
};

struct ChunkArgs {
  const void* q;
  int dtype;  // 0 fp32, 1 fp16, 2 bf16: of q and out
  const int8_t* k_cache;
  const float* k_scale;
  const int8_t* v_cache;  // null: only lse is computed
  const float* v_scale;
  const int32_t* tables;  // [seqs, width]
  const int32_t* lens;    // [seqs]
  const int32_t* cu;      // [seqs + 1]
  void* out;
  float* lse;  // nullable
  float* logits = nullptr;  // with lse alone: also the scores, [total_q * heads][width * block_size]
  ZeroArgs zero;
  int64_t total_q, num_blocks;
  int64_t q_token_stride, q_head_stride;  // elements, of 16 bytes
  int seqs, heads, kv_heads, dim, block_size, width;
  float sm_scale;
};
size_t chunk_workspace_size(const ChunkArgs& a);
int launch_chunk(const ChunkArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t stream);

// ---- weights.cu ------------------------------------------------------------
// q, the K cache and the tables of `a`, and a.lse as input (nullable: computed first);
// a.v_cache, a.v_scale and a.out are unused.  weights [num_blocks, block_size] is added to.
size_t accumulate_workspace_size(const ChunkArgs& a);
int launch_accumulate(const ChunkArgs& a, float* weights, void* workspace, size_t workspace_bytes,
                      cudaStream_t stream);

// ---- evict.cu ----------------------------------------------------------------
struct EvictArgs {
  int8_t* cache;   // [2, num_blocks, block_size, kv_heads, dim]
  float* scales;   // [2, num_blocks, kv_heads]
  float* weights;  // [num_blocks, block_size]
  const int32_t* tables;
  const int32_t* lens;
  int32_t* lens_out;
  int32_t* kept;   // [seqs, keep]
  int64_t num_blocks;
  int seqs, block_size, kv_heads, dim, width;
  int keep, sinks, recent;
};
int launch_evict(const EvictArgs& a, cudaStream_t stream);

}  // namespace pkv
