// extern "C" entry points of libpagedkv_sm100.so (declared in
// include/pagedkv_fusion.h): argument checks with the reference launcher's
// messages (csrc/eviction_score.cu:105-110, csrc/quant_paged_attention.cu:
// 181-197), then dispatch to the kernel launchers.
#include <cuda_runtime.h>
#include <algorithm>

#include <cstdint>
#include <mutex>
#include <string>

#include "../../include/pagedkv_fusion.h"
#include "pkv_common.cuh"
#include "pkv_internal.h"

namespace pkv {

namespace {
thread_local std::string g_last_error;
constexpr int kMaxDevices = 64;
}  // namespace

// One error word per device: a file-scope __device__ variable exists once
// in every device context that loads this library.
__device__ int g_device_error = 0;

void set_error(const std::string& msg) { g_last_error = msg; }

int* device_error_word() {
  static int* ptrs[kMaxDevices] = {nullptr};
  static std::mutex mu;
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return nullptr;
  std::lock_guard<std::mutex> lock(mu);
  if (ptrs[dev] == nullptr) {
    void* p = nullptr;
    if (cudaGetSymbolAddress(&p, g_device_error) != cudaSuccess) return nullptr;
    ptrs[dev] = static_cast<int*>(p);
  }
  return ptrs[dev];
}

void allow_shared_memory(const void* kernel, int bytes, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return;
  const uint64_t bit = 1ull << dev;
  if (done.load(std::memory_order_acquire) & bit) return;
  // on an error the launch fails and reports it
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) ==
      cudaSuccess)
    done.fetch_or(bit, std::memory_order_release);
}

}  // namespace pkv

using pkv::set_error;

namespace {

inline cudaStream_t as_stream(void* s) { return static_cast<cudaStream_t>(s); }

inline int fail(int code, const std::string& msg) {
  set_error(msg);
  return code;
}

inline void clear_error() { set_error(""); }

}  // namespace

extern "C" {

const char* pkv_last_error_string(void) { return pkv::g_last_error.c_str(); }

int pkv_version(void) { return 10000; }

int pkv_read_device_error(int32_t* code, int reset) {
  clear_error();
  cudaError_t e = cudaDeviceSynchronize();
  if (e != cudaSuccess)
    return fail(PKV_ERR_CUDA, std::string("device synchronize failed: ") + cudaGetErrorString(e));
  int v = 0;
  e = cudaMemcpyFromSymbol(&v, pkv::g_device_error, sizeof(int));
  if (e != cudaSuccess)
    return fail(PKV_ERR_CUDA, std::string("reading the device error word failed: ") +
                                  cudaGetErrorString(e));
  if (reset && v != 0) {
    const int zero = 0;
    e = cudaMemcpyToSymbol(pkv::g_device_error, &zero, sizeof(int));
    if (e != cudaSuccess)
      return fail(PKV_ERR_CUDA, std::string("clearing the device error word failed: ") +
                                    cudaGetErrorString(e));
  }
  if (code) *code = v;
  if (v != 0) return fail(PKV_ERR_DEVICE_INPUT, "a kernel recorded device error code " +
                                                    std::to_string(v));
  return PKV_OK;
}

int pkv_eviction_scores(const float* recency, const float* frequency, const float* attn_weights,
                        const uint8_t* valid_mask, float* scores, int64_t num_blocks,
                        int32_t block_size, float w_recency, float w_frequency,
                        float w_attention, void* stream) {
  clear_error();
  if (num_blocks < 0 || block_size < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "attn_weights must be [num_blocks, block_size]");
  if (num_blocks > 0 && (!recency || !frequency || !scores ||
                         (block_size > 0 && (!attn_weights || !valid_mask))))
    return fail(PKV_ERR_INVALID_ARGUMENT, "all inputs must be CUDA tensors");
  return pkv::launch_eviction_scores(recency, frequency, attn_weights, valid_mask, scores,
                                     num_blocks, block_size, w_recency, w_frequency, w_attention,
                                     as_stream(stream));
}

size_t pkv_eviction_select_workspace_size(int64_t num_blocks, int64_t k) {
  return pkv::scores_select_workspace_size(num_blocks, k);
}

static int check_select(int64_t n, int64_t k, const void* in, const void* out) {
  if (k < 0) return fail(PKV_ERR_INVALID_ARGUMENT, "k must be non-negative");
  if (n < 0) return fail(PKV_ERR_INVALID_ARGUMENT, "num_blocks must be non-negative");
  if (n > ((int64_t)1 << 31))
    return fail(PKV_ERR_UNSUPPORTED, "more than 2^31 blocks per selection");
  if (n > 0 && k > 0 && (!in || !out))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  return PKV_OK;
}

int pkv_eviction_select(const float* scores, int64_t num_blocks, int64_t k, int64_t* out_indices,
                        void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = check_select(num_blocks, k, scores, out_indices);
  if (rc != PKV_OK) return rc;
  return pkv::launch_select(scores, nullptr, num_blocks, k, 0, out_indices, nullptr, workspace,
                            workspace_bytes, as_stream(stream));
}

size_t pkv_eviction_scores_select_workspace_size(int64_t num_blocks, int64_t k) {
  return pkv::fused_select_workspace_size(num_blocks, k);
}

int pkv_eviction_scores_select(const float* recency, const float* frequency,
                               const float* attn_weights, const uint8_t* valid_mask,
                               float* scores, int64_t num_blocks, int32_t block_size,
                               float w_recency, float w_frequency, float w_attention, int64_t k,
                               int64_t* out_indices, void* workspace, size_t workspace_bytes,
                               void* stream) {
  clear_error();
  if (num_blocks < 0 || block_size < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "attn_weights must be [num_blocks, block_size]");
  int rc = check_select(num_blocks, k, recency, out_indices);
  if (rc != PKV_OK) return rc;
  if (num_blocks > 0 &&
      (!recency || !frequency || (block_size > 0 && (!attn_weights || !valid_mask))))
    return fail(PKV_ERR_INVALID_ARGUMENT, "all inputs must be CUDA tensors");
  return pkv::launch_scores_select(recency, frequency, attn_weights, valid_mask, scores,
                                   num_blocks, block_size, w_recency, w_frequency, w_attention,
                                   k, out_indices, workspace, workspace_bytes,
                                   as_stream(stream));
}

int pkv_eviction_local_candidates(const float* scores, int64_t num_blocks, int64_t k,
                                  int64_t id_offset, uint64_t* out_keys, void* workspace,
                                  size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = check_select(num_blocks, k, scores, out_keys);
  if (rc != PKV_OK) return rc;
  if (id_offset < 0 || id_offset + num_blocks > ((int64_t)1 << 32))
    return fail(PKV_ERR_INVALID_ARGUMENT, "global block ids must lie in [0, 2^32)");
  return pkv::launch_select(scores, nullptr, num_blocks, k, id_offset, nullptr, out_keys,
                            workspace, workspace_bytes, as_stream(stream));
}

size_t pkv_eviction_merge_workspace_size(int64_t num_keys, int64_t k) {
  return pkv::select_workspace_size(num_keys, k);
}

int pkv_eviction_merge(const uint64_t* keys, int64_t num_keys, int64_t k, int64_t* out_indices,
                       void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  int rc = check_select(num_keys, k, keys, out_indices);
  if (rc != PKV_OK) return rc;
  return pkv::launch_select(nullptr, keys, num_keys, k, 0, out_indices, nullptr, workspace,
                            workspace_bytes, as_stream(stream));
}

static int quantize_checked(const void* kv, int32_t kv_dtype, int8_t* q, float* scale,
                            int64_t num_blocks, int32_t block_size, int32_t num_kv_heads,
                            int32_t head_dim, const uint8_t* skip, void* stream) {
  if (num_blocks < 0 || block_size < 0 || num_kv_heads < 0 || head_dim < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "expected 4D [nb, bs, nkv, hd]");
  if (kv_dtype < 0 || kv_dtype > 2)
    return fail(PKV_ERR_INVALID_ARGUMENT, "kv must be float32, float16 or bfloat16");
  if (num_blocks > 0 && num_kv_heads > 0 && (!kv || !q || !scale))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (num_blocks > 0x7fffffffLL)
    return fail(PKV_ERR_UNSUPPORTED, "more than 2^31 - 1 blocks in one call");
  if ((int64_t)num_kv_heads * 4 > 48 * 1024)
    return fail(PKV_ERR_UNSUPPORTED, "num_kv_heads too large");
  if (num_kv_heads == 0) return PKV_OK;
  return pkv::launch_quantize(kv, kv_dtype, q, scale, num_blocks, block_size, num_kv_heads,
                              head_dim, skip, as_stream(stream));
}

int pkv_quantize_kv_per_block(const void* kv, int32_t kv_dtype, int8_t* q, float* scale,
                              int64_t num_blocks, int32_t block_size, int32_t num_kv_heads,
                              int32_t head_dim, void* stream) {
  clear_error();
  return quantize_checked(kv, kv_dtype, q, scale, num_blocks, block_size, num_kv_heads, head_dim,
                          nullptr, stream);
}

int pkv_quantize_kv_per_block_except(const void* kv, int32_t kv_dtype, const uint8_t* skip,
                                     int8_t* q, float* scale, int64_t num_blocks,
                                     int32_t block_size, int32_t num_kv_heads, int32_t head_dim,
                                     void* stream) {
  clear_error();
  if (num_blocks > 0 && !skip) return fail(PKV_ERR_INVALID_ARGUMENT, "null skip mask");
  return quantize_checked(kv, kv_dtype, q, scale, num_blocks, block_size, num_kv_heads, head_dim,
                          skip, stream);
}

size_t pkv_attention_stats_workspace_size(int64_t num_blocks, int32_t block_size,
                                          int32_t num_kv_heads) {
  if (num_blocks <= 0 || block_size <= 0 || num_kv_heads <= 0) return 0;
  return pkv::attention_stats_workspace_size(num_blocks, block_size, num_kv_heads);
}

int pkv_attention_stats(const void* k, int32_t k_dtype, const float* q, float* attn,
                        int64_t num_blocks, int32_t block_size, int32_t num_kv_heads,
                        int32_t head_dim, float sm_scale, void* workspace, size_t workspace_bytes,
                        void* stream) {
  clear_error();
  if (num_blocks < 0 || num_kv_heads <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "expected K [nb, bs, nkv, 128] and q [nkv, 128]");
  if (head_dim != 128) return fail(PKV_ERR_UNSUPPORTED, "attention statistics need head_dim 128");
  if (block_size != 16 && block_size != 32)
    return fail(PKV_ERR_UNSUPPORTED, "attention statistics need block_size 16 or 32");
  if (k_dtype < 0 || k_dtype > 2)
    return fail(PKV_ERR_INVALID_ARGUMENT, "k must be float32, float16 or bfloat16");
  if (num_blocks > 0 && (!k || !q || !attn))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  const size_t elem = k_dtype == 0 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(k) % (4 * elem) != 0 || reinterpret_cast<uintptr_t>(q) % 16 != 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "k and q must be aligned to 4 elements / 16 bytes");
  return pkv::launch_attention_stats(k, k_dtype, q, attn, num_blocks, block_size, num_kv_heads,
                                     sm_scale, workspace, workspace_bytes, as_stream(stream));
}

int pkv_mark_blocks(const int64_t* ids, int64_t num_ids, int64_t id_offset, int64_t num_blocks,
                    uint8_t* mask, void* stream) {
  clear_error();
  if (num_ids < 0 || num_blocks < 0) return fail(PKV_ERR_INVALID_ARGUMENT, "negative size");
  if ((num_ids > 0 && !ids) || (num_blocks > 0 && !mask))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  return pkv::launch_mark_blocks(ids, num_ids, id_offset, num_blocks, mask, as_stream(stream));
}

int pkv_compact_block_tables(const int32_t* block_tables, const int32_t* seq_lens,
                             const uint8_t* evicted, int32_t* tables_out, int32_t* lens_out,
                             int32_t num_seqs, int32_t max_blocks_per_seq, int32_t block_size,
                             int64_t num_blocks, void* stream) {
  clear_error();
  if (num_seqs < 0 || max_blocks_per_seq < 0 || block_size <= 0 || num_blocks < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "invalid table shape");
  if (num_seqs > 0 && (!block_tables || !seq_lens || !evicted || !tables_out || !lens_out))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  return pkv::launch_compact_tables(block_tables, seq_lens, evicted, tables_out, lens_out,
                                    num_seqs, max_blocks_per_seq, block_size, num_blocks,
                                    as_stream(stream));
}

static int check_decode(const pkv::DecodeArgs& a) {
  if (a.num_seqs < 0 || a.num_heads <= 0 || a.num_kv_heads <= 0 || a.head_dim <= 0 ||
      a.block_size <= 0 || a.num_blocks < 0 || a.max_blocks_per_seq < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "invalid decode shape");
  if (a.head_dim % 32 != 0 || a.head_dim > 256)
    return fail(PKV_ERR_INVALID_ARGUMENT, "supports head_dim % 32 == 0, <= 256");
  if (a.block_size > 64) return fail(PKV_ERR_INVALID_ARGUMENT, "supports block_size <= 64");
  if (a.num_heads % a.num_kv_heads != 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "GQA requires num_heads % num_kv_heads == 0");
  if (a.num_seqs > 0 && (!a.q || !a.k_cache || !a.k_scale || !a.v_cache || !a.v_scale ||
                         !a.seq_lens || !a.out || (a.max_blocks_per_seq > 0 && !a.block_tables)))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (a.num_heads > 65535) return fail(PKV_ERR_UNSUPPORTED, "num_heads > 65535");
  return PKV_OK;
}

static pkv::DecodeArgs decode_args(const float* q, const int8_t* k_cache, const float* k_scale,
                                   const int8_t* v_cache, const float* v_scale,
                                   const int32_t* block_tables, const int32_t* seq_lens,
                                   float* out, int32_t num_seqs, int32_t num_heads,
                                   int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                                   int64_t num_blocks, int32_t max_blocks_per_seq,
                                   float sm_scale) {
  pkv::DecodeArgs a;
  a.q = q;
  a.k_cache = k_cache;
  a.k_scale = k_scale;
  a.v_cache = v_cache;
  a.v_scale = v_scale;
  a.block_tables = block_tables;
  a.seq_lens = seq_lens;
  a.out = out;
  a.num_seqs = num_seqs;
  a.num_heads = num_heads;
  a.num_kv_heads = num_kv_heads;
  a.head_dim = head_dim;
  a.block_size = block_size;
  a.num_blocks = num_blocks;
  a.max_blocks_per_seq = max_blocks_per_seq;
  a.sm_scale = sm_scale;
  return a;
}

size_t pkv_quant_paged_attention_workspace_size(int32_t num_seqs, int32_t num_heads,
                                                int32_t num_kv_heads, int32_t head_dim,
                                                int32_t block_size,
                                                int32_t max_blocks_per_seq) {
  // Pointers are unknown here; size for the largest plan (16-byte aligned
  // pointers take the same or fewer splits).
  pkv::DecodeArgs a = decode_args(reinterpret_cast<const float*>(16),
                                  reinterpret_cast<const int8_t*>(16), nullptr,
                                  reinterpret_cast<const int8_t*>(16), nullptr, nullptr, nullptr,
                                  reinterpret_cast<float*>(16), num_seqs, num_heads, num_kv_heads,
                                  head_dim, block_size, 1, max_blocks_per_seq, 1.0f);
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || block_size <= 0) return 0;
  size_t fast = pkv::decode_workspace_size(a);
  a.q = reinterpret_cast<const float*>(4);  // force the generic plan
  size_t gen = pkv::decode_workspace_size(a);
  return fast > gen ? fast : gen;
}

int pkv_quant_paged_attention_kernel_launches(int32_t num_seqs, int32_t num_heads,
                                              int32_t num_kv_heads, int32_t head_dim,
                                              int32_t block_size, int32_t max_blocks_per_seq) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || block_size <= 0) return 0;
  const pkv::DecodeArgs a = decode_args(
      reinterpret_cast<const float*>(16), reinterpret_cast<const int8_t*>(16), nullptr,
      reinterpret_cast<const int8_t*>(16), nullptr, nullptr, nullptr, reinterpret_cast<float*>(16),
      num_seqs, num_heads, num_kv_heads, head_dim, block_size, 1, max_blocks_per_seq, 1.0f);
  return pkv::decode_kernel_launches(a);
}

int pkv_quant_paged_attention(const float* q, const int8_t* k_cache, const float* k_scale,
                              const int8_t* v_cache, const float* v_scale,
                              const int32_t* block_tables, const int32_t* seq_lens, float* out,
                              int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                              int32_t head_dim, int32_t block_size, int64_t num_blocks,
                              int32_t max_blocks_per_seq, float sm_scale, void* workspace,
                              size_t workspace_bytes, void* stream) {
  clear_error();
  pkv::DecodeArgs a = decode_args(q, k_cache, k_scale, v_cache, v_scale, block_tables, seq_lens,
                                  out, num_seqs, num_heads, num_kv_heads, head_dim, block_size,
                                  num_blocks, max_blocks_per_seq, sm_scale);
  int rc = check_decode(a);
  if (rc != PKV_OK) return rc;
  return pkv::launch_decode(a, workspace, workspace_bytes, as_stream(stream));
}

size_t pkv_write_to_cache_workspace_size(int64_t num_tokens, int32_t num_kv_heads) {
  return pkv::write_to_cache_workspace_size(num_tokens, num_kv_heads);
}

int pkv_write_to_cache(const void* key, const void* value, int32_t dtype, int8_t* kv_cache,
                       float* scale_cache, const int64_t* slot_mapping, int64_t num_tokens,
                       int64_t num_blocks, int32_t block_size, int32_t num_kv_heads,
                       int32_t head_dim, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (num_tokens < 0 || num_blocks < 0 || block_size <= 0 || num_kv_heads <= 0 || head_dim <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "invalid write_to_cache shape");
  if (dtype < 0 || dtype > 2)
    return fail(PKV_ERR_INVALID_ARGUMENT, "key/value must be float32, float16 or bfloat16");
  if (num_tokens > 0 && (!key || !value || !kv_cache || !scale_cache || !slot_mapping))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (num_tokens > 0x7fffffffLL)
    return fail(PKV_ERR_UNSUPPORTED, "more than 2^31 - 1 tokens in one call");
  return pkv::launch_write_to_cache(key, value, dtype, kv_cache, scale_cache, slot_mapping,
                                    num_tokens, num_blocks, block_size, num_kv_heads, head_dim,
                                    workspace, workspace_bytes, as_stream(stream));
}

static int check_rotary(int32_t head_dim, int32_t rotary_dim, int64_t num_positions) {
  if (head_dim <= 0 || head_dim > 256)
    return fail(PKV_ERR_INVALID_ARGUMENT, "head_dim must be 1 to 256");
  if (rotary_dim < 0 || rotary_dim > head_dim || rotary_dim % 2 != 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "rotary_dim must be even and at most head_dim");
  if (num_positions < 0) return fail(PKV_ERR_INVALID_ARGUMENT, "negative num_positions");
  return PKV_OK;
}

int pkv_qk_norm_rope(const void* q, const void* k, int32_t dtype, void* q_out, void* k_out,
                     const int64_t* positions, const float* rotary, const void* q_weight,
                     const void* k_weight, int32_t weights_f32, float eps, int64_t num_tokens,
                     int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                     int32_t rotary_dim, int64_t num_positions, int32_t interleaved,
                     int64_t q_token_stride, int64_t q_head_stride, int64_t k_token_stride,
                     int64_t k_head_stride, void* stream) {
  clear_error();
  if (num_tokens < 0 || num_heads < 0 || num_kv_heads < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "invalid qk_norm_rope shape");
  if (dtype < 0 || dtype > 2)
    return fail(PKV_ERR_INVALID_ARGUMENT, "q/k must be float32, float16 or bfloat16");
  int rc = check_rotary(head_dim, rotary_dim, num_positions);
  if (rc != PKV_OK) return rc;
  if (num_tokens > 0 && ((num_heads > 0 && (!q || !q_out)) || (num_kv_heads > 0 && (!k || !k_out)) ||
                         !positions || (rotary_dim > 0 && !rotary)))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  const bool norm = q_weight != nullptr || k_weight != nullptr;
  if (norm && ((num_heads > 0 && !q_weight) || (num_kv_heads > 0 && !k_weight)))
    return fail(PKV_ERR_INVALID_ARGUMENT, "q_weight and k_weight go together");
  if (num_tokens * ((int64_t)num_heads + num_kv_heads) > 0x7fffffffLL)
    return fail(PKV_ERR_UNSUPPORTED, "more than 2^31 - 1 rows in one call");
  pkv::QkNormRopeArgs a;
  a.q = q;
  a.k = num_kv_heads > 0 ? k : q;
  a.q_out = q_out;
  a.k_out = num_kv_heads > 0 ? k_out : q_out;
  a.dtype = dtype;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.k_token_stride = num_kv_heads > 0 ? k_token_stride : 0;
  a.k_head_stride = num_kv_heads > 0 ? k_head_stride : 0;
  a.positions = positions;
  a.table = rotary;
  a.q_weight = q_weight ? q_weight : k_weight;
  a.k_weight = k_weight ? k_weight : q_weight;
  a.weight_f32 = weights_f32 != 0;
  a.tokens = num_tokens;
  a.table_rows = num_positions;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.dim = head_dim;
  a.rot = rotary_dim;
  a.eps = eps;
  a.interleaved = interleaved != 0;
  return pkv::launch_qk_norm_rope(a, as_stream(stream));
}

size_t pkv_append_kv_workspace_size(int64_t num_tokens, int64_t num_blocks) {
  if (num_tokens <= 0 || num_blocks <= 0) return 0;
  return pkv::append_kv_workspace_size(num_tokens, num_blocks);
}

int pkv_append_kv(const void* key, const void* value, int32_t dtype, int8_t* kv_cache,
                  float* scale_cache, const int64_t* slot_mapping, const int64_t* positions,
                  const float* rotary, int64_t num_tokens, int64_t num_blocks, int32_t block_size,
                  int32_t num_kv_heads, int32_t head_dim, int32_t rotary_dim,
                  int64_t num_positions, int32_t interleaved, int64_t k_token_stride,
                  int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                  void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  if (num_tokens < 0 || num_blocks < 0 || num_kv_heads <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "invalid append_kv shape");
  if (block_size <= 0 || block_size > 64)
    return fail(PKV_ERR_INVALID_ARGUMENT, "supports block_size <= 64");
  if (dtype < 0 || dtype > 2)
    return fail(PKV_ERR_INVALID_ARGUMENT, "key/value must be float32, float16 or bfloat16");
  const int rc = check_rotary(head_dim, positions ? rotary_dim : 0, num_positions);
  if (rc != PKV_OK) return rc;
  if (num_tokens > 0 && (positions == nullptr) != (rotary == nullptr))
    return fail(PKV_ERR_INVALID_ARGUMENT, "positions and rotary go together");
  if (num_tokens > 0 && (!key || !value || !kv_cache || !scale_cache || !slot_mapping))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (num_tokens > 0x7ffffffeLL || num_blocks > 0x7ffffffeLL)
    return fail(PKV_ERR_UNSUPPORTED, "more than 2^31 - 2 tokens or blocks");
  pkv::AppendKvArgs a;
  a.key = key;
  a.value = value;
  a.dtype = dtype;
  a.k_token_stride = k_token_stride;
  a.k_head_stride = k_head_stride;
  a.v_token_stride = v_token_stride;
  a.v_head_stride = v_head_stride;
  a.cache = kv_cache;
  a.scales = scale_cache;
  a.slots = slot_mapping;
  a.positions = positions;
  a.table = rotary;
  a.tokens = num_tokens;
  a.blocks = num_blocks;
  a.table_rows = num_positions;
  a.block_size = block_size;
  a.kv_heads = num_kv_heads;
  a.dim = head_dim;
  a.rot = rotary_dim;
  a.interleaved = interleaved != 0;
  return pkv::launch_append_kv(a, workspace, workspace_bytes, as_stream(stream));
}

size_t pkv_prefill_attention_workspace_size(int64_t total_q, int64_t total_k, int32_t head_dim) {
  pkv::PrefillArgs a;
  a.total_q = std::max<int64_t>(total_q, 0);
  a.total_k = total_k;
  a.dim = head_dim;
  return pkv::prefill_workspace_size(a);
}

int pkv_prefill_attention_ws(const void* q, const void* k, const void* v, int32_t dtype, void* out,
                             float* lse, const int32_t* cu_seqlens_q,
                             const int32_t* cu_seqlens_k, int32_t num_seqs, int64_t total_q,
                             int64_t total_k, int32_t num_heads, int32_t num_kv_heads,
                             int32_t head_dim, int64_t q_token_stride, int64_t q_head_stride,
                             int64_t k_token_stride, int64_t k_head_stride,
                             int64_t v_token_stride, int64_t v_head_stride, float sm_scale,
                             int32_t causal, void* workspace, size_t workspace_bytes,
                             void* stream) {
  clear_error();
  if (num_seqs < 0 || total_q < 0 || total_k < 0 || num_heads <= 0 || num_kv_heads <= 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "invalid prefill shape");
  if (dtype != PKV_DTYPE_F16 && dtype != PKV_DTYPE_BF16)
    return fail(PKV_ERR_INVALID_ARGUMENT, "q/k/v must be float16 or bfloat16");
  if (head_dim <= 0 || head_dim > 128 || head_dim % 8 != 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "supports head_dim % 8 == 0, <= 128");
  if (num_heads % num_kv_heads != 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "GQA requires num_heads % num_kv_heads == 0");
  if (num_heads / num_kv_heads > 128)
    return fail(PKV_ERR_UNSUPPORTED, "more than 128 query heads per KV head");
  if (!(sm_scale > 0.0f) || sm_scale > 3.0e38f)
    return fail(PKV_ERR_INVALID_ARGUMENT, "sm_scale must be positive and finite");
  if (total_q > 0x7fffffffLL - 256 || total_k > 0x7fffffffLL - 256 ||
      num_seqs > 0x7fffffff - 256 ||
      (total_q + num_seqs + 2) * (int64_t)num_kv_heads > 0x7fffffffLL)
    return fail(PKV_ERR_UNSUPPORTED, "too many rows for one call");
  if (total_q == 0) return PKV_OK;
  if (!q || !out || !cu_seqlens_q || !cu_seqlens_k || (total_k > 0 && (!k || !v)))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  const int64_t strides[6] = {q_token_stride, q_head_stride, k_token_stride,
                              k_head_stride,  v_token_stride, v_head_stride};
  for (int i = 0; i < 6; ++i)
    if ((strides[i] <= 0 || strides[i] % 8 != 0) && (i < 2 || total_k > 0))
      return fail(PKV_ERR_INVALID_ARGUMENT, "strides must be positive multiples of 8 elements");
  if (reinterpret_cast<uintptr_t>(q) % 16 != 0 || reinterpret_cast<uintptr_t>(k) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(v) % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "q, k, v and out must be 16-byte aligned");
  pkv::PrefillArgs a;
  a.q = q;
  a.k = k;
  a.v = v;
  a.out = out;
  a.lse = lse;
  a.dtype = dtype;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.num_seqs = num_seqs;
  a.heads = num_heads;
  a.kv_heads = num_kv_heads;
  a.dim = head_dim;
  a.total_q = total_q;
  a.total_k = total_k;
  a.q_token_stride = q_token_stride;
  a.q_head_stride = q_head_stride;
  a.k_token_stride = k_token_stride;
  a.k_head_stride = k_head_stride;
  a.v_token_stride = v_token_stride;
  a.v_head_stride = v_head_stride;
  a.sm_scale = sm_scale;
  a.causal = causal != 0;
  return pkv::launch_prefill(a, workspace, workspace_bytes, as_stream(stream));
}

int pkv_prefill_attention(const void* q, const void* k, const void* v, int32_t dtype, void* out,
                          float* lse, const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                          int32_t num_seqs, int64_t total_q, int64_t total_k, int32_t num_heads,
                          int32_t num_kv_heads, int32_t head_dim, int64_t q_token_stride,
                          int64_t q_head_stride, int64_t k_token_stride, int64_t k_head_stride,
                          int64_t v_token_stride, int64_t v_head_stride, float sm_scale,
                          int32_t causal, void* stream) {
  return pkv_prefill_attention_ws(q, k, v, dtype, out, lse, cu_seqlens_q, cu_seqlens_k, num_seqs,
                                  total_q, total_k, num_heads, num_kv_heads, head_dim,
                                  q_token_stride, q_head_stride, k_token_stride, k_head_stride,
                                  v_token_stride, v_head_stride, sm_scale, causal, nullptr, 0,
                                  stream);
}

size_t pkv_shared_prefix_attention_workspace_size(int32_t num_seqs, int32_t num_heads,
                                                  int32_t num_kv_heads, int32_t head_dim,
                                                  int32_t block_size, int64_t num_blocks,
                                                  int32_t prefix_blocks,
                                                  int32_t max_blocks_per_seq) {
  if (num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || block_size <= 0 ||
      prefix_blocks < 0 || max_blocks_per_seq < 0 || num_heads % num_kv_heads != 0)
    return 0;
  pkv::SharedPrefixArgs a;
  a.own = decode_args(reinterpret_cast<const float*>(16), reinterpret_cast<const int8_t*>(16),
                      nullptr, reinterpret_cast<const int8_t*>(16), nullptr, nullptr, nullptr,
                      reinterpret_cast<float*>(16), num_seqs, num_heads, num_kv_heads, head_dim,
                      block_size, num_blocks, max_blocks_per_seq, 1.0f);
  a.prefix_table = nullptr;
  a.prefix_len = nullptr;
  a.prefix_width = prefix_blocks;
  return pkv::shared_prefix_workspace_size(a);
}

int pkv_shared_prefix_attention(const float* q, const int8_t* k_cache, const float* k_scale,
                                const int8_t* v_cache, const float* v_scale,
                                const int32_t* prefix_table, const int32_t* prefix_len,
                                const int32_t* block_tables, const int32_t* seq_lens, float* out,
                                int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                                int32_t head_dim, int32_t block_size, int64_t num_blocks,
                                int32_t prefix_blocks, int32_t max_blocks_per_seq, float sm_scale,
                                void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  pkv::SharedPrefixArgs a;
  a.own = decode_args(q, k_cache, k_scale, v_cache, v_scale, block_tables, seq_lens, out, num_seqs,
                      num_heads, num_kv_heads, head_dim, block_size, num_blocks,
                      max_blocks_per_seq, sm_scale);
  a.prefix_table = prefix_table;
  a.prefix_len = prefix_len;
  a.prefix_width = prefix_blocks;
  const int rc = check_decode(a.own);
  if (rc != PKV_OK) return rc;
  if (prefix_blocks < 0) return fail(PKV_ERR_INVALID_ARGUMENT, "invalid prefix table");
  if (head_dim > 128) return fail(PKV_ERR_INVALID_ARGUMENT, "supports head_dim % 32 == 0, <= 128");
  if (num_seqs > 0 && prefix_blocks > 0 && (!prefix_table || !prefix_len))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if ((int64_t)num_seqs * num_heads > 0x7fffffffLL - 256 ||
      (int64_t)prefix_blocks * block_size > 0x7fffffffLL - 256 ||
      num_blocks > 0x7fffffffLL / block_size)
    return fail(PKV_ERR_UNSUPPORTED, "more than 2^31 rows, prefix tokens or cache slots");
  if (reinterpret_cast<uintptr_t>(q) % 16 != 0 || reinterpret_cast<uintptr_t>(out) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(k_cache) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(v_cache) % 16 != 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "q, out and the caches must be 16-byte aligned");
  return pkv::launch_shared_prefix(a, workspace, workspace_bytes, as_stream(stream));
}

static pkv::ChunkArgs chunk_args(const void* q, int32_t dtype, const int8_t* k_cache,
                                 const float* k_scale, const int8_t* v_cache, const float* v_scale,
                                 const int32_t* tables, const int32_t* lens, const int32_t* cu,
                                 void* out, float* lse, int64_t total_q, int32_t seqs,
                                 int32_t heads, int32_t kv_heads, int32_t dim, int32_t block_size,
                                 int64_t num_blocks, int32_t width, int64_t q_tok, int64_t q_head,
                                 float sm_scale) {
  pkv::ChunkArgs a;
  a.q = q;
  a.dtype = dtype;
  a.k_cache = k_cache;
  a.k_scale = k_scale;
  a.v_cache = v_cache;
  a.v_scale = v_scale;
  a.tables = tables;
  a.lens = lens;
  a.cu = cu;
  a.out = out;
  a.lse = lse;
  a.total_q = total_q;
  a.num_blocks = num_blocks;
  a.q_token_stride = q_tok;
  a.q_head_stride = q_head;
  a.seqs = seqs;
  a.heads = heads;
  a.kv_heads = kv_heads;
  a.dim = dim;
  a.block_size = block_size;
  a.width = width;
  a.sm_scale = sm_scale;
  return a;
}

// What the two calls over new tokens and their pages have in common: sizes, and what
// they point to.
static int check_chunk_sizes(const pkv::ChunkArgs& a) {
  if (a.total_q < 0 || a.seqs < 0 || a.heads <= 0 || a.kv_heads <= 0 || a.num_blocks < 0 ||
      a.width < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "invalid query or cache shape");
  if (a.dtype < 0 || a.dtype > 2)
    return fail(PKV_ERR_INVALID_ARGUMENT, "q must be float32, float16 or bfloat16");
  if (a.heads % a.kv_heads != 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "num_heads must be a multiple of num_kv_heads");
  if (a.dim <= 0 || a.dim % 32 != 0 || a.dim > 256)
    return fail(PKV_ERR_INVALID_ARGUMENT, "supports head_dim % 32 == 0, <= 256");
  if (a.block_size <= 0 || a.block_size > 64)
    return fail(PKV_ERR_INVALID_ARGUMENT, "supports block_size <= 64");
  const int64_t most = 0x7fffffffLL - 1024;
  if (a.total_q * a.heads > most || a.total_q > most / a.heads ||
      (int64_t)a.width * a.block_size > most || a.num_blocks > most / a.block_size)
    return fail(PKV_ERR_UNSUPPORTED, "more than 2^31 rows, tokens of a table or cache slots");
  return PKV_OK;
}

static int check_chunk(const pkv::ChunkArgs& a) {
  const int rc = check_chunk_sizes(a);
  if (rc != PKV_OK) return rc;
  const int64_t per_16 = a.dtype == PKV_DTYPE_F32 ? 4 : 8;
  if (a.total_q > 0 && (a.q_token_stride % per_16 != 0 || a.q_head_stride % per_16 != 0))
    return fail(PKV_ERR_INVALID_ARGUMENT, "q's strides must be multiples of 16 bytes");
  if (reinterpret_cast<uintptr_t>(a.q) % 16 != 0 || reinterpret_cast<uintptr_t>(a.out) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(a.k_cache) % 16 != 0 ||
      reinterpret_cast<uintptr_t>(a.v_cache) % 16 != 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "q, out and the caches must be 16-byte aligned");
  if (a.total_q > 0 && (!a.q || !a.cu || (a.seqs > 0 && (!a.lens || (a.width > 0 && !a.tables)))))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (a.total_q > 0 && a.num_blocks > 0 && (!a.k_cache || !a.k_scale))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  return PKV_OK;
}

size_t pkv_chunk_attention_workspace_size(int64_t total_q, int32_t num_seqs, int32_t num_heads,
                                          int32_t num_kv_heads, int32_t head_dim,
                                          int32_t block_size, int32_t max_blocks_per_seq) {
  const pkv::ChunkArgs a = chunk_args(
      nullptr, 0, nullptr, nullptr, reinterpret_cast<const int8_t*>(16), nullptr, nullptr, nullptr,
      nullptr, nullptr, nullptr, total_q, num_seqs, num_heads, num_kv_heads, head_dim, block_size, 0,
      max_blocks_per_seq, 0, 0, 1.0f);
  if (check_chunk_sizes(a) != PKV_OK) return 0;
  return pkv::chunk_workspace_size(a);
}

int pkv_chunk_attention(const void* q, int32_t dtype, const int8_t* k_cache, const float* k_scale,
                        const int8_t* v_cache, const float* v_scale, const int32_t* block_tables,
                        const int32_t* seq_lens, const int32_t* cu_seqlens, void* out, float* lse,
                        int64_t total_q, int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
                        int32_t head_dim, int32_t block_size, int64_t num_blocks,
                        int32_t max_blocks_per_seq, int64_t q_token_stride, int64_t q_head_stride,
                        float sm_scale, void* workspace, size_t workspace_bytes, void* stream) {
  clear_error();
  pkv::ChunkArgs a =
      chunk_args(q, dtype, k_cache, k_scale, v_cache, v_scale, block_tables, seq_lens, cu_seqlens,
                 out, lse, total_q, num_seqs, num_heads, num_kv_heads, head_dim, block_size,
                 num_blocks, max_blocks_per_seq, q_token_stride, q_head_stride, sm_scale);
  const int rc = check_chunk(a);
  if (rc != PKV_OK) return rc;
  if (total_q > 0 && (!out || (num_blocks > 0 && (!v_cache || !v_scale))))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  // (an empty cache may have no address; without one the call would be for lse alone)
  if (a.v_cache == nullptr) a.v_cache = reinterpret_cast<const int8_t*>(16);
  return pkv::launch_chunk(a, workspace, workspace_bytes, as_stream(stream));
}

size_t pkv_accumulate_attention_workspace_size(int64_t total_q, int32_t num_seqs,
                                               int32_t num_heads, int32_t num_kv_heads,
                                               int32_t head_dim, int32_t block_size,
                                               int64_t num_blocks, int32_t max_blocks_per_seq,
                                               int32_t has_lse) {
  const pkv::ChunkArgs a = chunk_args(
      nullptr, 0, reinterpret_cast<const int8_t*>(16), nullptr, nullptr, nullptr, nullptr, nullptr, nullptr, nullptr,
      has_lse ? reinterpret_cast<float*>(16) : nullptr, total_q, num_seqs, num_heads, num_kv_heads,
      head_dim, block_size, 0, max_blocks_per_seq, 0, 0, 1.0f);
  if (num_blocks < 0 || check_chunk_sizes(a) != PKV_OK) return 0;
  pkv::ChunkArgs b = a;
  b.num_blocks = num_blocks;
  return pkv::accumulate_workspace_size(b);
}

int pkv_accumulate_attention(float* weights, const void* q, int32_t dtype, const int8_t* k_cache,
                             const float* k_scale, const int32_t* block_tables,
                             const int32_t* seq_lens, const int32_t* cu_seqlens, const float* lse,
                             int64_t total_q, int32_t num_seqs, int32_t num_heads,
                             int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                             int64_t num_blocks, int32_t max_blocks_per_seq, int64_t q_token_stride,
                             int64_t q_head_stride, float sm_scale, void* workspace,
                             size_t workspace_bytes, void* stream) {
  clear_error();
  const pkv::ChunkArgs a =
      chunk_args(q, dtype, k_cache, k_scale, nullptr, nullptr, block_tables, seq_lens, cu_seqlens,
                 nullptr, const_cast<float*>(lse), total_q, num_seqs, num_heads, num_kv_heads,
                 head_dim, block_size, num_blocks, max_blocks_per_seq, q_token_stride,
                 q_head_stride, sm_scale);
  const int rc = check_chunk(a);
  if (rc != PKV_OK) return rc;
  if (total_q > 0 && num_blocks > 0 && !weights)
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (total_q * num_heads > 1 << 25)
    return fail(PKV_ERR_UNSUPPORTED, "more than 2^25 rows of queries");
  return pkv::launch_accumulate(a, weights, workspace, workspace_bytes, as_stream(stream));
}

int pkv_evict_tokens(int8_t* kv_cache, float* scale_cache, float* weights,
                     const int32_t* block_tables, const int32_t* seq_lens, int32_t* lens_out,
                     int32_t* kept, int32_t num_seqs, int64_t num_blocks, int32_t block_size,
                     int32_t num_kv_heads, int32_t head_dim, int32_t max_blocks_per_seq,
                     int32_t keep, int32_t sinks, int32_t recent, void* stream) {
  clear_error();
  if (num_seqs < 0 || num_blocks < 0 || num_kv_heads <= 0 || max_blocks_per_seq < 0)
    return fail(PKV_ERR_INVALID_ARGUMENT, "invalid cache or table shape");
  if (head_dim <= 0 || head_dim > 256)
    return fail(PKV_ERR_INVALID_ARGUMENT, "head_dim must be 1 to 256");
  if (block_size <= 0 || block_size > 64)
    return fail(PKV_ERR_INVALID_ARGUMENT, "supports block_size <= 64");
  if (keep < 1 || sinks < 0 || recent < 0 || (int64_t)sinks + recent > keep)
    return fail(PKV_ERR_INVALID_ARGUMENT, "keep must be positive and hold sinks and recent");
  const int64_t most = 0x7fffffffLL - 65536;
  if ((int64_t)max_blocks_per_seq * block_size > most || num_blocks > most / block_size ||
      keep > most || (int64_t)num_seqs * (2 * (int64_t)num_kv_heads + 1) > most / 8)
    return fail(PKV_ERR_UNSUPPORTED, "more than 2^31 tokens of a table, cache slots or CTAs");
  if (num_seqs > 0 && (!seq_lens || !lens_out || !kept || (max_blocks_per_seq > 0 && !block_tables) ||
                       (num_blocks > 0 && (!kv_cache || !scale_cache || !weights))))
    return fail(PKV_ERR_INVALID_ARGUMENT, "null input or output pointer");
  if (num_seqs > 0 && lens_out == seq_lens)
    return fail(PKV_ERR_INVALID_ARGUMENT, "lens_out must not be seq_lens, which is read behind it");
  pkv::EvictArgs a;
  a.cache = kv_cache;
  a.scales = scale_cache;
  a.weights = weights;
  a.tables = block_tables;
  a.lens = seq_lens;
  a.lens_out = lens_out;
  a.kept = kept;
  a.num_blocks = num_blocks;
  a.seqs = num_seqs;
  a.block_size = block_size;
  a.kv_heads = num_kv_heads;
  a.dim = head_dim;
  a.width = max_blocks_per_seq;
  a.keep = keep;
  a.sinks = sinks;
  a.recent = recent;
  return pkv::launch_evict(a, as_stream(stream));
}

}  // extern "C"
