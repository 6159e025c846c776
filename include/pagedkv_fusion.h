/*
 * PagedKV-Fusion for NVIDIA B200 (sm_100a) -- C ABI of libpagedkv_sm100.so.
 *
 * This is the drop-in boundary that replaces the reference's pybind11
 * module (csrc/bindings.cpp:14-26, module pagedkv_fusion._C) and the torch /
 * library calls around it.  Every entry point takes plain device pointers
 * and sizes, enqueues its kernels on `stream` (a cudaStream_t; NULL is the
 * legacy default stream), never synchronizes, and returns a status code.
 * On failure the message of the last error on the calling thread is
 * available from pkv_last_error_string().
 *
 * Layouts (unchanged from the reference, csrc/quant_paged_attention.cu:4-8):
 *   paged cache   int8  [num_blocks, block_size, num_kv_heads, head_dim]
 *   scales        fp32  [num_blocks, num_kv_heads]
 *   block_tables  int32 [num_seqs, max_blocks_per_seq]  (-1 = unused)
 *   seq_lens      int32 [num_seqs]
 * All arrays are C-contiguous.  Kernels that find bad data on the device (a
 * block id outside [0, num_blocks), a slot outside the cache) skip it and
 * record a code in a per-device error word read by pkv_read_device_error();
 * they never trap.
 */
#ifndef PAGEDKV_FUSION_H
#define PAGEDKV_FUSION_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* Status codes returned by every entry point. */
#define PKV_OK 0
#define PKV_ERR_INVALID_ARGUMENT 1 /* shape / dtype / pointer precondition */
#define PKV_ERR_UNSUPPORTED 2      /* valid but outside this build's envelope */
#define PKV_ERR_WORKSPACE 3        /* workspace missing or too small */
#define PKV_ERR_CUDA 4             /* a CUDA runtime call or launch failed */
#define PKV_ERR_DEVICE_INPUT 5     /* pkv_read_device_error found bad input */

/* Device error codes recorded by kernels. */
#define PKV_DEVERR_NONE 0
#define PKV_DEVERR_BAD_BLOCK_ID 1
#define PKV_DEVERR_WAIT_TIMEOUT 2
#define PKV_DEVERR_BAD_SLOT 3
#define PKV_DEVERR_SEQ_TOO_LONG 4 /* seq_len beyond the block-table width */
#define PKV_DEVERR_BAD_POSITION 5 /* position outside the rotary table */
#define PKV_DEVERR_BAD_SEQLENS 6  /* cu_seqlens not ascending within the tensor */

/* Element types of floating-point KV inputs. */
#define PKV_DTYPE_F32 0
#define PKV_DTYPE_F16 1
#define PKV_DTYPE_BF16 2

/* Message of the last failing call on this thread ("" if none). */
const char *pkv_last_error_string(void);

/* ABI version: major * 10000 + minor * 100 + patch. */
int pkv_version(void);

/*
 * Reads (and, if `reset` != 0, clears) the error word of the current
 * device.  Synchronizes the device.  *code receives a PKV_DEVERR_* value.
 * Returns PKV_ERR_DEVICE_INPUT when the word was non-zero.
 */
int pkv_read_device_error(int32_t *code, int reset);

/*
 * Fused eviction score per KV block (lower = evict first):
 *   score[b] = w_recency*recency[b] + w_frequency*frequency[b]
 *            + w_attention*mean(attn_weights[b, t] over valid t)
 * bit-identical to pagedkv_fusion/reference.py:38-71 (NumPy float32).
 * valid_mask holds one byte per token (non-zero = valid).
 * Replaces eviction_scores_cuda (csrc/eviction_score.cu:97-136) bound at
 * csrc/bindings.cpp:16-20.
 */
int pkv_eviction_scores(const float *recency, const float *frequency,
                        const float *attn_weights, const uint8_t *valid_mask,
                        float *scores, int64_t num_blocks, int32_t block_size,
                        float w_recency, float w_frequency, float w_attention,
                        void *stream);

/*
 * Indices of the k lowest scores, ascending by (score, block id), -0.0 ==
 * +0.0, NaN last; min(k, num_blocks) int64 entries are written.  Matches
 * select_eviction_candidates_ref (pagedkv_fusion/reference.py:74-81) and
 * replaces torch.topk in pagedkv_fusion/ops.py:97-98.
 */
size_t pkv_eviction_select_workspace_size(int64_t num_blocks, int64_t k);
int pkv_eviction_select(const float *scores, int64_t num_blocks, int64_t k,
                        int64_t *out_indices, void *workspace,
                        size_t workspace_bytes, void *stream);

/*
 * Score and select in one call: writes scores (if non-NULL) and the
 * min(k, num_blocks) selected block ids.  Composition of
 * ops.eviction_scores + ops.select_eviction_candidates
 * (pagedkv_fusion/ops.py:63-98).
 */
size_t pkv_eviction_scores_select_workspace_size(int64_t num_blocks, int64_t k);
int pkv_eviction_scores_select(const float *recency, const float *frequency,
                               const float *attn_weights,
                               const uint8_t *valid_mask, float *scores,
                               int64_t num_blocks, int32_t block_size,
                               float w_recency, float w_frequency,
                               float w_attention, int64_t k,
                               int64_t *out_indices, void *workspace,
                               size_t workspace_bytes, void *stream);

/*
 * Sharded eviction (one rank's block range [id_offset, id_offset +
 * num_blocks)): the min(k, num_blocks) smallest candidate keys
 * (orderable(score) << 32 | (id_offset + i)), ascending.  No reference
 * counterpart: the reference is single-GPU (integration/vllm/
 * pagedkv_fusion_backend.py:23); these keys are what ranks exchange.
 */
int pkv_eviction_local_candidates(const float *scores, int64_t num_blocks,
                                  int64_t k, int64_t id_offset,
                                  uint64_t *out_keys, void *workspace,
                                  size_t workspace_bytes, void *stream);

/*
 * Global selection from gathered candidate keys: the block ids of the k
 * smallest keys, ascending.  Identical on every rank for identical input.
 */
size_t pkv_eviction_merge_workspace_size(int64_t num_keys, int64_t k);
int pkv_eviction_merge(const uint64_t *keys, int64_t num_keys, int64_t k,
                       int64_t *out_indices, void *workspace,
                       size_t workspace_bytes, void *stream);

/*
 * Symmetric per-(block, head) INT8 quantization of kv [num_blocks,
 * block_size, num_kv_heads, head_dim] (PKV_DTYPE_*): q int8 of the same
 * shape, scale fp32 [num_blocks, num_kv_heads].  Codes bit-identical to
 * quantize_kv_per_block_ref (pagedkv_fusion/reference.py:88-105); replaces
 * the torch ops of pagedkv_fusion/quantize.py:15-31.
 */
int pkv_quantize_kv_per_block(const void *kv, int32_t kv_dtype, int8_t *q,
                              float *scale, int64_t num_blocks,
                              int32_t block_size, int32_t num_kv_heads,
                              int32_t head_dim, void *stream);

/*
 * Per-token attention statistics derived from the keys, the input the
 * eviction score's attention term reads: for a K pool [num_blocks,
 * block_size, num_kv_heads, 128] (float32 / float16 / bfloat16, dtype codes
 * as for quantization) and one query vector per KV head q [num_kv_heads,
 * 128] float32,
 *   s_h[b, t]  = sm_scale * (q_h . K[b, t, h, :])
 *   attn[b, t] = mean_h exp(s_h[b, t] - max over the pool of s_h)
 * written to attn [num_blocks, block_size] float32, in (0, 1].  block_size
 * 16 or 32.  The workspace holds the logits and the per-head maxima.  No
 * counterpart in the reference, whose eviction statistics are given arrays
 * (pagedkv_fusion/reference.py:38-71); the definition is this library's.
 */
size_t pkv_attention_stats_workspace_size(int64_t num_blocks,
                                          int32_t block_size,
                                          int32_t num_kv_heads);
int pkv_attention_stats(const void *k, int32_t k_dtype, const float *q,
                        float *attn, int64_t num_blocks, int32_t block_size,
                        int32_t num_kv_heads, int32_t head_dim, float sm_scale,
                        void *workspace, size_t workspace_bytes, void *stream);

/*
 * pkv_quantize_kv_per_block for the blocks whose skip[b] byte is zero;
 * blocks with a nonzero byte are neither read nor written (their codes and
 * scale keep whatever they held).  Quantizes the blocks that survive an
 * eviction without touching the evicted ones.  No counterpart in the
 * reference: its end-to-end demo (scripts/run_end_to_end_demo.py:74-116)
 * scores and selects, then quantizes every block and decodes over the
 * unchanged tables.
 */
int pkv_quantize_kv_per_block_except(const void *kv, int32_t kv_dtype,
                                     const uint8_t *skip, int8_t *q,
                                     float *scale, int64_t num_blocks,
                                     int32_t block_size, int32_t num_kv_heads,
                                     int32_t head_dim, void *stream);

/*
 * mask[0 .. num_blocks) = 0, then mask[id - id_offset] = 1 for every id in
 * ids[0 .. num_ids) that falls in [id_offset, id_offset + num_blocks): the
 * local eviction mask of a rank holding blocks id_offset.. from the global
 * ids a (sharded) selection returned.  No counterpart in the reference.
 */
int pkv_mark_blocks(const int64_t *ids, int64_t num_ids, int64_t id_offset,
                    int64_t num_blocks, uint8_t *mask, void *stream);

/*
 * Removes evicted blocks from block tables.  For sequence s the first
 * ceil(seq_lens[s] / block_size) entries (clamped to the table width;
 * PKV_DEVERR_SEQ_TOO_LONG beyond it) are its pages, the last holding the
 * remainder; pages whose block has evicted[id] != 0 are dropped, the rest
 * are written in order to tables_out (row padded with -1) and lens_out[s]
 * is the number of tokens they hold.  Every kept page but the last is full,
 * so (tables_out, lens_out) is a valid input to pkv_quant_paged_attention.
 * Ids outside [0, num_blocks) are kept.  No counterpart in the reference.
 */
int pkv_compact_block_tables(const int32_t *block_tables,
                             const int32_t *seq_lens, const uint8_t *evicted,
                             int32_t *tables_out, int32_t *lens_out,
                             int32_t num_seqs, int32_t max_blocks_per_seq,
                             int32_t block_size, int64_t num_blocks,
                             void *stream);

/*
 * Decode-step attention over the INT8 paged cache: out[s, h, :] =
 * softmax(q[s, h] . K^T * sm_scale) V over the seq_lens[s] tokens reached
 * through block_tables[s], dequantized with the per-(block, head) scales;
 * GQA maps head h to kv head h / (num_heads / num_kv_heads).  A sequence of
 * length 0 yields zeros.  Replaces quant_paged_attention_cuda
 * (csrc/quant_paged_attention.cu:172-225) bound at csrc/bindings.cpp:21-25.
 * Envelope: head_dim % 32 == 0 and <= 256, block_size <= 64,
 * num_heads % num_kv_heads == 0.  The workspace holds the partial results
 * of sequences whose pages are split across CTAs, and one arrival counter
 * per (sequence, KV-head group); it needs no initialisation (the counters
 * carry a per-launch tag) and the call issues no memset.
 */
size_t pkv_quant_paged_attention_workspace_size(
    int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t block_size, int32_t max_blocks_per_seq);
int pkv_quant_paged_attention(const float *q, const int8_t *k_cache,
                              const float *k_scale, const int8_t *v_cache,
                              const float *v_scale, const int32_t *block_tables,
                              const int32_t *seq_lens, float *out,
                              int32_t num_seqs, int32_t num_heads,
                              int32_t num_kv_heads, int32_t head_dim,
                              int32_t block_size, int64_t num_blocks,
                              int32_t max_blocks_per_seq, float sm_scale,
                              void *workspace, size_t workspace_bytes,
                              void *stream);

/*
 * Number of kernels one pkv_quant_paged_attention call with these shapes
 * launches on its stream (16-byte aligned pointers): 1 for the persistent
 * stream kernel (up to 1,024 sequences with head_dim 128, block_size 16 or
 * 32 and a GQA group of 1, or 2/4/8 at block_size 32), 2 for the
 * tensor-core GQA kernel (block_size 16, groups of 2/4/8) or the split-K
 * kernel, each with its combine.  Lets a caller account for launches
 * without a profiler.  No counterpart in the reference.
 */
int pkv_quant_paged_attention_kernel_launches(int32_t num_seqs, int32_t num_heads,
                                              int32_t num_kv_heads, int32_t head_dim,
                                              int32_t block_size,
                                              int32_t max_blocks_per_seq);

/*
 * pkv_quant_paged_attention without a workspace argument, for callers that
 * cannot allocate device memory (a plugin whose host framework hands it
 * only input/output pointers and forbids allocation, or a serving path that
 * must not pay cudaMalloc's implicit synchronization).  Identical results.
 * The split-K partials live in a fixed pkv_noalloc_scratch_bytes() (32 MiB)
 * array inside the library, held on every GPU that loads the library until
 * exit; calls needing more are rejected with PKV_ERR_UNSUPPORTED.  The
 * first call on a device looks up the array's address (make it before any
 * stream capture).  Calls share the array: calls overlapping on the GPU
 * race.  No counterpart in the reference.
 */
size_t pkv_noalloc_scratch_bytes(void);
int pkv_quant_paged_attention_noalloc(const float *q, const int8_t *k_cache,
                                      const float *k_scale,
                                      const int8_t *v_cache,
                                      const float *v_scale,
                                      const int32_t *block_tables,
                                      const int32_t *seq_lens, float *out,
                                      int32_t num_seqs, int32_t num_heads,
                                      int32_t num_kv_heads, int32_t head_dim,
                                      int32_t block_size, int64_t num_blocks,
                                      int32_t max_blocks_per_seq,
                                      float sm_scale, void *stream);

/*
 * Quantize new K/V tokens and scatter them into the vLLM-shaped cache
 * kv_cache int8 [2, num_blocks, block_size, num_kv_heads, head_dim] and
 * scale_cache fp32 [2, num_blocks, num_kv_heads].  The tokens of one call
 * that land in the same block are quantized together and their scale
 * overwrites that block's scale, as PagedKVFusionBackend.write_to_cache
 * (integration/vllm/pagedkv_fusion_backend.py:63-95) does.
 */
size_t pkv_write_to_cache_workspace_size(int64_t num_tokens,
                                         int32_t num_kv_heads);
int pkv_write_to_cache(const void *key, const void *value, int32_t dtype,
                       int8_t *kv_cache, float *scale_cache,
                       const int64_t *slot_mapping, int64_t num_tokens,
                       int64_t num_blocks, int32_t block_size,
                       int32_t num_kv_heads, int32_t head_dim, void *workspace,
                       size_t workspace_bytes, void *stream);

/*
 * Per-head RMS norm and rotary position of queries and keys in one pass:
 *   n = x / sqrt(mean(x^2) + eps) * weight     (left out when both weights
 *                                               are NULL)
 *   a' = a cos - b sin, b' = b cos + a sin     over the first rotary_dim
 * channels of each head, pairs (i, i + rotary_dim / 2), or (2i, 2i + 1) when
 * `interleaved`; later channels are not rotated.  q [num_tokens, num_heads,
 * head_dim] and k [num_tokens, num_kv_heads, head_dim] (PKV_DTYPE_*) have
 * their own token and head strides, in elements, and contiguous channels;
 * q_out and k_out are contiguous and do not overlap the inputs.  rotary is
 * float32 [num_positions, rotary_dim]: rotary_dim / 2 cosines, then as many
 * sines.  positions int64 [num_tokens]; a position outside the table records
 * PKV_DEVERR_BAD_POSITION and its token's rows become zero.  The weights
 * [head_dim] are float32 when weights_f32, else of the inputs' type.  The
 * arithmetic is in 32 bits, rounded once to the output.  num_kv_heads may be
 * 0 (k unused).  head_dim <= 256, rotary_dim even and <= head_dim.
 */
int pkv_qk_norm_rope(const void *q, const void *k, int32_t dtype, void *q_out,
                     void *k_out, const int64_t *positions,
                     const float *rotary, const void *q_weight,
                     const void *k_weight, int32_t weights_f32, float eps,
                     int64_t num_tokens, int32_t num_heads,
                     int32_t num_kv_heads, int32_t head_dim,
                     int32_t rotary_dim, int64_t num_positions,
                     int32_t interleaved, int64_t q_token_stride,
                     int64_t q_head_stride, int64_t k_token_stride,
                     int64_t k_head_stride, void *stream);

/*
 * Appends keys and values to the vLLM-shaped cache kv_cache int8 [2,
 * num_blocks, block_size, num_kv_heads, head_dim] / scale_cache fp32 [2,
 * num_blocks, num_kv_heads], keeping the earlier tokens of a started page
 * readable (pkv_write_to_cache replaces a page's scale by that of the
 * call's tokens).  Keys are rotated on the way (as pkv_qk_norm_rope, each
 * 32-bit product and sum rounded) when positions and rotary are given.  Per
 * (page, head, K or V) with new tokens:
 *   step  = absmax(new values) / 127     (0 when that is 0 or NaN)
 *   scale = step, or 1 when step is 0    if the call writes offset 0: a page
 *                                        begun by this call
 *         = max(old scale, step)         otherwise
 *   codes at offsets below the lowest one written become
 *   rint(code * (old scale / scale)) where the scale grew; new codes are
 *   rint(value / scale), clamped to [-127, 127]; other codes stay.
 * slot_mapping int64 [num_tokens] holds block * block_size + offset; slot -1
 * is padding and skipped; other slots outside the cache record
 * PKV_DEVERR_BAD_SLOT and are skipped.  Of equal slots the last token
 * counts.  key and value have token and head strides, in elements.
 * block_size <= 64, head_dim <= 256.
 */
size_t pkv_append_kv_workspace_size(int64_t num_tokens, int64_t num_blocks);
int pkv_append_kv(const void *key, const void *value, int32_t dtype,
                  int8_t *kv_cache, float *scale_cache,
                  const int64_t *slot_mapping, const int64_t *positions,
                  const float *rotary, int64_t num_tokens, int64_t num_blocks,
                  int32_t block_size, int32_t num_kv_heads, int32_t head_dim,
                  int32_t rotary_dim, int64_t num_positions,
                  int32_t interleaved, int64_t k_token_stride,
                  int64_t k_head_stride, int64_t v_token_stride,
                  int64_t v_head_stride, void *workspace,
                  size_t workspace_bytes, void *stream);

/*
 * Attention over packed prompts: out[i, h, :] = softmax(sm_scale * q[i, h] .
 * K^T) V over the keys of token i's sequence, GQA as in decode, fp32
 * accumulation and softmax, probabilities rounded to the inputs' type for
 * the second product.  q, out [total_q, num_heads, head_dim], k, v [total_k,
 * num_kv_heads, head_dim] (PKV_DTYPE_F16 or PKV_DTYPE_BF16); sequence s is
 * rows cu_seqlens_q[s] .. cu_seqlens_q[s + 1] of q and cu_seqlens_k[s] ..
 * cu_seqlens_k[s + 1] of k and v (int32 [num_seqs + 1]).  Under `causal`,
 * token i of a sequence of Lq tokens and Lk keys sees keys j <= i + Lk - Lq
 * (a chunk of a longer prompt is a sequence with more keys than tokens).
 * Rows that see no key, and rows of q behind the last sequence or in front of
 * the first, become zero, with lse -inf; lse (nullable, float32 [total_q, num_heads]) is the natural
 * logarithm of the softmax denominator.  Values of keys that a row does not
 * see, NaN and infinities included, do not reach it.  Token and head strides
 * are in elements, multiples of 8, pointers 16-byte aligned, channels
 * contiguous, out contiguous.  head_dim a multiple of 8 up to 128, at most
 * 128 query heads per KV head, sm_scale > 0.  cu_seqlens that do not ascend
 * within the tensors record PKV_DEVERR_BAD_SEQLENS and are cut to the tensors,
 * those of q also to the largest entry before them; a sequence whose keys end
 * before they begin has none.
 */
int pkv_prefill_attention(const void *q, const void *k, const void *v,
                          int32_t dtype, void *out, float *lse,
                          const int32_t *cu_seqlens_q,
                          const int32_t *cu_seqlens_k, int32_t num_seqs,
                          int64_t total_q, int64_t total_k, int32_t num_heads,
                          int32_t num_kv_heads, int32_t head_dim,
                          int64_t q_token_stride, int64_t q_head_stride,
                          int64_t k_token_stride, int64_t k_head_stride,
                          int64_t v_token_stride, int64_t v_head_stride,
                          float sm_scale, int32_t causal, void *stream);

/*
 * The same with a workspace, which needs no initialisation.  The tensor cores
 * cut the bits of a product that the fp32 sum cannot hold: a sum over n keys
 * whose terms have one sign comes out too small by up to 6.6e-9 n of itself.
 * Sums are therefore rounded to nearest every 16,384 keys, which ends the loss
 * at 1.1e-4: with head_dim up to 64 in the call above too, above that where the
 * call has a workspace.  Its size is 0 for calls that need none (head_dim up to
 * 64, or no more than 16,384 keys in all).  workspace may be NULL.
 */
size_t pkv_prefill_attention_workspace_size(int64_t total_q, int64_t total_k,
                                            int32_t head_dim);
int pkv_prefill_attention_ws(const void *q, const void *k, const void *v,
                             int32_t dtype, void *out, float *lse,
                             const int32_t *cu_seqlens_q,
                             const int32_t *cu_seqlens_k, int32_t num_seqs,
                             int64_t total_q, int64_t total_k,
                             int32_t num_heads, int32_t num_kv_heads,
                             int32_t head_dim, int64_t q_token_stride,
                             int64_t q_head_stride, int64_t k_token_stride,
                             int64_t k_head_stride, int64_t v_token_stride,
                             int64_t v_head_stride, float sm_scale,
                             int32_t causal, void *workspace,
                             size_t workspace_bytes, void *stream);

/*
 * Decode-step attention for a batch that shares a prefix: as
 * pkv_quant_paged_attention over the tokens [prefix | own tokens] of each
 * sequence, where the prefix_len[0] tokens of the prefix are reached through
 * prefix_table (int32 [prefix_blocks], pages shared by every sequence, the
 * last one possibly partial) and the sequence's own seq_lens[s] tokens through
 * block_tables[s].  The prefix's pages are read once for the batch.  A
 * sequence without any token yields zeros.  A prefix_len or a sequence's length
 * beyond its table records PKV_DEVERR_SEQ_TOO_LONG and is cut to it; tokens on
 * a page outside the cache record PKV_DEVERR_BAD_BLOCK_ID and are not attended.
 * Envelope: head_dim % 32 == 0 and <= 128, block_size <= 64, num_heads %
 * num_kv_heads == 0; q, out and the caches 16-byte aligned.  prefix_blocks and
 * max_blocks_per_seq may be 0.  The workspace holds the partial results and
 * needs no initialisation.
 */
size_t pkv_shared_prefix_attention_workspace_size(
    int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t block_size, int64_t num_blocks, int32_t prefix_blocks,
    int32_t max_blocks_per_seq);
int pkv_shared_prefix_attention(
    const float *q, const int8_t *k_cache, const float *k_scale,
    const int8_t *v_cache, const float *v_scale, const int32_t *prefix_table,
    const int32_t *prefix_len, const int32_t *block_tables,
    const int32_t *seq_lens, float *out, int32_t num_seqs, int32_t num_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
    int64_t num_blocks, int32_t prefix_blocks, int32_t max_blocks_per_seq,
    float sm_scale, void *workspace, size_t workspace_bytes, void *stream);

/*
 * Attention of new tokens over the INT8 paged cache that they were appended to
 * (one token, a few, or a chunk of a prompt of each sequence): out[i, h, :] =
 * softmax(sm_scale * q[i, h] . K^T) V over the keys j <= i + L - Lq of token i's
 * sequence, where sequence s is rows cu_seqlens[s] .. cu_seqlens[s + 1] (Lq) of
 * q and out [total_q, num_heads, head_dim] (PKV_DTYPE_*) and its seq_lens[s] (L)
 * cached tokens, the new ones last, are reached through block_tables[s]; caches,
 * scales and GQA as in pkv_quant_paged_attention.  Rows that see no key, and rows
 * behind the last sequence or in front of the first, become zero, with lse -inf;
 * lse (nullable, float32 [total_q, num_heads]) is the natural logarithm of the
 * softmax denominator.  Lengths beyond the table record PKV_DEVERR_SEQ_TOO_LONG
 * and are cut to it; tokens on a page outside the cache record
 * PKV_DEVERR_BAD_BLOCK_ID and are not attended; cu_seqlens that do not ascend
 * within the tensor record PKV_DEVERR_BAD_SEQLENS and are cut as in
 * pkv_prefill_attention.  head_dim a multiple of 32 up to 256, block_size <= 64;
 * q's strides, in elements, of multiples of 16 bytes, channels contiguous, q, out
 * and the caches 16-byte aligned, out contiguous.  The workspace needs no
 * initialisation.
 */
size_t pkv_chunk_attention_workspace_size(int64_t total_q, int32_t num_seqs,
                                          int32_t num_heads,
                                          int32_t num_kv_heads, int32_t head_dim,
                                          int32_t block_size,
                                          int32_t max_blocks_per_seq);
int pkv_chunk_attention(const void *q, int32_t dtype, const int8_t *k_cache,
                        const float *k_scale, const int8_t *v_cache,
                        const float *v_scale, const int32_t *block_tables,
                        const int32_t *seq_lens, const int32_t *cu_seqlens,
                        void *out, float *lse, int64_t total_q, int32_t num_seqs,
                        int32_t num_heads, int32_t num_kv_heads, int32_t head_dim,
                        int32_t block_size, int64_t num_blocks,
                        int32_t max_blocks_per_seq, int64_t q_token_stride,
                        int64_t q_head_stride, float sm_scale, void *workspace,
                        size_t workspace_bytes, void *stream);

/*
 * Adds to weights (float32 [num_blocks, block_size], one per cached token) what the
 * call's tokens attend to it: the sum over tokens i and the mean over heads h of
 * exp(sm_scale * q[i, h] . k_j - lse[i, h]), tokens, keys and masks as in
 * pkv_chunk_attention.  lse (float32 [total_q, num_heads], contiguous) is what that
 * call returned, or NULL: then it is computed first.  A row whose lse is -inf adds
 * nothing; NaN reaches the weights of the keys that its row sees.  Pages may be in
 * several tables; the result does not depend on the order of execution (sums meet as
 * integers, in steps of 2^-37).  total_q * num_heads <= 2^25.
 */
size_t pkv_accumulate_attention_workspace_size(
    int64_t total_q, int32_t num_seqs, int32_t num_heads, int32_t num_kv_heads,
    int32_t head_dim, int32_t block_size, int64_t num_blocks,
    int32_t max_blocks_per_seq, int32_t has_lse);
int pkv_accumulate_attention(float *weights, const void *q, int32_t dtype,
                             const int8_t *k_cache, const float *k_scale,
                             const int32_t *block_tables, const int32_t *seq_lens,
                             const int32_t *cu_seqlens, const float *lse,
                             int64_t total_q, int32_t num_seqs, int32_t num_heads,
                             int32_t num_kv_heads, int32_t head_dim,
                             int32_t block_size, int64_t num_blocks,
                             int32_t max_blocks_per_seq, int64_t q_token_stride,
                             int64_t q_head_stride, float sm_scale,
                             void *workspace, size_t workspace_bytes,
                             void *stream);

/*
 * Evicts single tokens.  Of a sequence of L > keep tokens stay the first `sinks`, the
 * last `recent` and the heaviest of the others by `weights` (of equal ones the
 * earlier; NaN is heaviest), `keep` in all.  They move, in order, to the front of the
 * sequence's pages, in place, in kv_cache int8 [2, num_blocks, block_size,
 * num_kv_heads, head_dim], scale_cache fp32 [2, num_blocks, num_kv_heads] and weights
 * fp32 [num_blocks, block_size].  A page's new scale is the largest old scale of the
 * tokens it now holds, per KV head, K and V apart; codes become rint(code * (old /
 * new)) where old < new, clamped to -127 .. 127 where old is negative.  The slots
 * that the sequence no longer uses keep their codes and get weight 0.  lens_out int32
 * [num_seqs] (not seq_lens itself: both are read at the end) receives the new lengths,
 * kept int32 [num_seqs, keep] the old places of the tokens that stay, ascending, then -1.
 * Sequences of at most `keep` tokens stay as they are, and so do those with a page
 * outside the cache (PKV_DEVERR_BAD_BLOCK_ID; their row of kept is -1).  The pages of a
 * sequence that is cut must not be in another sequence's table, nor twice in its own.
 * keep >= 1, sinks + recent <= keep, block_size <= 64, head_dim <= 256.
 */
int pkv_evict_tokens(int8_t *kv_cache, float *scale_cache, float *weights,
                     const int32_t *block_tables, const int32_t *seq_lens,
                     int32_t *lens_out, int32_t *kept, int32_t num_seqs,
                     int64_t num_blocks, int32_t block_size,
                     int32_t num_kv_heads, int32_t head_dim,
                     int32_t max_blocks_per_seq, int32_t keep, int32_t sinks,
                     int32_t recent, void *stream);

#ifdef __cplusplus
}
#endif

#endif /* PAGEDKV_FUSION_H */
