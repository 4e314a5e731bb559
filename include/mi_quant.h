/*
 * mi_quant.h -- C ABI of libmi_attn.so for a K/V cache held in 8 bits: rows
 * quantised as they are written, read back, and attended over by single
 * tokens and by chunks of prompts. No counterpart in the reference.
 *
 * The rules of mi_attn.h hold: nothing here synchronises, allocates device
 * memory or records memset/memcpy nodes; element strides; MI_* status codes;
 * mi_last_error().
 *
 * The cache. key_cache and value_cache hold one byte a value, [num_blocks,
 * block_size, num_kv_heads, head_dim] through the same block, token and head
 * strides (head_dim contiguous, everything a multiple of 8 bytes); key_scales
 * and value_scales are float32 [num_blocks, num_kv_heads] through the same
 * block and head strides. A byte stands for code * scale:
 *   MI_CODE_E4M3  float8 e4m3 (no infinity, largest 448; NaN is 0x7f / 0xff)
 *   MI_CODE_INT8  -127 .. 127
 * head_dim is a power of two from 16 to 256, block_size a power of two
 * (MI_ERR_UNSUPPORTED / MI_ERR_INVALID_ARGUMENT otherwise). The readers take
 * any scales that are not negative (a NaN makes NaN of what it scales);
 * mi_quant_append writes powers of two.
 */
#ifndef MI_QUANT_H_
#define MI_QUANT_H_

#include <stdint.h>

#include "mi_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

#define MI_CODE_E4M3 0
#define MI_CODE_INT8 1

/*
 * Write the rows keys / values [num_tokens, num_kv_heads, head_dim] (dtype) at
 * slots (block * block_size + offset; negative or too large ones are skipped;
 * int32, or int64 where slots_are_int64). For every block that the call writes
 * to and every KV head, K and V apart, with `first` the lowest offset written:
 *   need = the least power of two s >= 2^-126 with |x| <= M s for every finite
 *          value x written (M: 448 or 127)
 *   s'   = need where first is 0, else max(s, need), s the block's scale
 *   rows below first (where first > 0): code' = round(code * (s / s'))
 *   written rows:                       code  = round(x / s')
 * rounding to nearest, ties to even. So a row at offset 0 begins its block
 * anew, and the rows of a block are written in order of their offsets, in as
 * many calls as it takes. Powers of two make the rounding of rows that are
 * held exact in e4m3 until they leave its normal range, and every dequantised
 * value a bf16 (and float32) number. Other rows of the block keep their bytes.
 * A value that is not finite is held as NaN; int8 has none, there the scale
 * becomes NaN, until the block begins anew. Of rows with the same slot one is
 * written, whichever.
 *
 * plan: what mi_quant_append_plan made of these slots (it serves every layer
 * of a step), or NULL, with at most 1024 tokens (the faster of the two up to
 * some hundred). block_size at most 1024. keys and values are 16-byte aligned,
 * with strides of whole 16-byte vectors.
 */
int32_t mi_quant_append(const void* keys, int64_t key_token_stride, int64_t key_head_stride,
                        const void* values, int64_t value_token_stride,
                        int64_t value_head_stride, void* key_cache, void* value_cache,
                        int64_t cache_block_stride, int64_t cache_token_stride,
                        int64_t cache_head_stride, float* key_scales, float* value_scales,
                        int64_t scale_block_stride, int64_t scale_head_stride,
                        const void* slots, int32_t slots_are_int64, const void* plan,
                        int64_t plan_bytes, int32_t num_tokens, int32_t num_kv_heads,
                        int32_t head_dim, int32_t block_size, int32_t num_blocks, int32_t dtype,
                        int32_t code, void* stream);

/*
 * The blocks that these slots write to, and their rows, found on the device.
 * plan: mi_quant_append_plan_bytes() bytes (4 for each position of the pool, and
 * 4 block_size + 8 for each token), 8-byte aligned, no initialisation.
 */
int64_t mi_quant_append_plan_bytes(int32_t num_tokens, int32_t block_size, int32_t num_blocks);
int32_t mi_quant_append_plan(const void* slots, int32_t slots_are_int64, int32_t num_tokens,
                             int32_t block_size, int32_t num_blocks, void* plan,
                             int64_t plan_bytes, void* stream);

/*
 * Read back: output row i (of total_rows) is position i - cu_seqlens_k[r] of
 * the request r that owns it, through its block table, as dtype:
 * round(code * scale). Rows of blocks outside the pool or the table are zeros.
 * key_out / value_out: [total_rows, num_kv_heads, head_dim], contiguous.
 */
int32_t mi_quant_gather(const void* key_cache, const void* value_cache,
                        int64_t cache_block_stride, int64_t cache_token_stride,
                        int64_t cache_head_stride, const float* key_scales,
                        const float* value_scales, int64_t scale_block_stride,
                        int64_t scale_head_stride, const int32_t* block_tables,
                        int64_t block_table_stride, int32_t block_table_width,
                        const int32_t* cu_seqlens_k, int32_t num_requests, int32_t total_rows,
                        void* key_out, void* value_out, int32_t num_kv_heads, int32_t head_dim,
                        int32_t block_size, int32_t num_blocks, int32_t dtype, int32_t code,
                        void* stream);

/*
 * Decode attention: mi_paged_decode over an 8-bit cache, one query row
 * (dtype) per sequence. mi_quant_decode_plan lays out a step on the device
 * from context_lens and zeroes counters (num_seqs * num_kv_heads int32);
 * mi_quant_decode runs a layer with the plan and leaves the counters zero, so
 * one plan serves all layers. Calls that may run concurrently need workspaces
 * and counters of their own. A negative or too large block id is masked;
 * sequences of context 0 give zeros; a NaN score makes its row NaN.
 *
 * plan: mi_quant_decode_plan_bytes() bytes, 32-byte aligned; workspace:
 * mi_quant_decode_workspace_bytes() bytes, 16-byte aligned, no
 * initialisation. At most 4096 sequences (MI_ERR_UNSUPPORTED). query and out
 * 16-byte aligned with strides of whole 16-byte vectors.
 */
int64_t mi_quant_decode_plan_bytes(int32_t num_seqs, int32_t num_kv_heads);
int64_t mi_quant_decode_workspace_bytes(int32_t num_seqs, int32_t num_q_heads,
                                        int32_t num_kv_heads, int32_t head_dim);
int32_t mi_quant_decode_plan(const int32_t* context_lens, int32_t num_seqs, int32_t num_q_heads,
                             int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                             int32_t block_table_width, int32_t dtype, void* plan,
                             int64_t plan_bytes, int32_t* counters, void* stream);
int32_t mi_quant_decode(const void* query, int64_t q_token_stride, int64_t q_head_stride,
                        const void* key_cache, const void* value_cache,
                        int64_t cache_block_stride, int64_t cache_token_stride,
                        int64_t cache_head_stride, const float* key_scales,
                        const float* value_scales, int64_t scale_block_stride,
                        int64_t scale_head_stride, const int32_t* block_tables,
                        int64_t block_table_stride, int32_t block_table_width, const void* plan,
                        int64_t plan_bytes, void* out, int64_t out_token_stride,
                        int64_t out_head_stride, void* workspace, int64_t workspace_bytes,
                        int32_t* counters, int32_t num_seqs, int32_t num_q_heads,
                        int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                        int32_t num_blocks, float scale, int32_t dtype, int32_t code,
                        void* stream);

/*
 * Varlen attention: mi_paged_prefill over an 8-bit cache. Request r's query
 * rows are cu_seqlens_q[r] .. cu_seqlens_q[r + 1], its context
 * cu_seqlens_k[r + 1] - cu_seqlens_k[r] positions, the mask causal and
 * bottom-right aligned. Rows that see no position give zeros; rows of no request
 * (behind the last, or ahead of the first) stay as they were. max_seqlen_q
 * bounds the query rows of any request: rows past it may stay unwritten. A NaN
 * makes NaN of the rows that see it; one in V may also do so to earlier rows of
 * its own request (0 times it is NaN), but to none of another, and what lies
 * behind a context or outside the pool reaches no row.
 *
 * Where mi_quant_prefill_workspace_bytes() is not 0, calls of these sizes take
 * a workspace of so many bytes (256-byte aligned) in which
 * mi_quant_prefill_plan has laid out the step, on the device, from the
 * cu_seqlens, for the same sizes, max_seqlen_q and table width; the plan serves
 * all layers, one call after the other. Calls that may run concurrently need
 * workspaces of their own. Long requests take room for 1024 parts of row blocks:
 * 71 MB with heads of 128, 38 MB with heads of 64, however few the tokens.
 *
 * Where it is 0, calls run without a plan or workspace on the vector kernel, 28 to
 * 46 times slower than the MFMA kernel where both were measured: other head sizes
 * and blocks of less than 16, groups of more than 128 query heads a KV head, heads of
 * 256 with more than 256 rows a request (4096 in all), and steps of more than 2048
 * requests or 4096 row blocks, of which a step has num_tokens / (128 / group) +
 * num_requests (65000 tokens of groups of 8, 16000 of groups of 32): split those.
 */
int64_t mi_quant_prefill_workspace_bytes(int32_t num_tokens, int32_t num_requests,
                                         int32_t max_seqlen_q, int32_t num_q_heads,
                                         int32_t num_kv_heads, int32_t head_dim,
                                         int32_t block_size);
int32_t mi_quant_prefill_plan(const int32_t* cu_seqlens_q, const int32_t* cu_seqlens_k,
                              int32_t num_tokens, int32_t num_requests, int32_t max_seqlen_q,
                              int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                              int32_t block_size, int32_t block_table_width, void* workspace,
                              int64_t workspace_bytes, void* stream);
int32_t mi_quant_prefill(const void* query, int64_t q_token_stride, int64_t q_head_stride,
                         const void* key_cache, const void* value_cache,
                         int64_t cache_block_stride, int64_t cache_token_stride,
                         int64_t cache_head_stride, const float* key_scales,
                         const float* value_scales, int64_t scale_block_stride,
                         int64_t scale_head_stride, const int32_t* cu_seqlens_q,
                         const int32_t* cu_seqlens_k, const int32_t* block_tables,
                         int64_t block_table_stride, int32_t block_table_width, void* out,
                         int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                         int64_t workspace_bytes, int32_t num_tokens, int32_t num_requests,
                         int32_t max_seqlen_q, int32_t num_q_heads, int32_t num_kv_heads,
                         int32_t head_dim, int32_t block_size, int32_t num_blocks, float scale,
                         int32_t dtype, int32_t code, void* stream);

/*
 * Which capture into a graph the stream is in: *id is 0 outside any, otherwise
 * the capture's own number. For callers that keep workspaces: two graphs that are
 * replayed at once must not share one.
 */
int32_t mi_stream_capture_id(void* stream, uint64_t* id);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* MI_QUANT_H_ */
