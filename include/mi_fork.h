/*
 * mi_fork.h -- C ABI of libmi_attn.so for several continuations of one
 * prompt: copies of cache pages (forks, beams, compaction), decode attention
 * of sequences that share their first pages, and log probabilities of tokens.
 * No counterpart in the reference.
 *
 * The rules of mi_attn.h hold: nothing here synchronises, allocates device
 * memory or records memset/memcpy nodes; element strides; MI_* status codes;
 * mi_last_error().
 */
#ifndef MI_FORK_H_
#define MI_FORK_H_

#include <stdint.h>

#include "mi_attn.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * Page copies inside a K/V pool: for every pair i, layer l, KV head and row
 * r < tokens[i] (all block_size rows where tokens is NULL),
 *   K[l, dst[i], r] = K'[l, src[i], r], V[l, dst[i], r] = V'[l, src[i], r]
 * where K', V' are the pools before the call: a parallel assignment, so a
 * block may be the source of several pairs, and a destination may be another
 * pair's source (moves in a chain, swaps, longer cycles). Other rows keep
 * their contents. Byte copies: bit-exact for every dtype.
 *
 * src, dst, tokens are HOST arrays of num_pairs entries, read before the call
 * returns; they travel with the launches, so a captured call replays the
 * pairs of its capture. Block ids lie in [0, num_blocks), tokens in
 * [0, block_size], and no dst appears twice (MI_ERR_INVALID_ARGUMENT). A
 * cycle of more than 255 blocks is MI_ERR_UNSUPPORTED. Every check runs
 * before the first launch. key_cache and value_cache are [num_layers,
 * num_blocks, block_size, num_kv_heads, head_dim] through the same layer,
 * block, token and head strides (in elements, not negative), head_dim
 * contiguous.
 */
int32_t mi_kv_copy_blocks(void* key_cache, void* value_cache, int64_t layer_stride,
                          int64_t block_stride, int64_t token_stride, int64_t head_stride,
                          const int32_t* src, const int32_t* dst, const int32_t* tokens,
                          int32_t num_pairs, int32_t num_layers, int32_t num_kv_heads,
                          int32_t head_dim, int32_t block_size, int32_t num_blocks,
                          int32_t dtype, void* stream);

/*
 * Decode attention of sequences that share their first blocks: the result of
 * mi_paged_decode with the same tables and lengths (up to rounding), with the
 * blocks that a group of sequences shares read once for every 64 query rows of
 * a KV head (64 / G sequences of G query heads per KV head).
 *
 * Group g is the sequences [group_starts[g], group_starts[g + 1]) (rising;
 * sequences outside every group are on their own), whose tables hold the same
 * ids in their first shared_blocks[g] columns; only whole blocks within every
 * one of the group's contexts count (the rest of shared_blocks[g] is not
 * taken as shared). A group of one shares nothing. Groups that break these
 * rules give wrong attention, never an access out of bounds.
 *
 * mi_shared_decode_plan makes a step's plan on the device from int32 device
 * arrays (context_lens [num_seqs], group_starts [num_groups + 1],
 * shared_blocks [num_groups]); mi_shared_decode runs a layer with it, so one
 * plan serves all layers of a step. A negative or too large block id is
 * masked; sequences of context 0 give zeros; a NaN score makes its row NaN
 * wherever the context is split. Both are capture-safe.
 *
 * plan: mi_shared_decode_plan_bytes() bytes, 32-byte aligned; workspace:
 * mi_shared_decode_workspace_bytes() bytes, 16-byte aligned, no
 * initialisation, its own for calls that may run concurrently. Both sizes
 * depend on their arguments only. bf16/f16, head_dim 128, at most 16 query
 * heads per KV head, block_size >= 16 and a power of two, at most 4096
 * sequences and groups, block tables of at most 2^30 positions
 * (MI_ERR_UNSUPPORTED otherwise: mi_paged_decode takes the other types, heads
 * and block sizes). query, the caches and out 16-byte aligned, with strides of
 * whole 16-byte vectors; block_tables may be NULL where it has no columns.
 */
int64_t mi_shared_decode_plan_bytes(int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads);
int64_t mi_shared_decode_workspace_bytes(int32_t num_seqs, int32_t num_q_heads,
                                         int32_t num_kv_heads);
int32_t mi_shared_decode_plan(const int32_t* context_lens, int32_t num_seqs,
                              const int32_t* group_starts, const int32_t* shared_blocks,
                              int32_t num_groups, int32_t num_q_heads, int32_t num_kv_heads,
                              int32_t head_dim, int32_t block_size, int32_t block_table_width,
                              int32_t dtype, void* plan, int64_t plan_bytes, void* stream);
int32_t mi_shared_decode(const void* query, int64_t q_token_stride, int64_t q_head_stride,
                         const void* key_cache, const void* value_cache,
                         int64_t cache_block_stride, int64_t cache_token_stride,
                         int64_t cache_head_stride, const int32_t* block_tables,
                         int64_t block_table_stride, int32_t block_table_width,
                         const void* plan, int64_t plan_bytes, void* out,
                         int64_t out_token_stride, int64_t out_head_stride, void* workspace,
                         int64_t workspace_bytes, int32_t num_seqs, int32_t num_q_heads,
                         int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                         int32_t num_blocks, float scale, int32_t dtype, void* stream);

/*
 * Log probabilities of given tokens, the entropy and the best alternatives of
 * each row of logits, in one launch. With x = logits[r] / temperatures[r] (1
 * where temperatures is NULL) and p = softmax(x), in float32:
 *   logprobs[r, i]     = ln p[tokens[r, i]], i < num_given
 *   entropy[r]         = -sum_v p[v] ln p[v]  (0 ln 0 = 0; NULL: not computed)
 *   top_tokens[r, i]   = the i-th largest logit's index, i < num_top
 *   top_logprobs[r, i] = ln p of it
 * The order is mi_greedy_argmax's: NaN above every number, the lowest index
 * first among equals. A masked logit (-inf) has probability 0 and log
 * probability -inf. A token outside [0, vocab_size) gives NaN, and so do all
 * of a row's log probabilities and its entropy where the row has a NaN, +inf
 * or nothing above -inf, or a temperature that is not finite or below the
 * smallest normal float32 (2^-126); its top_tokens are still in order.
 *
 * tokens (int64, row stride token_stride) and logprobs ([num_rows, num_given],
 * contiguous) may be NULL with num_given 0, top_tokens (int64) and
 * top_logprobs ([num_rows, num_top], contiguous) with num_top 0. num_top is
 * at most 32 and at most vocab_size; vocab_size at most 2^30; num_given at
 * most 65536.
 *
 * workspace: mi_token_logprobs_workspace_bytes(...) bytes, 16-byte aligned, no
 * initialisation (NULL where that is 0). counters: num_rows int32 that are
 * ZERO on entry and left zero (NULL where no workspace is needed). Launches
 * that may run concurrently need their own.
 */
int64_t mi_token_logprobs_workspace_bytes(int32_t num_rows, int32_t vocab_size, int32_t num_top,
                                          int32_t dtype);
int32_t mi_token_logprobs(const void* logits, int64_t row_stride, int32_t num_rows,
                          int32_t vocab_size, int32_t dtype, const float* temperatures,
                          const int64_t* tokens, int64_t token_stride, int32_t num_given,
                          float* logprobs, float* entropy, int64_t* top_tokens,
                          float* top_logprobs, int32_t num_top, void* workspace,
                          int64_t workspace_bytes, int32_t* counters, void* stream);

#ifdef __cplusplus
} /* extern "C" */
#endif

#endif /* MI_FORK_H_ */
