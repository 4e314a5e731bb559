// C entry points of attention over an 8-bit K/V cache.
#include <cmath>

#include "quant_mfma.h"

namespace mi {
namespace {

constexpr float kLog2e = 1.4426950408889634f;

int32_t check_heads(const std::string& fn, int32_t num_q_heads, int32_t num_kv_heads) {
  if (num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads % num_kv_heads != 0)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": Hq must be a positive multiple of Hkv");
  return MI_OK;
}

int32_t check_table(const std::string& fn, const int32_t* tables, int32_t width,
                    int32_t block_size) {
  if (width < 0) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": negative table width");
  if (width > 0 && !tables) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  if (static_cast<int64_t>(width) * block_size > (int64_t(1) << 30))
    return fail(MI_ERR_UNSUPPORTED, fn + ": tables of more than 2^30 positions");
  return MI_OK;
}

int32_t check_prefill_workspace(const std::string& fn, int32_t num_tokens, int32_t num_requests,
                                int32_t group, int32_t num_kv_heads, int32_t head_dim,
                                int32_t block_size, const void* workspace, int64_t bytes) {
  const int64_t need = quant_prefill_workspace(num_tokens, num_requests, group, num_kv_heads,
                                               head_dim, block_size);
  if (workspace == nullptr || bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return fail(MI_ERR_WORKSPACE, fn + ": workspace needs " + std::to_string(need) +
                                      " bytes, 256-byte aligned");
  return MI_OK;
}

}  // namespace
}  // namespace mi

extern "C" int64_t mi_quant_decode_plan_bytes(int32_t num_seqs, int32_t num_kv_heads) {
  return mi_decode_plan_bytes(num_seqs, num_kv_heads, 0);
}

extern "C" int64_t mi_quant_decode_workspace_bytes(int32_t num_seqs, int32_t num_q_heads,
                                                   int32_t num_kv_heads, int32_t head_dim) {
  using namespace mi;
  if (num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads <= 0 || head_dim <= 0) return 0;
  return static_cast<int64_t>(decode_max_items(num_seqs, num_kv_heads, 0)) * num_q_heads *
         (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

extern "C" int32_t mi_quant_decode_plan(const int32_t* context_lens, int32_t num_seqs,
                                        int32_t num_q_heads, int32_t num_kv_heads,
                                        int32_t head_dim, int32_t block_size,
                                        int32_t block_table_width, int32_t dtype, void* plan,
                                        int64_t plan_bytes, int32_t* counters, void* stream) {
  using namespace mi;
  clear_error();
  const std::string fn = "mi_quant_decode_plan";
  if (!valid_dtype(dtype)) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": bad dtype");
  int32_t st = check_heads(fn, num_q_heads, num_kv_heads);
  if (st != MI_OK) return st;
  if (num_seqs < 0 || head_dim <= 0 || block_table_width < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": invalid sizes");
  if (!is_pow2(block_size))
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": block_size must be a power of two");
  if (static_cast<int64_t>(block_table_width) * block_size > (int64_t(1) << 30))
    return fail(MI_ERR_UNSUPPORTED, fn + ": tables of more than 2^30 positions");
  if (num_seqs > kMaxPlanSeqs)
    return fail(MI_ERR_UNSUPPORTED, fn + ": more than 4096 sequences");
  if (num_seqs == 0) return MI_OK;
  if (!context_lens || !plan || !counters)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  if (plan_bytes < decode_plan_bytes(num_seqs, num_kv_heads, 0) ||
      reinterpret_cast<uintptr_t>(plan) % 32 != 0)
    return fail(MI_ERR_WORKSPACE, fn + ": plan buffer too small or misaligned");
  return launch_decode_plan(context_lens, num_seqs, num_kv_heads, block_size, block_table_width,
                            0,
                            !quant_decode_mfma_takes(head_dim, num_q_heads / num_kv_heads,
                                                     block_size),
                            static_cast<PlanItem*>(plan), counters,
                            static_cast<hipStream_t>(stream));
}

extern "C" int32_t mi_quant_decode(
    const void* query, int64_t q_token_stride, int64_t q_head_stride, const void* key_cache,
    const void* value_cache, int64_t cache_block_stride, int64_t cache_token_stride,
    int64_t cache_head_stride, const float* key_scales, const float* value_scales,
    int64_t scale_block_stride, int64_t scale_head_stride, const int32_t* block_tables,
    int64_t block_table_stride, int32_t block_table_width, const void* plan, int64_t plan_bytes,
    void* out, int64_t out_token_stride, int64_t out_head_stride, void* workspace,
    int64_t workspace_bytes, int32_t* counters, int32_t num_seqs, int32_t num_q_heads,
    int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t num_blocks, float scale,
    int32_t dtype, int32_t code, void* stream) {
  using namespace mi;
  clear_error();
  const std::string fn = "mi_quant_decode";
  int32_t st = check_quant_cache(
      fn, key_cache, value_cache, cache_block_stride, cache_token_stride, cache_head_stride,
      key_scales, value_scales, scale_block_stride, scale_head_stride, num_kv_heads, head_dim,
      block_size, num_blocks, dtype, code);
  if (st == MI_OK) st = check_heads(fn, num_q_heads, num_kv_heads);
  if (st == MI_OK) st = check_table(fn, block_tables, block_table_width, block_size);
  if (st != MI_OK) return st;
  if (num_seqs < 0) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": negative num_seqs");
  if (num_seqs > kMaxPlanSeqs)
    return fail(MI_ERR_UNSUPPORTED, fn + ": more than 4096 sequences");
  if (num_seqs == 0) return MI_OK;
  if (!query || !out || !plan) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  if (!whole_vectors(query, q_token_stride, q_head_stride, dtype) ||
      !whole_vectors(out, out_token_stride, out_head_stride, dtype))
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": misaligned rows");
  if (plan_bytes < decode_plan_bytes(num_seqs, num_kv_heads, 0) ||
      reinterpret_cast<uintptr_t>(plan) % 32 != 0)
    return fail(MI_ERR_WORKSPACE, fn + ": plan buffer too small or misaligned");
  const int64_t need =
      mi_quant_decode_workspace_bytes(num_seqs, num_q_heads, num_kv_heads, head_dim);
  if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 16 != 0 ||
      !counters)
    return fail(MI_ERR_WORKSPACE, fn + ": workspace needs " + std::to_string(need) +
                                      " bytes, 16-byte aligned, and counters");
  QuantAttnArgs a{};
  a.q = query;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.c = make_quant_cache(key_cache, value_cache, cache_block_stride, cache_token_stride,
                         cache_head_stride, key_scales, value_scales, scale_block_stride,
                         scale_head_stride, num_kv_heads, head_dim, block_size, num_blocks);
  a.tables = block_tables;
  a.t_stride = block_table_stride;
  a.t_width = block_table_width;
  a.out = out;
  a.o_ts = out_token_stride;
  a.o_hs = out_head_stride;
  a.max_items = decode_max_items(num_seqs, num_kv_heads, 0);
  a.ws_acc = static_cast<float*>(workspace);
  a.ws_ml = a.ws_acc + static_cast<int64_t>(a.max_items) * num_q_heads * head_dim;
  a.counters = counters;
  a.plan = static_cast<const PlanItem*>(plan);
  a.num_seqs = a.num_rows = num_seqs;
  a.group = num_q_heads / num_kv_heads;
  a.scale_log2 = scale * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (quant_decode_mfma_supported(a)) return launch_quant_decode_mfma(a, dtype, code, s);
  return launch_quant_vector(a, dtype, code, s);
}

extern "C" int64_t mi_quant_prefill_workspace_bytes(int32_t num_tokens, int32_t num_requests,
                                                    int32_t num_q_heads, int32_t num_kv_heads,
                                                    int32_t head_dim, int32_t block_size) {
  if (num_kv_heads <= 0 || num_q_heads <= 0 || num_q_heads % num_kv_heads) return 0;
  return mi::quant_prefill_workspace(num_tokens, num_requests, num_q_heads / num_kv_heads,
                                     num_kv_heads, head_dim, block_size);
}

extern "C" int32_t mi_quant_prefill_plan(const int32_t* cu_seqlens_q,
                                         const int32_t* cu_seqlens_k, int32_t num_tokens,
                                         int32_t num_requests, int32_t num_q_heads,
                                         int32_t num_kv_heads, int32_t head_dim,
                                         int32_t block_size, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
  using namespace mi;
  clear_error();
  const std::string fn = "mi_quant_prefill_plan";
  int32_t st = check_heads(fn, num_q_heads, num_kv_heads);
  if (st != MI_OK) return st;
  const int32_t group = num_q_heads / num_kv_heads;
  if (quant_prefill_workspace(num_tokens, num_requests, group, num_kv_heads, head_dim,
                              block_size) == 0)
    return fail(MI_ERR_UNSUPPORTED, fn + ": these sizes take no plan");
  if (!cu_seqlens_q || !cu_seqlens_k)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  st = check_prefill_workspace(fn, num_tokens, num_requests, group, num_kv_heads, head_dim,
                               block_size, workspace, workspace_bytes);
  if (st != MI_OK) return st;
  return launch_quant_prefill_plan(cu_seqlens_q, cu_seqlens_k, num_tokens, num_requests, group,
                                   num_kv_heads, head_dim, workspace,
                                   static_cast<hipStream_t>(stream));
}

extern "C" int32_t mi_quant_prefill(
    const void* query, int64_t q_token_stride, int64_t q_head_stride, const void* key_cache,
    const void* value_cache, int64_t cache_block_stride, int64_t cache_token_stride,
    int64_t cache_head_stride, const float* key_scales, const float* value_scales,
    int64_t scale_block_stride, int64_t scale_head_stride, const int32_t* cu_seqlens_q,
    const int32_t* cu_seqlens_k, const int32_t* block_tables, int64_t block_table_stride,
    int32_t block_table_width, void* out, int64_t out_token_stride, int64_t out_head_stride,
    void* workspace, int64_t workspace_bytes, int32_t num_tokens, int32_t num_requests,
    int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
    int32_t num_blocks, float scale, int32_t dtype, int32_t code, void* stream) {
  using namespace mi;
  clear_error();
  const std::string fn = "mi_quant_prefill";
  int32_t st = check_quant_cache(
      fn, key_cache, value_cache, cache_block_stride, cache_token_stride, cache_head_stride,
      key_scales, value_scales, scale_block_stride, scale_head_stride, num_kv_heads, head_dim,
      block_size, num_blocks, dtype, code);
  if (st == MI_OK) st = check_heads(fn, num_q_heads, num_kv_heads);
  if (st == MI_OK) st = check_table(fn, block_tables, block_table_width, block_size);
  if (st != MI_OK) return st;
  if (num_tokens < 0 || num_requests < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": negative sizes");
  if (num_tokens == 0) return MI_OK;
  if (num_requests == 0) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": tokens without requests");
  if (!query || !out || !cu_seqlens_q || !cu_seqlens_k)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  if (!whole_vectors(query, q_token_stride, q_head_stride, dtype) ||
      !whole_vectors(out, out_token_stride, out_head_stride, dtype))
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": misaligned rows");
  QuantAttnArgs a{};
  a.q = query;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.c = make_quant_cache(key_cache, value_cache, cache_block_stride, cache_token_stride,
                         cache_head_stride, key_scales, value_scales, scale_block_stride,
                         scale_head_stride, num_kv_heads, head_dim, block_size, num_blocks);
  a.tables = block_tables;
  a.t_stride = block_table_stride;
  a.t_width = block_table_width;
  a.cu_q = cu_seqlens_q;
  a.cu_k = cu_seqlens_k;
  a.out = out;
  a.o_ts = out_token_stride;
  a.o_hs = out_head_stride;
  a.num_seqs = num_requests;
  a.num_rows = num_tokens;
  a.group = num_q_heads / num_kv_heads;
  a.scale_log2 = scale * kLog2e;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (!quant_prefill_mfma_supported(a)) return launch_quant_vector(a, dtype, code, s);
  st = check_prefill_workspace(fn, num_tokens, num_requests, a.group, num_kv_heads, head_dim,
                               block_size, workspace, workspace_bytes);
  if (st != MI_OK) return st;
  return launch_quant_prefill_mfma(a, dtype, code, workspace, s);
}
