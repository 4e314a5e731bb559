// C entry points of attention over an 8-bit K/V cache.
#include <algorithm>
#include <climits>

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

// A part of a sequence has at least so many positions, twice those of a 16-bit
// cache: as many bytes (four layers of one sequence of 1000 tokens with 64 / 128 /
// 192 / 256 41.3 / 38.2 / 40.3 / 40.7 us, four of up to 600 37.7 / 36.5 / 38.7 /
// 39.5).
constexpr int32_t kMinPart = 128;
// A sequence of up to so many is not cut at all: eight waves have two tiles of 32
// in flight each, so 384 cost one memory round trip, and a merge two more (one of
// 300 tokens 34.7 us whole, 36.4 in parts; of 500 38.7 and 36.6). Where sequences
// and KV heads alone make workgroups for much of the chip, eight times their
// number: 12 of 500 44 whole, 48 in parts, 16 of 900-1100 59 and 62, 24 of 500
// 48 and 55, 24 of 1000 61 and 67. More is worse where lengths differ (16 of 100 to
// 2000 with up to 1024 / 1536 / 2048 62 / 67 / 70).
int32_t whole_positions(int32_t num_seqs, int32_t num_kv_heads) {
  return static_cast<int32_t>(
      std::min<int64_t>(std::max<int64_t>(int64_t(8) * num_seqs * num_kv_heads, 384), 1536));
}

// Whether decode steps go to the MFMA kernel, cache alignment aside.
bool decode_on_mfma(int32_t head_dim, int32_t group, int32_t block_size) {
  return quant_decode_mfma_takes(head_dim, block_size) &&
         quant_decode_row_groups(group, head_dim) == 1;
}

// Varlen calls of at most kFewRows rows of a request at a KV head, or kFewInAll of
// all requests, are laid out and run like decode steps. Four layers of 32 query
// and 8 KV heads of 128, us like that / as longer ones: a token on 16000
// positions (one query head a KV head) 72 / 248, 8 tokens 117 / 249, 16 on 8000
// 105 / 200, 32 on 8000 154 / 202, 64 on 8000 260 / 212; 16 requests of 4 tokens
// on 4000 155 / 200, 32 of 8 on 2000 160 / 193, 64 of 4 234 / 277, 64 of 8 295 /
// 279, 8 of 16 on 4000 199 / 183, 32 of 16 on 2000 255 / 221.
constexpr int32_t kFewRows = 32;
constexpr int32_t kFewInAll = 128;
// Of heads of 256, whose longer requests are the vector kernel's, up to so many of
// a request, and so many of all for the workspace's size (8 requests of 30 tokens
// on 4000 531 us, on the vector kernel 6420).
constexpr int32_t kFewRows256 = 256;
constexpr int32_t kFewInAll256 = 4096;

// A varlen call's sizes and where its workspace holds what.
struct VarlenLayout {
  bool few;
  int32_t rows;  // few: of a request at a KV head, at most
  int32_t items;
  int64_t num_counters;
  int64_t lens, counters, plan, acc, ml;  // few: offsets
  int64_t total;  // 0: these sizes take no plan
};

VarlenLayout varlen_layout(int32_t num_tokens, int32_t num_requests, int32_t max_seqlen_q,
                           int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                           int32_t block_size) {
  VarlenLayout l{};
  if (num_tokens <= 0 || num_requests <= 0 || max_seqlen_q <= 0 || num_kv_heads <= 0 ||
      num_q_heads <= 0 || num_q_heads % num_kv_heads != 0)
    return l;
  const int32_t group = num_q_heads / num_kv_heads;
  const int64_t rows = static_cast<int64_t>(std::min(max_seqlen_q, num_tokens)) * group;
  const int64_t in_all = rows * num_requests;
  l.few = (rows <= kFewRows || in_all <= kFewInAll ||
           (head_dim == 256 && rows <= kFewRows256 && in_all <= kFewInAll256)) &&
          num_requests <= kMaxPlanSeqs && quant_decode_mfma_takes(head_dim, block_size);
  if (!l.few) {
    l.total = quant_prefill_workspace(num_tokens, num_requests, group, num_kv_heads, head_dim,
                                      block_size);
    return l;
  }
  l.rows = static_cast<int32_t>(rows);
  l.items = decode_max_items(num_requests, num_kv_heads, 0);
  l.num_counters = static_cast<int64_t>(num_requests) * num_kv_heads *
                   quant_decode_row_groups(l.rows, head_dim);
  if (l.num_counters > INT_MAX) return l;
  auto room = [&](int64_t bytes) {
    const int64_t at = l.total;
    l.total += (bytes + 255) / 256 * 256;
    return at;
  };
  const int64_t slots = static_cast<int64_t>(l.items) * num_kv_heads * rows;
  l.lens = room(num_requests * int64_t(4));
  l.counters = room(l.num_counters * 4);
  l.plan = room(decode_plan_bytes(num_requests, num_kv_heads, 0));
  l.acc = room(slots * head_dim * 4);
  l.ml = room(slots * 2 * 4);
  return l;
}

int32_t check_varlen_workspace(const std::string& fn, const VarlenLayout& l,
                               const void* workspace, int64_t bytes) {
  if (workspace == nullptr || bytes < l.total || reinterpret_cast<uintptr_t>(workspace) % 256 != 0)
    return fail(MI_ERR_WORKSPACE, fn + ": workspace needs " + std::to_string(l.total) +
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
  const bool mfma = decode_on_mfma(head_dim, num_q_heads / num_kv_heads, block_size);
  return launch_decode_plan(context_lens, num_seqs, num_kv_heads, block_size, block_table_width,
                            0, !mfma, static_cast<PlanItem*>(plan), counters,
                            static_cast<hipStream_t>(stream),
                            mfma ? kMinPart : kMinPartPositions,
                            mfma ? whole_positions(num_seqs, num_kv_heads) : 0);
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
  if (decode_on_mfma(head_dim, a.group, block_size) && quant_mfma_aligned(a.c))
    return launch_quant_decode_mfma(a, a.group, dtype, code, s);
  return launch_quant_vector(a, dtype, code, s);
}

extern "C" int64_t mi_quant_prefill_workspace_bytes(int32_t num_tokens, int32_t num_requests,
                                                    int32_t max_seqlen_q, int32_t num_q_heads,
                                                    int32_t num_kv_heads, int32_t head_dim,
                                                    int32_t block_size) {
  return mi::varlen_layout(num_tokens, num_requests, max_seqlen_q, num_q_heads, num_kv_heads,
                           head_dim, block_size).total;
}

extern "C" int32_t mi_quant_prefill_plan(const int32_t* cu_seqlens_q,
                                         const int32_t* cu_seqlens_k, int32_t num_tokens,
                                         int32_t num_requests, int32_t max_seqlen_q,
                                         int32_t num_q_heads, int32_t num_kv_heads,
                                         int32_t head_dim, int32_t block_size,
                                         int32_t block_table_width, void* workspace,
                                         int64_t workspace_bytes, void* stream) {
  using namespace mi;
  clear_error();
  const std::string fn = "mi_quant_prefill_plan";
  int32_t st = check_heads(fn, num_q_heads, num_kv_heads);
  if (st != MI_OK) return st;
  const VarlenLayout l = varlen_layout(num_tokens, num_requests, max_seqlen_q, num_q_heads,
                                       num_kv_heads, head_dim, block_size);
  if (l.total == 0) return fail(MI_ERR_UNSUPPORTED, fn + ": these sizes take no plan");
  if (!is_pow2(block_size))
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": block_size must be a power of two");
  if (block_table_width < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": negative table width");
  if (static_cast<int64_t>(block_table_width) * block_size > (int64_t(1) << 30))
    return fail(MI_ERR_UNSUPPORTED, fn + ": tables of more than 2^30 positions");
  if (!cu_seqlens_q || !cu_seqlens_k)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  st = check_varlen_workspace(fn, l, workspace, workspace_bytes);
  if (st != MI_OK) return st;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  if (!l.few)
    return launch_quant_prefill_plan(cu_seqlens_q, cu_seqlens_k, num_tokens, num_requests,
                                     num_q_heads / num_kv_heads, num_kv_heads, head_dim,
                                     workspace, s);
  char* ws = static_cast<char*>(workspace);
  int32_t* lens = reinterpret_cast<int32_t*>(ws + l.lens);
  st = launch_few_rows(cu_seqlens_q, cu_seqlens_k, num_requests, lens,
                       reinterpret_cast<int32_t*>(ws + l.counters),
                       static_cast<int32_t>(l.num_counters), s);
  if (st != MI_OK) return st;
  return launch_decode_plan(lens, num_requests, num_kv_heads, block_size, block_table_width, 0,
                            false, reinterpret_cast<PlanItem*>(ws + l.plan), nullptr, s,
                            kMinPart, whole_positions(num_requests, num_kv_heads));
}

extern "C" int32_t mi_quant_prefill(
    const void* query, int64_t q_token_stride, int64_t q_head_stride, const void* key_cache,
    const void* value_cache, int64_t cache_block_stride, int64_t cache_token_stride,
    int64_t cache_head_stride, const float* key_scales, const float* value_scales,
    int64_t scale_block_stride, int64_t scale_head_stride, const int32_t* cu_seqlens_q,
    const int32_t* cu_seqlens_k, const int32_t* block_tables, int64_t block_table_stride,
    int32_t block_table_width, void* out, int64_t out_token_stride, int64_t out_head_stride,
    void* workspace, int64_t workspace_bytes, int32_t num_tokens, int32_t num_requests,
    int32_t max_seqlen_q, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t block_size, int32_t num_blocks, float scale, int32_t dtype, int32_t code,
    void* stream) {
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
  if (max_seqlen_q <= 0)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": max_seqlen_q must be positive");
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
  const VarlenLayout l = varlen_layout(num_tokens, num_requests, max_seqlen_q, num_q_heads,
                                       num_kv_heads, head_dim, block_size);
  if (l.total == 0 || !quant_mfma_aligned(a.c)) return launch_quant_vector(a, dtype, code, s);
  st = check_varlen_workspace(fn, l, workspace, workspace_bytes);
  if (st != MI_OK) return st;
  if (!l.few) return launch_quant_prefill_mfma(a, dtype, code, workspace, s);
  char* ws = static_cast<char*>(workspace);
  a.max_items = l.items;
  a.plan = reinterpret_cast<const PlanItem*>(ws + l.plan);
  a.counters = reinterpret_cast<int32_t*>(ws + l.counters);
  a.ws_acc = reinterpret_cast<float*>(ws + l.acc);
  a.ws_ml = reinterpret_cast<float*>(ws + l.ml);
  return launch_quant_decode_mfma(a, l.rows, dtype, code, s);
}

extern "C" int32_t mi_stream_capture_id(void* stream, uint64_t* id) {
  using namespace mi;
  clear_error();
  if (id == nullptr) return fail(MI_ERR_INVALID_ARGUMENT, "mi_stream_capture_id: null pointer");
  hipStreamCaptureStatus status = hipStreamCaptureStatusNone;
  unsigned long long number = 0;
  const hipError_t err =
      hipStreamGetCaptureInfo(static_cast<hipStream_t>(stream), &status, &number);
  if (err != hipSuccess)
    return fail(MI_ERR_HIP, std::string("mi_stream_capture_id: ") + hipGetErrorString(err));
  *id = status == hipStreamCaptureStatusNone ? 0 : number;
  return MI_OK;
}
