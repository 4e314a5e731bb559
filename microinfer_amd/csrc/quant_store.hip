// Writes into and reads out of an 8-bit K/V cache (mi_quant_append,
// mi_quant_append_plan, mi_quant_gather).
//
// Append. A block's scale depends on all of its rows, so one wave has the
// whole (block, KV head) of K or of V: it finds the call's rows of the block,
// takes their largest magnitude, settles the scale, rounds the rows that are
// held again where the scale rose, and the new ones. Bound by HBM for prompts
// (es + 1 bytes a value), by a chain of dependent loads for decode steps.
#include <algorithm>

#include "quant.h"

namespace mi {

int32_t check_quant_cache(const std::string& fn, const void* key_cache, const void* value_cache,
                          int64_t block_stride, int64_t token_stride, int64_t head_stride,
                          const float* key_scales, const float* value_scales,
                          int64_t scale_block_stride, int64_t scale_head_stride,
                          int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                          int32_t num_blocks, int32_t dtype, int32_t code) {
  if (!valid_dtype(dtype)) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": bad dtype");
  if (code != MI_CODE_E4M3 && code != MI_CODE_INT8)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": bad code");
  if (num_kv_heads <= 0 || head_dim <= 0 || num_blocks <= 0)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": sizes must be positive");
  if (!is_pow2(head_dim) || head_dim < 16 || head_dim > 256)
    return fail(MI_ERR_UNSUPPORTED, fn + ": head_dim must be a power of two from 16 to 256");
  if (!is_pow2(block_size))
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": block_size must be a power of two");
  if (num_kv_heads > 65535)
    return fail(MI_ERR_UNSUPPORTED, fn + ": more than 65535 KV heads");
  if (!key_cache || !value_cache || !key_scales || !value_scales)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  if (block_stride < 0 || token_stride < 0 || head_stride < 0 || scale_block_stride < 0 ||
      scale_head_stride < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": negative stride");
  if ((reinterpret_cast<uintptr_t>(key_cache) | reinterpret_cast<uintptr_t>(value_cache) |
       block_stride | token_stride | head_stride) & 7)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": misaligned cache");
  if ((reinterpret_cast<uintptr_t>(key_scales) | reinterpret_cast<uintptr_t>(value_scales)) & 3)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": misaligned scales");
  return MI_OK;
}

QuantCache make_quant_cache(const void* key_cache, const void* value_cache, int64_t block_stride,
                            int64_t token_stride, int64_t head_stride, const float* key_scales,
                            const float* value_scales, int64_t scale_block_stride,
                            int64_t scale_head_stride, int32_t num_kv_heads, int32_t head_dim,
                            int32_t block_size, int32_t num_blocks) {
  return QuantCache{static_cast<const uint8_t*>(key_cache),
                    static_cast<const uint8_t*>(value_cache),
                    block_stride,
                    token_stride,
                    head_stride,
                    key_scales,
                    value_scales,
                    scale_block_stride,
                    scale_head_stride,
                    num_kv_heads,
                    head_dim,
                    block_size,
                    ilog2(block_size),
                    num_blocks};
}

namespace {

constexpr int kMaxScan = 1024;   // rows whose slot list a workgroup reads itself
constexpr int kMaxBlock = 1024;  // tokens a block
constexpr int kGroupRows = 16;   // list entries of a workgroup, with a plan
constexpr int kAppendThreads = 256;

// A row's slot, -1 where it is skipped.
__device__ __forceinline__ int64_t slot_of(const void* slots, int is64, int t, int64_t end) {
  const int64_t s = is64 ? static_cast<const int64_t*>(slots)[t]
                         : static_cast<const int32_t*>(slots)[t];
  return s >= 0 && s < end ? s : -1;
}

__global__ __launch_bounds__(256) void append_plan_kernel(const void* __restrict__ slots, int is64,
                                                          int num_tokens, int64_t end,
                                                          int32_t* __restrict__ rows) {
  const int t = blockIdx.x * 256 + threadIdx.x;
  if (t >= num_tokens) return;
  const int64_t s = slot_of(slots, is64, t, end);
  if (s >= 0) rows[s] = t;
}

struct AppendArgs {
  const void* keys;
  const void* values;
  int64_t k_ts, k_hs, v_ts, v_hs;
  QuantCache c;
  const void* slots;
  const int32_t* rows;  // null: scan the list
  int32_t is64, num_tokens;
};

// The least power of two s >= 2^-126 with most <= C::kMost s (most >= 0, finite).
template <typename C>
__device__ __forceinline__ float least_scale(float most) {
  // most = m 2^e and kMost = f 2^k with m, f in [1, 2): 2^(e - k), twice that where m > f.
  constexpr uint32_t kBits = __builtin_bit_cast(uint32_t, C::kMost);
  constexpr uint32_t kFraction = kBits & 0x7fffffu;
  constexpr int kExponent = static_cast<int>(kBits >> 23) - 127;
  const int e = static_cast<int>((__float_as_uint(most) + 0x7fffffu - kFraction) >> 23);
  return __uint_as_float(static_cast<uint32_t>(max(e - kExponent, 1)) << 23);
}

// x / s by a product where s is a power of two, as it is unless the caller
// filled in other scales.
__device__ __forceinline__ void divide8(float* x, float s) {
  const uint32_t bits = __float_as_uint(s);
  const bool power = (bits & 0x7fffffu) == 0 && bits >= (1u << 23) && bits < (253u << 23);
  if (power) {
    const float inv = __uint_as_float((254u << 23) - bits);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] *= inv;
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] /= s;
  }
}

// K or V of one (block, KV head), by one wave. `tok`: the call's row of every
// offset of the block, -1 where none. A row is spread over LPR lanes, eight
// values each.
template <typename E, typename C, int LPR>
__device__ __forceinline__ void append_block(const typename E::raw* src, int64_t ts, uint8_t* dst,
                                             int64_t c_ts, float* scale, const int* tok,
                                             int block_size, int first, int lane) {
  constexpr int kStep = kWave / LPR;  // rows at once
  const int grp = lane / LPR, d0 = lane % LPR * 8;
  float most = 0.f;
  bool odd = false;  // a value that is not finite
  for (int o = grp; o < block_size; o += kStep) {
    const int t = tok[o];
    if (t < 0) continue;
    float x[8];
    load8<E>(src + t * ts + d0, x);
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float a = fabsf(x[i]);
      odd |= !(a < INFINITY);
      most = a < INFINITY ? fmaxf(most, a) : most;
    }
  }
  most = xor_max<1, kWave>(most);
  odd = __ballot(odd) != 0;
  const float need = !C::kHasNan && odd ? NAN : least_scale<C>(most);
  const float old = first > 0 ? *scale : 0.f;
  float now = need;
  if (first > 0 && !(old <= need)) now = need != need ? need : old;
  if (first > 0 && now != old && now == now) {
    const float ratio = old / now;
    for (int o = grp; o < first; o += kStep) {
      Codes8* at = reinterpret_cast<Codes8*>(dst + o * c_ts + d0);
      float x[8];
      widen8<C>(*at, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= ratio;
      *at = narrow8<C>(x);
    }
  }
  for (int o = grp; o < block_size; o += kStep) {
    const int t = tok[o];
    if (t < 0) continue;
    float x[8];
    load8<E>(src + t * ts + d0, x);
    divide8(x, now);
    *reinterpret_cast<Codes8*>(dst + o * c_ts + d0) = narrow8<C>(x);
  }
  if (lane == 0) *scale = now;
}

// blockIdx.x: `group` entries of the slot list; blockIdx.y: KV head. The first
// row of a block (its lowest offset) has the block.
template <typename E, typename C, int LPR>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(const AppendArgs a, int group) {
  extern __shared__ int s_tok[];  // [group][block_size]
  __shared__ int s_first[kGroupRows];
  const int tid = threadIdx.x;
  const int threads = blockDim.x;
  const QuantCache& c = a.c;
  const int64_t end = static_cast<int64_t>(c.num_blocks) * c.block_size;
  const int t0 = blockIdx.x * group;
  const int entries = min(group, a.num_tokens - t0);
  for (int i = tid; i < group * c.block_size; i += threads) s_tok[i] = -1;
  if (tid < kGroupRows) s_first[tid] = c.block_size;
  __syncthreads();
  if (a.rows != nullptr) {
    for (int i = tid; i < entries * c.block_size; i += threads) {
      const int e = i >> c.log2_block, o = i & (c.block_size - 1);
      const int64_t s = slot_of(a.slots, a.is64, t0 + e, end);
      if (s < 0) continue;
      const int64_t at = (s & ~static_cast<int64_t>(c.block_size - 1)) + o;
      const int t = a.rows[at];
      if (t >= 0 && t < a.num_tokens && slot_of(a.slots, a.is64, t, end) == at) s_tok[i] = t;
    }
  } else {  // one entry
    const int64_t s = slot_of(a.slots, a.is64, t0, end);
    if (s < 0) return;  // the whole workgroup
    for (int t = tid; t < a.num_tokens; t += threads) {
      const int64_t u = slot_of(a.slots, a.is64, t, end);
      if (u >= 0 && (u >> c.log2_block) == (s >> c.log2_block))
        atomicMax(&s_tok[u & (c.block_size - 1)], t);
    }
  }
  __syncthreads();
  for (int i = tid; i < entries * c.block_size; i += threads)
    if (s_tok[i] >= 0) atomicMin(&s_first[i >> c.log2_block], i & (c.block_size - 1));
  __syncthreads();
  const int lane = tid % kWave;
  const int64_t head = blockIdx.y;
  for (int u = tid / kWave; u < 2 * entries; u += threads / kWave) {
    const int e = u / 2;
    const int first = s_first[e];
    if (first == c.block_size || s_tok[e * c.block_size + first] != t0 + e) continue;
    const int64_t blk = slot_of(a.slots, a.is64, t0 + e, end) >> c.log2_block;
    const bool is_v = u & 1;
    using R = typename E::raw;
    const R* src = static_cast<const R*>(is_v ? a.values : a.keys) +
                   head * (is_v ? a.v_hs : a.k_hs);
    uint8_t* dst = const_cast<uint8_t*>(is_v ? c.v : c.k) + blk * c.bs + head * c.hs;
    float* scale = const_cast<float*>(is_v ? c.vs : c.ks) + blk * c.s_bs + head * c.s_hs;
    append_block<E, C, LPR>(src, is_v ? a.v_ts : a.k_ts, dst, c.ts, scale,
                            s_tok + e * c.block_size, c.block_size, first, lane);
  }
}

// Thread -> eight values of one (output row, head) of K and of V.
template <typename E, typename C>
__global__ __launch_bounds__(256) void gather_kernel(const QuantCache c,
                                                     const int32_t* __restrict__ tables,
                                                     int64_t t_stride, int t_width,
                                                     const int32_t* __restrict__ cu_k,
                                                     int num_requests, int total_rows,
                                                     typename E::raw* __restrict__ k_out,
                                                     typename E::raw* __restrict__ v_out) {
  const int per_row = c.heads * c.dim / 8;
  const int64_t i = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (i >= static_cast<int64_t>(total_rows) * per_row) return;
  const int row = static_cast<int>(i / per_row);
  const int in_row = static_cast<int>(i % per_row) * 8;
  const int head = in_row / c.dim, d0 = in_row % c.dim;
  int lo = 0, hi = num_requests - 1;  // the last request with cu_k <= row
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (cu_k[mid] <= row) lo = mid; else hi = mid - 1;
  }
  const int pos = row - cu_k[lo];
  float k[8] = {}, v[8] = {};
  if (pos >= 0 && (pos >> c.log2_block) < t_width) {
    const int blk = tables[lo * t_stride + (pos >> c.log2_block)];
    if (blk >= 0 && blk < c.num_blocks) {
      const int64_t at = blk * c.bs + (pos & (c.block_size - 1)) * c.ts + head * c.hs + d0;
      const int64_t s = blk * c.s_bs + head * c.s_hs;
      widen8<C>(*reinterpret_cast<const Codes8*>(c.k + at), k);
      widen8<C>(*reinterpret_cast<const Codes8*>(c.v + at), v);
      const float ks = c.ks[s], vs = c.vs[s];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        k[j] *= ks;
        v[j] *= vs;
      }
    }
  }
  store8<E>(k_out + i * 8, k);
  store8<E>(v_out + i * 8, v);
}

}  // namespace
}  // namespace mi

extern "C" int32_t mi_quant_append_plan(const void* slots, int32_t slots_are_int64,
                                        int32_t num_tokens, int32_t block_size,
                                        int32_t num_blocks, int32_t* rows, void* stream) {
  using namespace mi;
  clear_error();
  if (num_tokens < 0 || num_blocks <= 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_quant_append_plan: invalid sizes");
  if (!is_pow2(block_size))
    return fail(MI_ERR_INVALID_ARGUMENT,
                "mi_quant_append_plan: block_size must be a power of two");
  if (num_tokens == 0) return MI_OK;
  if (!slots || !rows) return fail(MI_ERR_INVALID_ARGUMENT, "mi_quant_append_plan: null pointer");
  append_plan_kernel<<<(num_tokens - 1) / 256 + 1, 256, 0, static_cast<hipStream_t>(stream)>>>(
      slots, slots_are_int64, num_tokens, static_cast<int64_t>(num_blocks) * block_size, rows);
  return check_launch("mi_quant_append_plan");
}

extern "C" int32_t mi_quant_append(
    const void* keys, int64_t key_token_stride, int64_t key_head_stride, const void* values,
    int64_t value_token_stride, int64_t value_head_stride, void* key_cache, void* value_cache,
    int64_t cache_block_stride, int64_t cache_token_stride, int64_t cache_head_stride,
    float* key_scales, float* value_scales, int64_t scale_block_stride,
    int64_t scale_head_stride, const void* slots, int32_t slots_are_int64, const int32_t* rows,
    int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
    int32_t num_blocks, int32_t dtype, int32_t code, void* stream) {
  using namespace mi;
  clear_error();
  const std::string fn = "mi_quant_append";
  const int32_t st = check_quant_cache(
      fn, key_cache, value_cache, cache_block_stride, cache_token_stride, cache_head_stride,
      key_scales, value_scales, scale_block_stride, scale_head_stride, num_kv_heads, head_dim,
      block_size, num_blocks, dtype, code);
  if (st != MI_OK) return st;
  if (num_tokens < 0) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": negative num_tokens");
  if (block_size > kMaxBlock)
    return fail(MI_ERR_UNSUPPORTED, fn + ": blocks of more than 1024 tokens");
  if (num_tokens == 0) return MI_OK;
  if (!keys || !values || !slots) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  if (!whole_vectors(keys, key_token_stride, key_head_stride, dtype) ||
      !whole_vectors(values, value_token_stride, value_head_stride, dtype))
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": misaligned rows");
  if (rows == nullptr && num_tokens > kMaxScan)
    return fail(MI_ERR_UNSUPPORTED, fn + ": more than 1024 tokens need mi_quant_append_plan");
  AppendArgs a{};
  a.keys = keys;
  a.values = values;
  a.k_ts = key_token_stride;
  a.k_hs = key_head_stride;
  a.v_ts = value_token_stride;
  a.v_hs = value_head_stride;
  a.c = make_quant_cache(key_cache, value_cache, cache_block_stride, cache_token_stride,
                         cache_head_stride, key_scales, value_scales, scale_block_stride,
                         scale_head_stride, num_kv_heads, head_dim, block_size, num_blocks);
  a.slots = slots;
  a.rows = rows;
  a.is64 = slots_are_int64;
  a.num_tokens = num_tokens;
  const int group = rows == nullptr ? 1 : std::max(1, std::min(kGroupRows, kMaxBlock / block_size));
  const dim3 grid((num_tokens - 1) / group + 1, num_kv_heads);
  const size_t lds = sizeof(int) * group * block_size;
  return with_types(dtype, code, [&](auto e, auto c) {
    using E = decltype(e);
    using C = decltype(c);
    auto go = [&](auto kernel) {
      kernel<<<grid, kAppendThreads, lds, static_cast<hipStream_t>(stream)>>>(a, group);
      return check_launch("mi_quant_append");
    };
    switch (head_dim) {
      case 16: return go(append_kernel<E, C, 2>);
      case 32: return go(append_kernel<E, C, 4>);
      case 64: return go(append_kernel<E, C, 8>);
      case 128: return go(append_kernel<E, C, 16>);
      default: return go(append_kernel<E, C, 32>);
    }
  });
}

extern "C" int32_t mi_quant_gather(
    const void* key_cache, const void* value_cache, int64_t cache_block_stride,
    int64_t cache_token_stride, int64_t cache_head_stride, const float* key_scales,
    const float* value_scales, int64_t scale_block_stride, int64_t scale_head_stride,
    const int32_t* block_tables, int64_t block_table_stride, int32_t block_table_width,
    const int32_t* cu_seqlens_k, int32_t num_requests, int32_t total_rows, void* key_out,
    void* value_out, int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
    int32_t num_blocks, int32_t dtype, int32_t code, void* stream) {
  using namespace mi;
  clear_error();
  const std::string fn = "mi_quant_gather";
  const int32_t st = check_quant_cache(
      fn, key_cache, value_cache, cache_block_stride, cache_token_stride, cache_head_stride,
      key_scales, value_scales, scale_block_stride, scale_head_stride, num_kv_heads, head_dim,
      block_size, num_blocks, dtype, code);
  if (st != MI_OK) return st;
  if (num_requests < 0 || total_rows < 0 || block_table_width < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": invalid sizes");
  if (total_rows == 0) return MI_OK;
  if (num_requests == 0) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": rows without requests");
  if (!cu_seqlens_k || !key_out || !value_out || (!block_tables && block_table_width > 0))
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  if (!whole_vectors(key_out, 0, 0, dtype) || !whole_vectors(value_out, 0, 0, dtype))
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": misaligned output");
  const int64_t groups = static_cast<int64_t>(total_rows) * num_kv_heads * head_dim / 8;
  if (groups > (int64_t(1) << 38))
    return fail(MI_ERR_UNSUPPORTED, fn + ": too many rows for one launch");
  const QuantCache cache = make_quant_cache(
      key_cache, value_cache, cache_block_stride, cache_token_stride, cache_head_stride,
      key_scales, value_scales, scale_block_stride, scale_head_stride, num_kv_heads, head_dim,
      block_size, num_blocks);
  return with_types(dtype, code, [&](auto e, auto c) {
    using E = decltype(e);
    using C = decltype(c);
    using R = typename E::raw;
    gather_kernel<E, C><<<static_cast<uint32_t>((groups - 1) / 256 + 1), 256, 0,
                          static_cast<hipStream_t>(stream)>>>(
        cache, block_tables, block_table_stride, block_table_width, cu_seqlens_k, num_requests,
        total_rows, static_cast<R*>(key_out), static_cast<R*>(value_out));
    return check_launch("mi_quant_gather");
  });
}
