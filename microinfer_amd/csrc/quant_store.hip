// Writes into and reads out of an 8-bit K/V cache (mi_quant_append,
// mi_quant_append_plan, mi_quant_gather).
//
// Append. A block's scale depends on all of its rows, so one wave has the
// whole (block, KV head) of K or of V: with the call's rows of the block it
// takes their largest magnitude, settles the scale, rounds the new ones and,
// where the scale rose, those that are held. Bound by HBM for prompts (es + 1
// bytes a value), by a chain of dependent loads for decode steps. With 8 heads of
// 128 in bf16 and blocks of 16: 16384 rows of a prompt 24.2 us (100 MB, 4.2 TB/s),
// 4096 8.1, 512 4.0; rows of as many sequences, 8 3.6, 64 3.8, 256 4.4, of which
// an empty launch has about 2.
//
// Which rows are a block's: calls of few rows look through the slot list, a
// workgroup for itself (us, of 64 / 256 / 512 rows of one prompt 4.3 / 5.5 / 7.8, of
// as many sequences 3.8 / 4.4 / 6.0); of many, a plan of two launches (5 us) says it
// for all layers of a step (3.8 / 3.9 / 3.9, and 4.7 / 12.2 / 12.4).
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

constexpr int kGatherThreads = 256;

// Eight elements of a row, past the caches: rows are written once and are many.
template <typename E>
__device__ __forceinline__ void store8_past(typename E::raw* p, const float* x) {
  using R = typename E::raw;
  typedef uint32_t u4 __attribute__((ext_vector_type(4)));
  constexpr int N = 16 / sizeof(R);
#pragma unroll
  for (int j = 0; j < 8; j += N) {
    Pack<R, N> v;
#pragma unroll
    for (int i = 0; i < N; ++i) v.v[i] = E::store(x[j + i]);
    __builtin_nontemporal_store(__builtin_bit_cast(u4, v), reinterpret_cast<u4*>(p + j));
  }
}
constexpr int kMaxScan = 1024;   // rows whose slot list a workgroup reads itself
constexpr int kMaxBlock = 1024;  // tokens a block
constexpr int kHeads = 4;      // KV heads of a workgroup, two waves each
constexpr int kAppendThreads = 2 * kHeads * kWave;
constexpr int kChunk = 256;   // list entries that a plan's workgroup looks through
constexpr int kPerChunk = 32;  // workgroups that share their blocks

// A row's slot, -1 where it is skipped.
__device__ __forceinline__ int64_t slot_of(const void* slots, int is64, int t, int64_t end) {
  const int64_t s = is64 ? static_cast<const int64_t*>(slots)[t]
                         : static_cast<const int32_t*>(slots)[t];
  return s >= 0 && s < end ? s : -1;
}

// A plan: for each chunk of the list the blocks that rows of it come first in
// (the list's, not yet the block's), with the row of every offset.
struct PlanBlock {
  int32_t block;  // kSkip: another entry has it; kEnd: no more in this chunk
  int32_t first;  // lowest offset
};
constexpr int kSkip = -1, kEnd = -2;
struct AppendPlan {
  PlanBlock* blocks;  // [chunks, kChunk]
  int32_t* tok;       // [chunks, kChunk, block_size]; -1: none
  int32_t* rows;      // [num_blocks, block_size]: a row written to the slot
  int64_t bytes;
};
AppendPlan append_plan_of(void* memory, int32_t num_tokens, int32_t block_size,
                          int32_t num_blocks) {
  AppendPlan p{};
  const int64_t entries = (static_cast<int64_t>(num_tokens) + kChunk - 1) / kChunk * kChunk;
  char* at = static_cast<char*>(memory);
  p.blocks = reinterpret_cast<PlanBlock*>(at);
  at += entries * static_cast<int64_t>(sizeof(PlanBlock));
  p.tok = reinterpret_cast<int32_t*>(at);
  at += entries * block_size * 4;
  p.rows = reinterpret_cast<int32_t*>(at);
  at += static_cast<int64_t>(num_blocks) * block_size * 4;
  p.bytes = at - static_cast<char*>(memory);
  return p;
}

__global__ __launch_bounds__(kChunk) void append_map_kernel(const void* __restrict__ slots,
                                                            int is64, int num_tokens, int64_t end,
                                                            int32_t* __restrict__ rows) {
  const int t = blockIdx.x * kChunk + threadIdx.x;
  if (t >= num_tokens) return;
  const int64_t s = slot_of(slots, is64, t, end);
  if (s >= 0) rows[s] = t;
}

// Entry t has its block if it is the row of the lowest offset written. An entry
// of `rows` counts if its row is in the list with that slot: what an earlier
// plan, or nobody, wrote there does not matter.
__global__ __launch_bounds__(kChunk) void append_blocks_kernel(const void* __restrict__ slots,
                                                               int is64, int num_tokens,
                                                               int64_t end, int log2_block,
                                                               AppendPlan p) {
  __shared__ int s_count;
  __shared__ int s_row[kChunk], s_first[kChunk];
  const int tid = threadIdx.x;
  const int block_size = 1 << log2_block;
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kChunk;
  if (tid == 0) s_count = 0;
  s_first[tid] = block_size;
  __syncthreads();
  const int64_t t = base + tid;
  if (t < num_tokens) {
    const int64_t s = slot_of(slots, is64, static_cast<int>(t), end);
    const int64_t before = t > 0 ? slot_of(slots, is64, static_cast<int>(t) - 1, end) : -1;
    // Not behind a lower row of its block in the list, as most of a prompt's are.
    if (s >= 0 && !(before >= 0 && before < s && before >> log2_block == s >> log2_block))
      s_row[atomicAdd(&s_count, 1)] = static_cast<int>(t);  // blocks have no order
  }
  __syncthreads();
  const int count = s_count;
  for (int64_t i = tid; i < static_cast<int64_t>(count) << log2_block; i += kChunk) {
    const int e = static_cast<int>(i >> log2_block), o = static_cast<int>(i & (block_size - 1));
    const int64_t at = (slot_of(slots, is64, s_row[e], end) >> log2_block << log2_block) + o;
    int u = p.rows[at];
    if (u < 0 || u >= num_tokens || slot_of(slots, is64, u, end) != at) u = -1;
    p.tok[(base << log2_block) + i] = u;
    if (u >= 0) atomicMin(&s_first[e], o);
  }
  __syncthreads();
  PlanBlock b{kEnd, 0};
  if (tid < count) {
    const int64_t block = slot_of(slots, is64, s_row[tid], end) >> log2_block;
    const int first = s_first[tid];
    const bool mine =
        first < block_size && p.rows[(block << log2_block) + first] == s_row[tid];
    b = PlanBlock{mine ? static_cast<int32_t>(block) : kSkip, first};
  }
  p.blocks[base + tid] = b;
}

struct AppendArgs {
  const void* keys;
  const void* values;
  int64_t k_ts, k_hs, v_ts, v_hs;
  QuantCache c;
  const void* slots;
  AppendPlan plan;
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

// x / s as a product with 1 / s where s is a power of two, as it is unless the
// caller filled in other scales.
struct Divisor {
  float s, inverse;
  bool power;
  explicit __device__ __forceinline__ Divisor(float scale) : s(scale) {
    const uint32_t bits = __float_as_uint(s);
    power = (bits & 0x7fffffu) == 0 && bits >= (1u << 23) && bits < (253u << 23);
    inverse = __uint_as_float((254u << 23) - bits);
  }
  template <typename C>
  __device__ __forceinline__ Codes8 encode(const float* x) const {
    float q[8];
    if (power) {
#pragma unroll
      for (int i = 0; i < 8; ++i) q[i] = x[i] * inverse;
    } else {
#pragma unroll 1
      for (int i = 0; i < 8; ++i) q[i] = x[i] / s;
    }
    return narrow8<C>(q);
  }
};

// Eight neighbouring elements as they are, and the largest of their magnitudes'
// bits (which order as the magnitudes do; NaN above infinity).
template <typename E>
struct Row8 {
  using R = typename E::raw;
  static constexpr int kWords = 2 * sizeof(R);  // of 32 bits
  static constexpr uint32_t kInfinity =
      std::is_same<E, F32>::value ? 0x7f800000u : std::is_same<E, BF16>::value ? 0x7f80u : 0x7c00u;
  Pack<uint32_t, 4> v[kWords / 4];
  __device__ __forceinline__ void load(const R* p) {
#pragma unroll
    for (int j = 0; j < kWords / 4; ++j)
      v[j] = load_pack<uint32_t, 4>(reinterpret_cast<const uint32_t*>(p) + 4 * j);
  }
  __device__ __forceinline__ void widen(float* x) const {
    const Pack<R, 8> r = __builtin_bit_cast(Pack<R, 8>, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) x[j] = E::load(r.v[j]);
  }
};
typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
// top = the larger of top and the row's, two 16-bit ones side by side.
template <typename E>
__device__ __forceinline__ void see(const Row8<E>& r, bool there, uint32_t& top) {
#pragma unroll
  for (int j = 0; j < Row8<E>::kWords; ++j) {
    const uint32_t w = there ? r.v[j / 4].v[j % 4] : 0;
    if constexpr (std::is_same<E, F32>::value)
      top = max(top, w & 0x7fffffffu);
    else
      top = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(
                                             __builtin_bit_cast(u16x2_t, top),
                                             __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu)));
  }
}

__device__ __forceinline__ uint32_t wave_max(uint32_t v, int lane) {
  auto as_float = [](uint32_t u) { return __builtin_bit_cast(float, u); };
  auto as_uint = [](float f) { return __builtin_bit_cast(uint32_t, f); };
  v = max(v, as_uint(dpp_move<0xB1>(as_float(v))));
  v = max(v, as_uint(dpp_move<0x4E>(as_float(v))));
  v = max(v, as_uint(dpp_move<0x141>(as_float(v))));
  v = max(v, as_uint(dpp_move<0x140>(as_float(v))));
  v = max(v, as_uint(lane_xor16(as_float(v), lane)));
  return max(v, as_uint(lane_xor32(as_float(v), lane)));
}

constexpr int kKept = 4;  // rounds of rows that a wave keeps between its two passes

// K or V of one (block, KV head), by one wave. `tok`: the call's row of every
// offset of the block, -1 where none. A row is spread over LPR lanes, eight
// values each; the rows of the first kKept rounds (a block of 16 of 128 dims)
// are read once, all together, those of larger blocks a second time, from the
// caches. No load waits for a branch: where there is no row, row 0 is read.
template <typename E, typename C, int LPR>
__device__ __forceinline__ void append_block(const typename E::raw* src, int64_t ts, uint8_t* dst,
                                             int64_t c_ts, float* scale, const int* tok,
                                             int num_tokens, int block_size, int first,
                                             int lane) {
  constexpr int kStep = kWave / LPR;  // rows at once
  const int grp = lane / LPR, d0 = lane % LPR * 8;
  const float old = *scale;  // of use where first > 0
  // A plan that is not this call's may name any row.
  auto row_of = [&](int o) {
    const int t = tok[min(o, block_size - 1)];
    return o < block_size && t < num_tokens ? t : -1;
  };
  int row[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) row[i] = row_of(grp + i * kStep);
  Row8<E> kept[kKept];
#pragma unroll
  for (int i = 0; i < kKept; ++i) kept[i].load(src + max(row[i], 0) * ts + d0);
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kKept; ++i) see<E>(kept[i], row[i] >= 0, top);
  for (int o = grp + kKept * kStep; o < block_size; o += kStep) {
    const int t = row_of(o);
    Row8<E> r;
    r.load(src + max(t, 0) * ts + d0);
    see<E>(r, t >= 0, top);
  }
  if constexpr (!std::is_same<E, F32>::value) top = max(top & 0xffffu, top >> 16);
  top = __builtin_amdgcn_readfirstlane(wave_max(top, lane));
  bool odd = false;  // a value that is not finite
  float most;
  if (top < Row8<E>::kInfinity) {
    most = std::is_same<E, F32>::value ? __uint_as_float(top)
                                       : E::load(static_cast<typename E::raw>(top));
  } else {  // the largest of those that are
    odd = true;
    most = 0.f;
    for (int o = grp; o < block_size; o += kStep) {
      const int t = row_of(o);
      if (t < 0) continue;
      float x[8];
      load8<E>(src + t * ts + d0, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float a = fabsf(x[i]);
        most = a < INFINITY ? fmaxf(most, a) : most;
      }
    }
    most = xor_max<1, kWave>(most);
  }
  const float need = !C::kHasNan && odd ? NAN : least_scale<C>(most);
  float now = need;
  if (first > 0 && !(old <= need)) now = need != need ? need : old;
  const Divisor by(now);
#pragma unroll
  for (int i = 0; i < kKept; ++i) {
    if (row[i] < 0) continue;
    float x[8];
    kept[i].widen(x);
    *reinterpret_cast<Codes8*>(dst + (grp + i * kStep) * c_ts + d0) = by.encode<C>(x);
  }
  for (int o = grp + kKept * kStep; o < block_size; o += kStep) {
    const int t = row_of(o);
    if (t < 0) continue;
    float x[8];
    load8<E>(src + t * ts + d0, x);
    *reinterpret_cast<Codes8*>(dst + o * c_ts + d0) = by.encode<C>(x);
  }
  if (first > 0 && now != old && now == now) {  // the rows that are held, again
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
  if (lane == 0 && (first == 0 || now != old)) *scale = now;
}

// One block of kHeads KV heads, K and V of each by a wave.
template <typename E, typename C, int LPR>
__device__ __forceinline__ void append_heads(const AppendArgs& a, int64_t blk, const int* tok,
                                             int first) {
  using R = typename E::raw;
  const QuantCache& c = a.c;
  const int wave = threadIdx.x / kWave;
  const int64_t head = blockIdx.y * kHeads + wave / 2;
  if (head >= c.heads) return;
  const bool is_v = wave & 1;
  const R* src = static_cast<const R*>(is_v ? a.values : a.keys) + head * (is_v ? a.v_hs : a.k_hs);
  uint8_t* dst = const_cast<uint8_t*>(is_v ? c.v : c.k) + blk * c.bs + head * c.hs;
  float* scale = const_cast<float*>(is_v ? c.vs : c.ks) + blk * c.s_bs + head * c.s_hs;
  append_block<E, C, LPR>(src, is_v ? a.v_ts : a.k_ts, dst, c.ts, scale, tok, a.num_tokens,
                          c.block_size, first, threadIdx.x % kWave);
}

// Few rows: workgroup = list entry x kHeads KV heads. It reads the whole list for
// the rows of its block, and goes on if its own has the lowest offset.
template <typename E, typename C, int LPR>
__global__ __launch_bounds__(kAppendThreads) void append_scan_kernel(const AppendArgs a) {
  extern __shared__ int s_tok[];  // [block_size]
  __shared__ int s_first;
  const int tid = threadIdx.x;
  const QuantCache& c = a.c;
  const int64_t end = static_cast<int64_t>(c.num_blocks) * c.block_size;
  const int t0 = blockIdx.x;
  const int64_t mine = slot_of(a.slots, a.is64, t0, end);
  const int64_t before = t0 > 0 ? slot_of(a.slots, a.is64, t0 - 1, end) : -1;
  if (mine < 0 || (before >= 0 && before < mine &&
                   before >> c.log2_block == mine >> c.log2_block))
    return;  // the whole workgroup
  for (int i = tid; i < c.block_size; i += kAppendThreads) s_tok[i] = -1;
  if (tid == 0) s_first = c.block_size;
  __syncthreads();
  for (int t = tid; t < a.num_tokens; t += kAppendThreads) {
    const int64_t u = slot_of(a.slots, a.is64, t, end);
    if (u >= 0 && u >> c.log2_block == mine >> c.log2_block) {
      const int o = static_cast<int>(u & (c.block_size - 1));
      atomicMax(&s_tok[o], t);
      atomicMin(&s_first, o);
    }
  }
  __syncthreads();
  if (s_tok[s_first] != t0) return;
  append_heads<E, C, LPR>(a, mine >> c.log2_block, s_tok, s_first);
}

// Many: kPerChunk workgroups x kHeads KV heads for each chunk of the plan.
template <typename E, typename C, int LPR>
__global__ __launch_bounds__(kAppendThreads) void append_planned_kernel(const AppendArgs a) {
  const QuantCache& c = a.c;
  const int64_t base = static_cast<int64_t>(blockIdx.x / kPerChunk) * kChunk;
  for (int i = blockIdx.x % kPerChunk; i < kChunk; i += kPerChunk) {
    const PlanBlock b = a.plan.blocks[base + i];
    if (b.block == kEnd) return;
    if (b.block < 0 || b.block >= c.num_blocks || b.first < 0) continue;
    append_heads<E, C, LPR>(a, b.block, a.plan.tok + (base + i) * c.block_size, b.first);
  }
}

// A wave reads an output row, eight values a lane at a time; whose row it is is
// searched for in scalars. Bound by HBM: one context of 30000 tokens in bf16 (184
// MB) takes 30.3 us a layer, 6.1 TB/s. With stores through the caches it took
// 38.7, with two and four rows a wave (fewer and longer waves) 40.6 and 43.7.
template <typename E, typename C>
__global__ __launch_bounds__(kGatherThreads) void gather_kernel(
    const QuantCache c, const int32_t* __restrict__ tables, int64_t t_stride, int t_width,
    const int32_t* __restrict__ cu_k, int num_requests, int total_rows, int log2_dim,
    typename E::raw* __restrict__ k_out, typename E::raw* __restrict__ v_out) {
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  const ConstI32* cu = (const ConstI32*)cu_k;
  const int row = __builtin_amdgcn_readfirstlane(static_cast<int>(
      blockIdx.x * (kGatherThreads / kWave) + threadIdx.x / kWave));
  if (row >= total_rows) return;
  int req = 0, hi = num_requests - 1;  // the last request with cu_k <= row
  while (req < hi) {
    const int mid = (req + hi + 1) >> 1;
    if (cu[mid] <= row) req = mid; else hi = mid - 1;
  }
  const int pos = row - cu[req];
  int64_t blk = -1;
  if (pos >= 0 && pos >> c.log2_block < t_width)
    blk = ((const ConstI32*)tables)[req * t_stride + (pos >> c.log2_block)];
  const bool there = blk >= 0 && blk < c.num_blocks;
  if (!there) blk = 0;  // read, and left out
  const int64_t at = blk * c.bs + (pos & (c.block_size - 1)) * c.ts;
  const int elems = c.heads << log2_dim;
  for (int e = threadIdx.x % kWave * 8; e < elems; e += kWave * 8) {
    const int64_t head = e >> log2_dim;
    const int64_t from = at + head * c.hs + (e & (c.dim - 1));
    const Codes8 k = *reinterpret_cast<const Codes8*>(c.k + from);
    const Codes8 v = *reinterpret_cast<const Codes8*>(c.v + from);
    const float ks = c.ks[blk * c.s_bs + head * c.s_hs];
    const float vs = c.vs[blk * c.s_bs + head * c.s_hs];
    float x[8], y[8];
    widen8<C>(k, x);
    widen8<C>(v, y);
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      x[j] = there ? x[j] * ks : 0.f;
      y[j] = there ? y[j] * vs : 0.f;
    }
    const int64_t to = static_cast<int64_t>(row) * elems + e;
    store8_past<E>(k_out + to, x);
    store8_past<E>(v_out + to, y);
  }
}

}  // namespace
}  // namespace mi

extern "C" int64_t mi_quant_append_plan_bytes(int32_t num_tokens, int32_t block_size,
                                              int32_t num_blocks) {
  if (num_tokens <= 0 || num_blocks <= 0 || !mi::is_pow2(block_size)) return 0;
  return mi::append_plan_of(nullptr, num_tokens, block_size, num_blocks).bytes;
}

extern "C" int32_t mi_quant_append_plan(const void* slots, int32_t slots_are_int64,
                                        int32_t num_tokens, int32_t block_size,
                                        int32_t num_blocks, void* plan, int64_t plan_bytes,
                                        void* stream) {
  using namespace mi;
  clear_error();
  const std::string fn = "mi_quant_append_plan";
  if (num_tokens < 0 || num_blocks <= 0)
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": invalid sizes");
  if (!is_pow2(block_size))
    return fail(MI_ERR_INVALID_ARGUMENT, fn + ": block_size must be a power of two");
  if (num_tokens == 0) return MI_OK;
  if (!slots || !plan) return fail(MI_ERR_INVALID_ARGUMENT, fn + ": null pointer");
  const AppendPlan p = append_plan_of(plan, num_tokens, block_size, num_blocks);
  if (plan_bytes < p.bytes || reinterpret_cast<uintptr_t>(plan) % 8 != 0)
    return fail(MI_ERR_WORKSPACE, fn + ": plan needs " + std::to_string(p.bytes) +
                                      " bytes, 8-byte aligned");
  const uint32_t grid = (num_tokens - 1) / kChunk + 1;
  const int64_t end = static_cast<int64_t>(num_blocks) * block_size;
  const hipStream_t s = static_cast<hipStream_t>(stream);
  append_map_kernel<<<grid, kChunk, 0, s>>>(slots, slots_are_int64, num_tokens, end, p.rows);
  append_blocks_kernel<<<grid, kChunk, 0, s>>>(slots, slots_are_int64, num_tokens, end,
                                               ilog2(block_size), p);
  return check_launch("mi_quant_append_plan");
}

extern "C" int32_t mi_quant_append(
    const void* keys, int64_t key_token_stride, int64_t key_head_stride, const void* values,
    int64_t value_token_stride, int64_t value_head_stride, void* key_cache, void* value_cache,
    int64_t cache_block_stride, int64_t cache_token_stride, int64_t cache_head_stride,
    float* key_scales, float* value_scales, int64_t scale_block_stride,
    int64_t scale_head_stride, const void* slots, int32_t slots_are_int64, const void* plan,
    int64_t plan_bytes, int32_t num_tokens, int32_t num_kv_heads, int32_t head_dim,
    int32_t block_size, int32_t num_blocks, int32_t dtype, int32_t code, void* stream) {
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
  if (plan == nullptr && num_tokens > kMaxScan)
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
  a.is64 = slots_are_int64;
  a.num_tokens = num_tokens;
  if (plan != nullptr) {
    a.plan = append_plan_of(const_cast<void*>(plan), num_tokens, block_size, num_blocks);
    if (plan_bytes < a.plan.bytes || reinterpret_cast<uintptr_t>(plan) % 8 != 0)
      return fail(MI_ERR_WORKSPACE, fn + ": plan needs " + std::to_string(a.plan.bytes) +
                                        " bytes, 8-byte aligned");
  }
  const int64_t groups =
      plan == nullptr ? num_tokens
                      : (static_cast<int64_t>(num_tokens - 1) / kChunk + 1) * kPerChunk;
  const dim3 grid(static_cast<uint32_t>(groups), (num_kv_heads - 1) / kHeads + 1);
  const size_t lds = sizeof(int) * block_size;
  return with_types(dtype, code, [&](auto e, auto c) {
    using E = decltype(e);
    using C = decltype(c);
    auto go = [&](auto scan, auto planned) {
      if (plan == nullptr)
        scan<<<grid, kAppendThreads, lds, static_cast<hipStream_t>(stream)>>>(a);
      else
        planned<<<grid, kAppendThreads, lds, static_cast<hipStream_t>(stream)>>>(a);
      return check_launch("mi_quant_append");
    };
    switch (head_dim) {
      case 16: return go(append_scan_kernel<E, C, 2>, append_planned_kernel<E, C, 2>);
      case 32: return go(append_scan_kernel<E, C, 4>, append_planned_kernel<E, C, 4>);
      case 64: return go(append_scan_kernel<E, C, 8>, append_planned_kernel<E, C, 8>);
      case 128: return go(append_scan_kernel<E, C, 16>, append_planned_kernel<E, C, 16>);
      default: return go(append_scan_kernel<E, C, 32>, append_planned_kernel<E, C, 32>);
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
  const QuantCache cache = make_quant_cache(
      key_cache, value_cache, cache_block_stride, cache_token_stride, cache_head_stride,
      key_scales, value_scales, scale_block_stride, scale_head_stride, num_kv_heads, head_dim,
      block_size, num_blocks);
  return with_types(dtype, code, [&](auto e, auto c) {
    using E = decltype(e);
    using C = decltype(c);
    using R = typename E::raw;
    constexpr int kRows = kGatherThreads / kWave;
    gather_kernel<E, C><<<(total_rows - 1) / kRows + 1, kGatherThreads, 0,
                          static_cast<hipStream_t>(stream)>>>(
        cache, block_tables, block_table_stride, block_table_width, cu_seqlens_k, num_requests,
        total_rows, ilog2(head_dim), static_cast<R*>(key_out), static_cast<R*>(value_out));
    return check_launch("mi_quant_gather");
  });
}
