// Shared by the kernels over an 8-bit K/V cache: the codes and their
// conversions, the arguments, the argument checks.
#pragma once

#include "mi_common.h"
#include "mi_quant.h"
#include "paged_attention.h"

namespace mi {

typedef float f32x2_t __attribute__((ext_vector_type(2)));

// float8 e4m3: gfx950 converts both ways in hardware, to nearest even; NaN and
// what lies beyond 464 become NaN.
struct E4M3 {
  static constexpr float kMost = 448.f;
  static constexpr bool kHasNan = true;
  // Bytes 0 .. 3 of a word to float32.
  static __device__ __forceinline__ void widen4(uint32_t w, float* x) {
    const f32x2_t lo = __builtin_amdgcn_cvt_pk_f32_fp8(w, false);
    const f32x2_t hi = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = lo.x;
    x[1] = lo.y;
    x[2] = hi.x;
    x[3] = hi.y;
  }
  static __device__ __forceinline__ uint32_t narrow4(const float* x) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(x[0], x[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(x[2], x[3], w, true);
  }
};

struct Int8 {
  static constexpr float kMost = 127.f;
  static constexpr bool kHasNan = false;
  static __device__ __forceinline__ void widen4(uint32_t w, float* x) {
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = static_cast<float>(static_cast<int8_t>(w >> (8 * i)));
  }
  // NaN becomes 0: its scale is NaN.
  static __device__ __forceinline__ uint32_t narrow4(const float* x) {
    uint32_t w = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      w |= (static_cast<uint32_t>(static_cast<int32_t>(rintf(x[i]))) & 0xffu) << (8 * i);
    return w;
  }
};

// Eight codes, a lane's share of a row.
struct Codes8 {
  uint32_t lo, hi;
};
template <typename C>
__device__ __forceinline__ void widen8(Codes8 c, float* x) {
  C::widen4(c.lo, x);
  C::widen4(c.hi, x + 4);
}
template <typename C>
__device__ __forceinline__ Codes8 narrow8(const float* x) {
  return Codes8{C::narrow4(x), C::narrow4(x + 4)};
}

// Eight neighbouring elements as float32.
template <typename E>
__device__ __forceinline__ void load8(const typename E::raw* p, float* x) {
  using R = typename E::raw;
  constexpr int N = 16 / sizeof(R);
#pragma unroll
  for (int j = 0; j < 8; j += N) {
    const Pack<R, N> v = load_pack<R, N>(p + j);
#pragma unroll
    for (int i = 0; i < N; ++i) x[j + i] = E::load(v.v[i]);
  }
}

// The cache of mi_quant.h.
struct QuantCache {
  const uint8_t* k;
  const uint8_t* v;
  int64_t bs, ts, hs;  // bytes
  const float* ks;
  const float* vs;
  int64_t s_bs, s_hs;  // elements
  int32_t heads, dim, block_size, log2_block, num_blocks;
};

struct QuantAttnArgs {
  const void* q;
  int64_t q_ts, q_hs;
  QuantCache c;
  const int32_t* tables;
  int64_t t_stride;
  int32_t t_width;
  const int32_t* cu_q;  // varlen (null: decode)
  const int32_t* cu_k;
  void* out;
  int64_t o_ts, o_hs;
  float* ws_acc;  // partials: [items, Hkv, rows, D] unnormalised sums
  float* ws_ml;   // [items, Hkv, rows, 2]: log2-domain maximum, sum
  int32_t* counters;  // [num_seqs, row groups, Hkv], zero on entry and exit
  const PlanItem* plan;  // decode: [max_items]
  int32_t num_seqs, num_rows, group, max_items;
  // MFMA kernel of few rows: at most so many of a sequence's at a KV head, in
  // so many groups.
  int32_t head_rows, row_groups;
  uint32_t group_inverse;  // 2^24 / group, rounded up
  float scale_log2;
};

// Whether an item names a sequence and partials that are there: any memory may be
// taken for a plan (one that a graph has not replayed yet), so no sum that can overflow.
__device__ __forceinline__ bool item_fits(const PlanItem& it, const QuantAttnArgs& a) {
  return it.seq >= 0 && it.seq < a.num_seqs && it.part >= 0 && it.part < it.nparts &&
         it.first_item >= 0 && it.nparts <= a.max_items - it.first_item;
}

// Host side: checks of a cache's description. Returns an MI_* status.
int32_t check_quant_cache(const std::string& fn, const void* key_cache, const void* value_cache,
                          int64_t block_stride, int64_t token_stride, int64_t head_stride,
                          const float* key_scales, const float* value_scales,
                          int64_t scale_block_stride, int64_t scale_head_stride,
                          int32_t num_kv_heads, int32_t head_dim, int32_t block_size,
                          int32_t num_blocks, int32_t dtype, int32_t code);
QuantCache make_quant_cache(const void* key_cache, const void* value_cache, int64_t block_stride,
                            int64_t token_stride, int64_t head_stride, const float* key_scales,
                            const float* value_scales, int64_t scale_block_stride,
                            int64_t scale_head_stride, int32_t num_kv_heads, int32_t head_dim,
                            int32_t block_size, int32_t num_blocks);

// Whether rows at `p` with these element strides are whole 16-byte vectors.
inline bool whole_vectors(const void* p, int64_t s0, int64_t s1, int32_t dtype) {
  const int64_t vec = 16 / static_cast<int64_t>(dtype_size(dtype));
  return reinterpret_cast<uintptr_t>(p) % 16 == 0 && s0 % vec == 0 && s1 % vec == 0;
}

int32_t launch_quant_vector(const QuantAttnArgs& a, int32_t dtype, int32_t code,
                            hipStream_t stream);

// Calls f with the element and the code type of the two codes.
template <typename F>
int32_t with_types(int32_t dtype, int32_t code, F f) {
  auto with_code = [&](auto e) {
    return code == MI_CODE_E4M3 ? f(e, E4M3{}) : f(e, Int8{});
  };
  if (dtype == MI_DTYPE_BF16) return with_code(BF16{});
  if (dtype == MI_DTYPE_F16) return with_code(F16{});
  return with_code(F32{});
}

}  // namespace mi
