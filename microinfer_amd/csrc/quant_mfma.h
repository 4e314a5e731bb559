// Matrix-instruction pieces shared by the attention kernels over an 8-bit K/V
// cache: codes widened to bf16 or f16 (exactly: both types have at most eight
// significant bits), float32 values split into bf16 parts.
#pragma once

#include "quant.h"

namespace mi {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x16_t __attribute__((ext_vector_type(16)));
typedef int int2v_t __attribute__((ext_vector_type(2)));

typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));

// What a query meets the codes as, with all of its bits: 16-bit ones as they are,
// f32 ones in three bf16 parts.
template <typename E>
using QueryOperand =
    typename std::conditional<std::is_same<E, F16>::value, f16x8_t, bf16x8_t>::type;
template <typename E>
constexpr int kQueryParts = std::is_same<E, F32>::value ? 3 : 1;

struct Word4 {
  uint32_t w[4];
};

// Two of a word's codes (the upper two: HIGH) as a pair of bf16.
template <typename C, bool HIGH>
__device__ __forceinline__ uint32_t widen_pair(uint32_t w) {
  if constexpr (std::is_same<C, E4M3>::value) {
    return __builtin_bit_cast(uint32_t,
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, HIGH));
  } else {
    constexpr int s = HIGH ? 16 : 0;
    const float lo = static_cast<float>(static_cast<int8_t>(w >> s));
    const float hi = static_cast<float>(static_cast<int8_t>(w >> (s + 8)));
    // Eight significant bits: the upper halves of the float32 values.
    return __builtin_amdgcn_perm(__float_as_uint(hi), __float_as_uint(lo), 0x07060302u);
  }
}

// The same as a pair of f16, which hold the codes as exactly.
template <typename C, bool HIGH>
__device__ __forceinline__ uint32_t widen_pair_f16(uint32_t w) {
  if constexpr (std::is_same<C, E4M3>::value) {
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(w, 1.f, HIGH));
  } else {
    // 0x6400 + u is 1024 + u, for u = code + 128.
    const uint32_t u = w ^ 0x80808080u;
    const uint32_t x = __builtin_amdgcn_perm(0x64646464u, u, HIGH ? 0x04030402u : 0x04010400u);
    const f16x2_t bias = {static_cast<_Float16>(1152.f), static_cast<_Float16>(1152.f)};
    return __builtin_bit_cast(uint32_t, __builtin_bit_cast(f16x2_t, x) - bias);
  }
}

template <typename C>
__device__ __forceinline__ f16x8_t widen_operand_f16(uint32_t lo, uint32_t hi) {
  Word4 r;
  r.w[0] = widen_pair_f16<C, false>(lo);
  r.w[1] = widen_pair_f16<C, true>(lo);
  r.w[2] = widen_pair_f16<C, false>(hi);
  r.w[3] = widen_pair_f16<C, true>(hi);
  return __builtin_bit_cast(f16x8_t, r);
}

// Eight codes (two words) as a matrix operand.
template <typename C>
__device__ __forceinline__ bf16x8_t widen_operand(uint32_t lo, uint32_t hi) {
  Word4 r;
  r.w[0] = widen_pair<C, false>(lo);
  r.w[1] = widen_pair<C, true>(lo);
  r.w[2] = widen_pair<C, false>(hi);
  r.w[3] = widen_pair<C, true>(hi);
  return __builtin_bit_cast(bf16x8_t, r);
}

// Eight codes as an operand of either type.
template <typename V, typename C>
__device__ __forceinline__ V widen(uint32_t lo, uint32_t hi) {
  if constexpr (std::is_same<V, bf16x8_t>::value)
    return widen_operand<C>(lo, hi);
  else
    return widen_operand_f16<C>(lo, hi);
}

// x = part[0] + part[1] + ... in bf16 (or f16), each what the ones before
// leave, rounded.
template <int N, typename V>
__device__ __forceinline__ void split8(const float* x, V* part) {
  using T = typename std::conditional<std::is_same<V, bf16x8_t>::value, __bf16, _Float16>::type;
  // The compiler may fuse a product with its conversion to f16, which rounds
  // once instead of twice, in one of its uses: parts would not fit each other.
  static_assert(N == 1 || std::is_same<T, __bf16>::value, "parts are bf16");
  float rest[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) rest[i] = x[i];
#pragma unroll
  for (int n = 0; n < N; ++n) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const T r = static_cast<T>(rest[i]);
      part[n][i] = r;
      if (n + 1 < N) rest[i] -= static_cast<float>(r);
    }
  }
}

// Direct global -> LDS load of 4 bytes per lane (lane i's at lds_dst + 4 i),
// untracked by the compiler like lds_load16.
__device__ __forceinline__ void lds_load4(const void* src, const void* lds_dst) {
  const uint32_t lds = static_cast<uint32_t>(reinterpret_cast<uintptr_t>(
      (const __attribute__((address_space(3))) void*)(lds_dst)));
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dword %0, off"
               :
               : "v"(src), "s"(lds)
               : "memory", "m0");
}

// Eight one-byte elements, transposed across each group of 16 lanes
// (ds_read_b64_tr_b8): lane i of a group receives byte i % 8 of the eight
// bytes read by lanes i / 8, i / 8 + 2, ..., i / 8 + 14.
__device__ __forceinline__ int2v_t read_tr8(const void* lds) {
  return __builtin_amdgcn_ds_read_tr8_b64_v2i32(
      (__attribute__((address_space(3))) int2v_t*)(lds));
}

// MFMA varlen kernel (quant_prefill.hip): its workspace (0: it does not take
// calls of these sizes), its plan in the workspace, and its launch with that.
int64_t quant_prefill_workspace(int32_t num_rows, int32_t num_seqs, int32_t group, int32_t heads,
                                int32_t dim, int32_t block_size);
int32_t launch_quant_prefill_plan(const int32_t* cu_q, const int32_t* cu_k, int32_t num_rows,
                                  int32_t num_seqs, int32_t group, int32_t heads, int32_t dim,
                                  void* workspace, hipStream_t stream);
int32_t launch_quant_prefill_mfma(const QuantAttnArgs& a, int32_t dtype, int32_t code,
                                  void* workspace, hipStream_t stream);

// MFMA kernel of few rows (quant_decode.hip): whether it takes caches of this
// shape, the workgroups that share a sequence's `rows` at a KV head, the launch;
// the lengths of requests for its plan.
bool quant_decode_mfma_takes(int32_t head_dim, int32_t block_size);
bool quant_mfma_aligned(const QuantCache& c);
int32_t quant_decode_row_groups(int32_t rows, int32_t head_dim);
int32_t launch_quant_decode_mfma(QuantAttnArgs a, int32_t rows, int32_t dtype, int32_t code,
                                 hipStream_t stream);
int32_t launch_few_rows(const int32_t* cu_q, const int32_t* cu_k, int32_t num_seqs, int32_t* lens,
                        int32_t* counters, int32_t num_counters, hipStream_t stream);

}  // namespace mi
