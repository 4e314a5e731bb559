// Attention over an 8-bit K/V cache without matrix instructions: every head
// size, group and block size (the MFMA kernels take the common ones).
//
// Workgroup = (decode: plan item; varlen: query row) x KV head x up to four of
// its query heads. A cache row is spread over LPR = D / 8 lanes, eight codes
// each; the lane groups of the four waves take positions in turn, each with an
// online softmax of its own in the log2 domain, merged through LDS at the end.
// Scores meet the K scale after the sum over dims, weights the V scale.
// Decode partitions publish (acc, m, l); the last arrival merges them in
// partition order. Bound by its vector instructions: 16 contexts of 1000, 16 / 8
// heads, four layers, us: heads of 32 79, of 128 in blocks of 8 205 (55 on MFMA in
// blocks of 16, with 32 / 8); 64 of 128-2048 in blocks of 8 645 (129). In varlen calls
// every row reads its whole context: 512 tokens on 7700 10900 (392), six prompts of
// 40-1400 17300 (380).
#include "quant.h"

namespace mi {
namespace {

constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kHeads = 4;  // query heads of a workgroup

template <typename E, typename C, int LPR>
__global__ __launch_bounds__(kThreads) void quant_vector_kernel(const QuantAttnArgs a,
                                                                int chunks) {
  using R = typename E::raw;
  constexpr int D = 8 * LPR;
  constexpr int kGroups = kThreads / LPR;  // lane groups of the workgroup
  __shared__ float s_acc[kGroups][kHeads][D];
  __shared__ float s_m[kGroups][kHeads], s_l[kGroups][kHeads];
  __shared__ int s_arrived;
  const QuantCache& c = a.c;
  const int tid = threadIdx.x;
  const int grp = tid / LPR, d0 = tid % LPR * 8;
  const int chunk = blockIdx.x % chunks;
  const int head = blockIdx.x / chunks % c.heads;
  const int w = blockIdx.x / chunks / c.heads;
  const int G = a.group;
  const int g0 = chunk * kHeads;

  int seq, row, begin, end;
  PlanItem it{};
  it.nparts = 1;
  if (a.cu_q != nullptr) {
    row = w;
    int lo = 0, hi = a.num_seqs - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.cu_q[mid] <= row) lo = mid; else hi = mid - 1;
    }
    seq = lo;
    const int64_t ctx = static_cast<int64_t>(a.cu_k[lo + 1]) - a.cu_k[lo];
    const int64_t seen = ctx - (a.cu_q[lo + 1] - row) + 1;
    begin = 0;
    end = static_cast<int>(
        max(int64_t(0), min(seen, static_cast<int64_t>(a.t_width) * c.block_size)));
    // Rows of no request stay as they were, as on the MFMA kernels (uniform).
    if (row < a.cu_q[lo] || row >= a.cu_q[lo + 1]) return;
  } else {
    it = a.plan[w];
    if (!item_fits(it, a)) return;  // unused slot
    seq = row = it.seq;
    const int most = a.t_width << c.log2_block;
    begin = min(max(it.blk_begin, 0), a.t_width) << c.log2_block;
    end = min(min(max(it.ctx, 0), most), min(max(it.blk_end, 0), a.t_width) << c.log2_block);
  }

  float q[kHeads][8], acc[kHeads][8], m[kHeads], l[kHeads];
#pragma unroll
  for (int g = 0; g < kHeads; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) q[g][i] = acc[g][i] = 0.f;
    if (g0 + g < G)
      load8<E>(static_cast<const R*>(a.q) + row * a.q_ts +
                   static_cast<int64_t>(head * G + g0 + g) * a.q_hs + d0, q[g]);
  }
  const int32_t* table = a.tables + seq * a.t_stride;
  for (int p0 = begin; p0 < end; p0 += kGroups) {
    const int p = p0 + grp;
    int blk = -1;
    if (p < end) blk = table[p >> c.log2_block];
    const bool ok = blk >= 0 && blk < c.num_blocks;
    float k[8] = {}, v[8] = {};
    float ks = 0.f, vs = 0.f;
    if (ok) {
      const int64_t at = blk * c.bs + (p & (c.block_size - 1)) * c.ts + head * c.hs + d0;
      const int64_t s = blk * c.s_bs + head * c.s_hs;
      widen8<C>(*reinterpret_cast<const Codes8*>(c.k + at), k);
      widen8<C>(*reinterpret_cast<const Codes8*>(c.v + at), v);
      ks = c.ks[s] * a.scale_log2;
      vs = c.vs[s];
    }
#pragma unroll
    for (int g = 0; g < kHeads; ++g) {
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < 8; ++i) dot = fmaf(q[g][i], k[i], dot);
      const float score = group_sum<LPR>(dot) * ks;
      if (!ok) continue;
      const float mnew = fmaxf(m[g], score);
      const float base = mnew == -INFINITY ? 0.f : mnew;
      const float alpha = fast_exp2(m[g] - base);
      const float weight = fast_exp2(score - base);
      l[g] = fmaf(l[g], alpha, weight);
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[g][i] = fmaf(acc[g][i], alpha, weight * vs * v[i]);
      m[g] = mnew;
    }
  }
#pragma unroll
  for (int g = 0; g < kHeads; ++g) {
#pragma unroll
    for (int i = 0; i < 8; ++i) s_acc[grp][g][d0 + i] = acc[g][i];
    if (d0 == 0) {
      s_m[grp][g] = l[g] == l[g] ? m[g] : 0.f;  // NaN weighs, whatever its maximum
      s_l[grp][g] = l[g];
    }
  }
  __syncthreads();
  const int heads = min(kHeads, G - g0);
  R* out = static_cast<R*>(a.out) + row * a.o_ts;
  const int64_t unit = static_cast<int64_t>(it.first_item + it.part) * c.heads + head;
  for (int e = tid; e < heads * D; e += kThreads) {
    const int g = e / D, d = e % D;
    float mx = -INFINITY, ls = 0.f, os = 0.f;
    for (int i = 0; i < kGroups; ++i) mx = fmaxf(mx, s_m[i][g]);
    for (int i = 0; i < kGroups; ++i) {
      const float f = s_m[i][g] == -INFINITY ? 0.f : fast_exp2(s_m[i][g] - mx);
      ls = fmaf(f, s_l[i][g], ls);
      os = fmaf(f, s_acc[i][g][d], os);
    }
    if (it.nparts == 1) {
      out[(head * G + g0 + g) * a.o_hs + d] = E::store(ls == 0.f ? 0.f : os / ls);
    } else {
      const int64_t r = unit * G + g0 + g;
      store_coherent(a.ws_acc + r * D + d, os);
      if (d == 0) {
        store_coherent(a.ws_ml + r * 2, mx);
        store_coherent(a.ws_ml + r * 2 + 1, ls);
      }
    }
  }
  if (it.nparts == 1) return;
  int32_t* counter = a.counters + static_cast<int64_t>(seq) * c.heads + head;
  wait_stores();
  __syncthreads();  // every thread's partials are at the coherent level
  if (tid == 0)
    s_arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_arrived != it.nparts * chunks - 1) return;
  for (int e = tid; e < G * D; e += kThreads) {
    const int g = e / D, d = e % D;
    float mx = -INFINITY, ls = 0.f, os = 0.f;
    for (int p = 0; p < it.nparts; ++p) {
      const int64_t r = (static_cast<int64_t>(it.first_item + p) * c.heads + head) * G + g;
      const float mp = load_coherent(a.ws_ml + r * 2);
      const float lp = load_coherent(a.ws_ml + r * 2 + 1);
      const float op = load_coherent(a.ws_acc + r * D + d);
      if (mp == -INFINITY) continue;
      const float mnew = fmaxf(mx, mp);
      const float fo = fast_exp2(mx - mnew), fp = fast_exp2(mp - mnew);
      ls = fmaf(ls, fo, lp * fp);
      os = fmaf(os, fo, op * fp);
      mx = mnew;
    }
    out[(head * G + g) * a.o_hs + d] = E::store(ls == 0.f ? 0.f : os / ls);
  }
  if (tid == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace

int32_t launch_quant_vector(const QuantAttnArgs& a, int32_t dtype, int32_t code,
                            hipStream_t stream) {
  const int chunks = (a.group - 1) / kHeads + 1;
  const int64_t items = a.cu_q != nullptr ? a.num_rows : a.max_items;
  const int64_t grid = items * a.c.heads * chunks;
  if (grid > (int64_t(1) << 31) - 1)
    return fail(MI_ERR_UNSUPPORTED, "quantized attention: too many rows for one launch");
  return with_types(dtype, code, [&](auto e, auto c) {
    using E = decltype(e);
    using C = decltype(c);
    auto go = [&](auto kernel) {
      kernel<<<static_cast<uint32_t>(grid), kThreads, 0, stream>>>(a, chunks);
      return check_launch("quantized attention");
    };
    switch (a.c.dim) {
      case 16: return go(quant_vector_kernel<E, C, 2>);
      case 32: return go(quant_vector_kernel<E, C, 4>);
      case 64: return go(quant_vector_kernel<E, C, 8>);
      case 128: return go(quant_vector_kernel<E, C, 16>);
      default: return go(quant_vector_kernel<E, C, 32>);
    }
  });
}

}  // namespace mi
