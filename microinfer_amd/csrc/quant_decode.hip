// Decode attention over an 8-bit K/V cache on MFMA: head_dim 64 or 128, up to
// 16 query heads per KV head, blocks of at least 16, queries of any type.
//
// out = softmax(scale * q . (k * ks)) (v * vs), with one ks and vs for each
// block and KV head. Bound by HBM for long contexts (two bytes a position and
// dim), by latency for few short ones.
//
//  * Workgroup = plan item (sequence, block range) x KV head, all its query
//    heads, so a cache row is read once. Its waves take tiles of 32 positions
//    in turn: two halves of 16, each in one block.
//  * Tiles come into a ring of LDS slots of the wave's own by direct loads
//    (waited for by count, so a slot per wave stays in flight), the four scales
//    of a tile with them.
//  * Scores S^T[pos][head] = K . Q^T on v_mfma_f32_16x16x32_bf16, a half at a
//    time; codes are widened to bf16 on their way from LDS, which loses nothing,
//    and a query comes in as many bf16 parts as hold all of its bits (1 for
//    bf16, 2 for f16, 3 for f32). The K scale meets the score in float32.
//  * The lanes that hold a tile's scores hold the weights that
//    O^T[dim][head] += V^T . P^T wants from them, with V's bytes transposed on
//    their way out of LDS (ds_read_b64_tr_b8). A weight times the V scale goes
//    in as two bf16 parts (three for f32 queries), so that it loses less than
//    the output's rounding: in bf16, whose range is float32's, however far
//    apart the scales of the blocks are.
//  * Online softmax in the log2 domain; the reference moves only when a score
//    exceeds it by more than 15.
//  * Waves are joined through LDS, partitions by their last arrival, in order.
#include "quant_mfma.h"

namespace mi {
namespace {

constexpr int kHalf = 16;   // positions of a half: one block's
constexpr int kTile = 32;   // positions of a tile
constexpr int kHeads = 16;  // MFMA columns
constexpr float kRescaleSlack = 15.f;

// One step of the running merge of partitions, in the log2 domain; an empty
// partition (mb = -inf) weighs nothing.
__device__ __forceinline__ void merge_step(float& mx, float& ls, float& os, float mb, float lb,
                                           float ob) {
  if (mb == -INFINITY) return;
  const float mnew = fmaxf(mx, mb);
  const float fo = mx == -INFINITY ? 0.f : fast_exp2(mx - mnew);
  const float fb = fast_exp2(mb - mnew);
  ls = fmaf(ls, fo, lb * fb);
  os = fmaf(os, fo, ob * fb);
  mx = mnew;
}

// LDS: a half's rows are D bytes, 16-byte chunk c of row r at cell
// r * (D / 16) + (c ^ swz(r)). LDS serves 16 cells of distinct place modulo 16
// at once: for K the 16 rows' chunk c, for V chunk c of rows r .. r + 7 of both
// halves.
template <int D>
__device__ __forceinline__ int swz_k(int r) {
  return D == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <int D>
__device__ __forceinline__ int swz_v(int r, int half) {
  return D == 128 ? ((r >> 1) & 3) ^ (4 * half) : ((r >> 2) & 1) ^ (2 * half);
}

template <typename E, typename C, int D, int NW, int NS>
__global__ __launch_bounds__(kWave * NW, NS == 1 ? 4 : 2) void quant_decode_kernel(const QuantAttnArgs a) {
  using R = typename E::raw;
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  constexpr int kParts = kQueryParts<E>;
  constexpr int kWeights = std::is_same<E, F32>::value ? 3 : 2;
  constexpr int kHalfBytes = kHalf * D;           // K or V of a half
  constexpr int kLoads = kHalfBytes / 1024;       // direct loads of one
  constexpr int kScaleBytes = 4 * kWave;          // the tile's scales, 16 times over
  constexpr int kSlotBytes = 4 * kHalfBytes + kScaleBytes;
  constexpr int kTileLoads = 4 * kLoads + 1;
  constexpr int kChunks = D / 16;
  constexpr int kSteps = D / 32;  // MFMAs of a half's scores
  constexpr int kRowsPerLoad = 1024 / D;
  static_assert(NS >= 1 && NS <= 2 && kHeads * D * 4 <= NS * kSlotBytes, "ring");

  __shared__ __attribute__((aligned(16))) char s_ring[NW * NS * kSlotBytes];
  __shared__ float s_m[NW][kHeads];
  __shared__ float s_l[NW][kHeads];
  __shared__ int s_arrived;

  const QuantCache& c = a.c;
  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int head = blockIdx.x % c.heads;
  const int w = blockIdx.x / c.heads;
  const int G = a.group;
  const int col = lane % 16;
  const int quad = lane / 16;

  // The item, checked so that a stale or foreign plan gives wrong attention
  // but no access out of bounds.
  typedef int32_t int8v __attribute__((ext_vector_type(8)));
  using ConstItem = __attribute__((address_space(4))) const int8v;
  const PlanItem it = __builtin_bit_cast(PlanItem, ((ConstItem*)(a.plan))[w]);
  if (it.seq < 0 || it.seq >= a.num_seqs || it.nparts < 1 || it.part < 0 ||
      it.part >= it.nparts || it.first_item < 0 || it.first_item + it.nparts > a.max_items)
    return;  // unused slot (uniform across the workgroup)
  const int seq = it.seq;
  const int lb = c.log2_block;
  const int ctx = min(max(it.ctx, 0), a.t_width << lb);
  const int blk_begin = max(it.blk_begin, 0);
  const int blk_end = min(it.blk_end, a.t_width);
  const int nparts = it.nparts;
  const int pos_begin = blk_begin << lb;
  const int pos_end = min(ctx, blk_end << lb);
  const int ntiles = pos_end > pos_begin ? (pos_end - pos_begin + kTile - 1) / kTile : 0;
  const ConstI32* ctab = (const ConstI32*)(a.tables + seq * a.t_stride);

  const uint8_t* kc = c.k + head * c.hs;
  const uint8_t* vc = c.v + head * c.hs;
  // Byte offsets of a lane's loads: load u of a half brings LDS cells 64 u +
  // lane, row u * kRowsPerLoad + lane / kChunks.
  uint32_t off_k[kLoads], off_v[2][kLoads];
#pragma unroll
  for (int u = 0; u < kLoads; ++u) {
    const int row = u * kRowsPerLoad + lane / kChunks;
    const int cell = lane % kChunks;
    const uint32_t at = static_cast<uint32_t>(row * static_cast<int>(c.ts));
    off_k[u] = at + (cell ^ swz_k<D>(row)) * 16;
    off_v[0][u] = at + (cell ^ swz_v<D>(row, 0)) * 16;
    off_v[1][u] = at + (cell ^ swz_v<D>(row, 1)) * 16;
  }
  // Lane i fetches scale i % 4 of a tile: K of the halves, then V.
  const float* my_scale = (lane & 2 ? c.vs : c.ks) + head * c.s_hs;
  char* my_ring = s_ring + wave * NS * kSlotBytes;

  // Starts tile k's loads into a slot. Bit j of the result: half j is there
  // (an invalid block reads block 0 and is masked).
  auto issue = [&](int slot, int k) -> int {
    const int p0 = pos_begin + k * kTile;
    char* dst = my_ring + slot * kSlotBytes;
    int mask = 0;
    int64_t at[2];
    int page[2];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      const int p = p0 + kHalf * j;
      // A half past the end reads the tile's first block.
      const int blk = ctab[(p < pos_end ? p : p0) >> lb];
      const bool ok = p < pos_end && blk >= 0 && blk < c.num_blocks;
      mask |= ok ? 1 << j : 0;
      page[j] = ok ? blk : 0;
      at[j] = ok ? blk * c.bs + (p & (c.block_size - 1)) * c.ts : 0;
    }
#pragma unroll
    for (int j = 0; j < 2; ++j) {
#pragma unroll
      for (int u = 0; u < kLoads; ++u) {
        lds_load16_sbase(kc + at[j], off_k[u], dst + j * kHalfBytes + u * 1024);
        lds_load16_sbase(vc + at[j], off_v[j][u], dst + (2 + j) * kHalfBytes + u * 1024);
      }
    }
    lds_load4(my_scale + static_cast<int64_t>(lane & 1 ? page[1] : page[0]) * c.s_bs,
              dst + 4 * kHalfBytes);
    return mask;
  };

  // Query operand of MFMA step 2 j + h: dims 16 (quad + 4 j) + 8 h .. + 7 of
  // head `col`, the order in which a lane reads K.
  bf16x8_t qf[kParts][kSteps];
  auto load_q = [&]() {
    const R* row = static_cast<const R*>(a.q) + seq * a.q_ts +
                   static_cast<int64_t>(head * G + col) * a.q_hs;
#pragma unroll
    for (int s = 0; s < kSteps; ++s) {
      float x[8] = {};
      if (col < G) load8<E>(row + 16 * (quad + 4 * (s / 2)) + 8 * (s % 2), x);
      bf16x8_t part[kParts];
      split8<kParts>(x, part);
#pragma unroll
      for (int n = 0; n < kParts; ++n) qf[n][s] = part[n];
    }
  };

  f32x4_t o[D / 16];
#pragma unroll
  for (int db = 0; db < D / 16; ++db) o[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = -INFINITY, l = 0.f;

  auto compute = [&](int k, const char* slot, int mask) {
    const f32x4_t scales = *reinterpret_cast<const f32x4_t*>(slot + 4 * kHalfBytes);
    Word4 kw[2][kSteps / 2];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
      for (int i = 0; i < kSteps / 2; ++i)
        kw[j][i] = *reinterpret_cast<const Word4*>(
            slot + j * kHalfBytes + col * D + ((quad + 4 * i) ^ swz_k<D>(col)) * 16);
    // Lane s of a group of 16 reads row 4 quad + (s / 2) % 4 of half s / 8.
    int2v_t vw[D / 16];
    {
      const int half = col / 8, row = 4 * quad + (col / 2) % 4;
      const char* base = slot + (2 + half) * kHalfBytes + row * D + 8 * (col & 1);
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        vw[db] = read_tr8(base + (db ^ swz_v<D>(row, half)) * 16);
    }
    const int p = pos_begin + k * kTile + 4 * quad;
    float sc[8];
    float tmax = -INFINITY;
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const bf16x8_t kf =
            widen_operand<C>(kw[j][i / 2].w[2 * (i % 2)], kw[j][i / 2].w[2 * (i % 2) + 1]);
#pragma unroll
        for (int n = 0; n < kParts; ++n)
          s = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kf, qf[n][i], s, 0, 0, 0);
      }
      const float factor = scales[j] * a.scale_log2;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[4 * j + i] =
            (mask >> j & 1) && p + kHalf * j + i < pos_end ? s[i] * factor : -INFINITY;
        tmax = fmaxf(tmax, sc[4 * j + i]);
      }
    }
    tmax = fmaxf(tmax, lane_xor16(tmax, lane));
    tmax = fmaxf(tmax, lane_xor32(tmax, lane));
    if (__ballot(tmax > m + kRescaleSlack) != 0) {
      const float mnew = fmaxf(m, tmax);
      const float alpha = mnew == -INFINITY ? 1.f : fast_exp2(m - mnew);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < D / 16; ++db) o[db] *= alpha;
      m = mnew;
    }
    const float base = m == -INFINITY ? 0.f : m;
    float weight[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float e = fast_exp2(sc[i] - base);
      l += e;
      // A half that is not there has a scale that is not its own.
      weight[i] = e * (mask >> (i / 4) & 1 ? scales[2 + i / 4] : 0.f);
    }
    bf16x8_t pf[kWeights];
    split8<kWeights>(weight, pf);
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      const bf16x8_t vf = widen_operand<C>(vw[db].x, vw[db].y);
#pragma unroll
      for (int n = 0; n < kWeights; ++n)
        o[db] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(vf, pf[n], o[db], 0, 0, 0);
    }
  };

  // Wave w takes tiles w, w + NW, ...; up to NS of them in flight.
  if (wave < ntiles) {
    int mask_slot[NS] = {};
    mask_slot[0] = issue(0, wave);
    load_q();
    // The query and the first tile are waited for together, so that the
    // compiler has no load of its own left to wait for in the loop.
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    if (NS > 1 && wave + NW < ntiles) mask_slot[NS - 1] = issue(NS - 1, wave + NW);
    int k = wave, slot = 0;
    while (true) {
      if (NS > 1 && k + NW < ntiles)
        __builtin_amdgcn_s_waitcnt(vmcnt_only(kTileLoads));
      else
        __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      char* cur = my_ring + slot * kSlotBytes;
      const int mask = NS > 1 && slot ? mask_slot[NS - 1] : mask_slot[0];
      const int p0 = pos_begin + k * kTile;
      if (mask != 3 || p0 + kTile > pos_end) {
        // What lies behind the context or in another block may be NaN, and 0
        // times that is too: their V rows are zeroed (K's scores are replaced).
        // Two lanes a row.
        const int r = lane / 2, half = r / kHalf;
        if (!(mask >> half & 1) || p0 + r >= pos_end) {
          char* row = cur + 2 * kHalfBytes + r * D + lane % 2 * (D / 2);
#pragma unroll
          for (int i = 0; i < D / 2; i += 16)
            *reinterpret_cast<Word4*>(row + i) = Word4{};
        }
      }
      compute(k, cur, mask);
      if (k + NW >= ntiles) break;
      if (k + NS * NW < ntiles) {
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0): the slot has been read
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        const int next = issue(slot, k + NS * NW);
        if (NS > 1 && slot) mask_slot[NS - 1] = next; else mask_slot[0] = next;
      }
      k += NW;
      slot = slot + 1 == NS ? 0 : slot + 1;
    }
  }
  // No load may be in flight when the ring is used again.
  __builtin_amdgcn_s_waitcnt(0x0070);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);

  l += lane_xor16(l, lane);
  l += lane_xor32(l, lane);
  if (!(l == l)) m = 0.f;  // NaN counts, whatever the maximum

  // The wave's state into its own drained ring: acc[h][d].
  float* my_acc = reinterpret_cast<float*>(my_ring);
  if (col < G) {
#pragma unroll
    for (int db = 0; db < D / 16; ++db)
      *reinterpret_cast<f32x4_t*>(my_acc + col * D + db * 16 + 4 * quad) = o[db];
  }
  if (lane < kHeads) {
    s_m[wave][lane] = m;
    s_l[wave][lane] = l;
  }
  __syncthreads();

  const int elems = G * D;
  constexpr int kThreads = NW * kWave;
  constexpr int kPer = kHeads * D / kThreads;
  float acc_v[kPer], m_v[kPer], l_v[kPer];
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = tid + j * kThreads;
    acc_v[j] = 0.f;
    m_v[j] = -INFINITY;
    l_v[j] = 0.f;
    if (e < elems) {
      const int h = e / D, d = e % D;
      float mx = -INFINITY;
#pragma unroll
      for (int wv = 0; wv < NW; ++wv) mx = fmaxf(mx, s_m[wv][h]);
      float ls = 0.f, os = 0.f;
#pragma unroll
      for (int wv = 0; wv < NW; ++wv) {
        const float mw = s_m[wv][h];
        const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - mx);
        ls = fmaf(f, s_l[wv][h], ls);
        os = fmaf(f, reinterpret_cast<const float*>(s_ring + wv * NS * kSlotBytes)[h * D + d], os);
      }
      acc_v[j] = os;
      m_v[j] = mx;
      l_v[j] = ls;
    }
  }

  R* out = static_cast<R*>(a.out) + seq * a.o_ts + static_cast<int64_t>(head * G) * a.o_hs;
  if (nparts == 1) {
#pragma unroll
    for (int j = 0; j < kPer; ++j) {
      const int e = tid + j * kThreads;
      if (e < elems) {
        const float inv = l_v[j] != 0.f ? 1.f / l_v[j] : 0.f;
        out[(e / D) * a.o_hs + e % D] = E::store(acc_v[j] * inv);
      }
    }
    return;
  }

  int32_t* counter = a.counters + static_cast<int64_t>(seq) * c.heads + head;
  const int64_t base = (static_cast<int64_t>(it.first_item + it.part) * c.heads + head) * G;
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = tid + j * kThreads;
    if (e < elems) {
      const int h = e / D, d = e % D;
      store_coherent(a.ws_acc + (base + h) * D + d, acc_v[j]);
      if (d == 0) {
        store_coherent(a.ws_ml + (base + h) * 2, m_v[j]);
        store_coherent(a.ws_ml + (base + h) * 2 + 1, l_v[j]);
      }
    }
  }
  wait_stores();
  __syncthreads();  // every thread's partials are at the coherent level
  if (tid == 0)
    s_arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_arrived != nparts - 1) return;

  constexpr int kBatch = 8;  // partitions whose loads are in flight together
#pragma unroll
  for (int j = 0; j < kPer; ++j) {
    const int e = tid + j * kThreads;
    if (e >= elems) continue;
    const int h = e / D, d = e % D;
    float mx = -INFINITY, ls = 0.f, os = 0.f;
    for (int p0 = 0; p0 < nparts; p0 += kBatch) {
      float mb[kBatch], lbv[kBatch], ob[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int p = min(p0 + b, nparts - 1);
        const int64_t row = (static_cast<int64_t>(it.first_item + p) * c.heads + head) * G + h;
        mb[b] = load_coherent(a.ws_ml + row * 2);
        lbv[b] = load_coherent(a.ws_ml + row * 2 + 1);
        ob[b] = load_coherent(a.ws_acc + row * D + d);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b)
        if (p0 + b < nparts) merge_step(mx, ls, os, mb[b], lbv[b], ob[b]);
    }
    const float inv = ls != 0.f ? 1.f / ls : 0.f;
    out[h * a.o_hs + d] = E::store(os * inv);
  }
  if (tid == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

}  // namespace

bool quant_decode_mfma_takes(int32_t head_dim, int32_t group, int32_t block_size) {
  return (head_dim == 128 || head_dim == 64) && group <= kHeads && block_size >= kHalf;
}

bool quant_decode_mfma_supported(const QuantAttnArgs& a) {
  const QuantCache& c = a.c;
  const auto low = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | c.bs |
                   c.ts | c.hs;
  return quant_decode_mfma_takes(c.dim, a.group, c.block_size) && low % 16 == 0 &&
         c.ts < (int64_t(1) << 26);
}

int32_t launch_quant_decode_mfma(const QuantAttnArgs& a, int32_t dtype, int32_t code,
                                 hipStream_t stream) {
  const dim3 grid(static_cast<uint32_t>(a.max_items) * a.c.heads);
  const bool narrow = static_cast<int64_t>(a.num_seqs) * a.c.heads > device_cus();
  return with_types(dtype, code, [&](auto e, auto co) {
    using E = decltype(e);
    using C = decltype(co);
    auto go = [&](auto kernel) {
      kernel<<<grid, kWave * 8, 0, stream>>>(a);
      return check_launch("quantized decode");
    };
    if (a.c.dim == 128)
      return narrow ? go(quant_decode_kernel<E, C, 128, 8, 1>)
                    : go(quant_decode_kernel<E, C, 128, 8, 2>);
    return narrow ? go(quant_decode_kernel<E, C, 64, 8, 1>)
                  : go(quant_decode_kernel<E, C, 64, 8, 2>);
  });
}

}  // namespace mi
