// Attention of few query rows over an 8-bit K/V cache on MFMA: decode steps, and
// requests of a few tokens (drafts to verify, ends of prompts). head_dim 64, 128
// or 256, blocks of at least 16, queries of any type.
//
// out = softmax(scale * q . (k * ks)) (v * vs), with one ks and vs for each
// block and KV head. Bound by HBM for long contexts (two bytes a position and
// dim), by latency for few short ones.
//
//  * A sequence's rows at a KV head are its tokens times the group's query heads.
//    Workgroup = plan item (sequence, block range) x KV head x up to 16 NC of
//    them, so a cache row is read once for those. Its waves take tiles of 32
//    positions in turn: two halves of 16, each in one block.
//  * Tiles come into a ring of LDS slots of the wave's own by direct loads
//    (waited for by count, so a slot per wave stays in flight), the four scales
//    of a tile with them.
//  * Scores S^T[pos][row] = K . Q^T on v_mfma_f32_16x16x32_bf16, a half at a
//    time, or f16 for f16 queries; codes are widened to that on their way from LDS,
//    which loses nothing. f32 queries come in three bf16 parts, which hold all of
//    their bits. The K scale meets the score in float32.
//  * The lanes that hold a tile's scores hold the weights that
//    O^T[dim][row] += V^T . P^T wants from them, with V's bytes transposed on
//    their way out of LDS (ds_read_b64_tr_b8). A weight times the V scale goes
//    in as two bf16 parts (three for f32 queries), so that it loses less than
//    the output's rounding: in bf16, whose range is float32's, however far
//    apart the scales of the blocks are.
//  * Online softmax in the log2 domain; the reference moves only when a score
//    exceeds it by more than 15.
//  * Waves are joined through LDS, partitions by their last arrival, in order.
//
// Four layers with their plan, captured, 8 KV heads of 128, us (the 16-bit cache's
// kernel): 64 contexts of 128-2048 with 32 heads 129 (218; 480 MB, 3.7 TB/s), two of
// 62000 217 (363; 4.6 TB/s), 24 of 300-2500 in f16 82 (129), four of 150-500 36 (37),
// where launches and one chain of loads (item, table, tile, merge) are the time.
// Passes among others take 125 us of the first and 212 of the second: a replayed
// graph's start is 4 us. Targets of 256, 384 and 512 items where the plan has 192 took
// 131, 133 and 141 us there, 226, 255 and 246: their last round is partly empty.
#include <algorithm>
#include <climits>

#include "quant_mfma.h"

namespace mi {
namespace {

constexpr int kHalf = 16;   // positions of a half: one block's
constexpr int kTile = 32;   // positions of a tile
constexpr int kCols = 16;   // MFMA columns: query rows
constexpr float kRescaleSlack = 15.f;

// Maximum over aligned groups of 16 lanes.
__device__ __forceinline__ float max16(float v) {
  v = fmaxf(v, dpp_move<0xB1>(v));
  v = fmaxf(v, dpp_move<0x4E>(v));
  v = fmaxf(v, dpp_move<0x141>(v));
  return fmaxf(v, dpp_move<0x140>(v));
}

__device__ __forceinline__ f32x4_t mma(bf16x8_t a, bf16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x4_t mma(f16x8_t a, f16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

// LDS: a half's rows are D bytes, 16-byte chunk c of row r at cell
// r * (D / 16) + (c ^ swz(r)). LDS serves 16 cells of distinct place modulo 16
// at once: for K the 16 rows' chunk c, for V chunk c of rows r .. r + 7 of both
// halves.
template <int D>
__device__ __forceinline__ int swz_k(int r) {
  return D == 256 ? r & 15 : D == 128 ? (r >> 1) & 7 : (r >> 2) & 3;
}
template <int D>
__device__ __forceinline__ int swz_v(int r, int half) {
  return D == 256   ? (r & 7) ^ (8 * half)
         : D == 128 ? ((r >> 1) & 3) ^ (4 * half)
                    : ((r >> 2) & 1) ^ (2 * half);
}

// Waves a SIMD that the registers are kept for: of the workgroups that a CU's LDS
// has room for.
constexpr int waves_of(int D, int NS) { return D < 256 && NS == 1 ? 4 : 2; }

template <typename E, typename C, int D, int NC, int NW, int NS>
__global__ __launch_bounds__(kWave * NW, waves_of(D, NS)) void quant_decode_kernel(
    const QuantAttnArgs a) {
  using R = typename E::raw;
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  using Query = QueryOperand<E>;
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
  static_assert(NS >= 1 && NS <= 2 && NC * kCols * D * 4 <= NS * kSlotBytes, "ring");

  __shared__ __attribute__((aligned(16))) char s_ring[NW * NS * kSlotBytes];
  __shared__ __attribute__((aligned(16))) float s_m[NC * kCols][NW];
  __shared__ __attribute__((aligned(16))) float s_l[NC * kCols][NW];
  __shared__ float s_row[2][NC * kCols];
  __shared__ int s_arrived;

  const QuantCache& c = a.c;
  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int head = blockIdx.x % c.heads;
  const int group = blockIdx.x / c.heads % a.row_groups;
  const int w = blockIdx.x / c.heads / a.row_groups;
  const int G = a.group;
  const int col = lane % 16;
  const int quad = lane / 16;

  // The item, checked so that a stale or foreign plan gives wrong attention
  // but no access out of bounds.
  typedef int32_t int8v __attribute__((ext_vector_type(8)));
  using ConstItem = __attribute__((address_space(4))) const int8v;
  const PlanItem it = __builtin_bit_cast(PlanItem, ((ConstItem*)(a.plan))[w]);
  if (!item_fits(it, a)) return;  // unused slot (uniform across the workgroup)
  const int seq = it.seq;
  const int lb = c.log2_block;
  const int ctx = min(max(it.ctx, 0), a.t_width << lb);
  const int blk_begin = min(max(it.blk_begin, 0), a.t_width);
  const int blk_end = min(max(it.blk_end, 0), a.t_width);
  const int nparts = it.nparts;
  // The rows: of a decode step, or of a request's tokens, which see less of its
  // end the earlier they are.
  int q_begin = seq, q_len = 1, seen = INT_MAX;  // by the first token
  if (a.cu_q != nullptr) {
    const ConstI32* cu_q = (const ConstI32*)(a.cu_q);
    const ConstI32* cu_k = (const ConstI32*)(a.cu_k);
    q_begin = max(cu_q[seq], 0);
    q_len = cu_q[seq + 1] - q_begin;
    seen = cu_k[seq + 1] - cu_k[seq] - q_len + 1;
    q_len = min(q_len, a.num_rows - q_begin);
  }
  const int row0 = group * NC * kCols;
  const int rows =
      min(static_cast<int>(min(int64_t(q_len) * G, int64_t(a.head_rows))) - row0, NC * kCols);
  if (rows <= 0) return;  // in every part
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

  // Row r's token: r and G are small enough for this to be r / G.
  auto token_of = [&](int r) { return static_cast<int>(uint32_t(r) * a.group_inverse >> 24); };
  // Query operand of MFMA step 2 j + h: dims 16 (quad + 4 j) + 8 h .. + 7 of
  // row `col`, the order in which a lane reads K.
  Query qf[NC][kParts][kSteps];
  int limit[NC];  // the row sees positions below
  auto load_q = [&]() {
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      const bool there = n * kCols + col < rows;
      const int r = row0 + (there ? n * kCols + col : 0);
      const int token = token_of(r), g = r - token * G;
      limit[n] = there ? min(static_cast<int>(min(static_cast<int64_t>(seen) + token,
                                                  int64_t(INT_MAX))), pos_end) : 0;
      const R* row = static_cast<const R*>(a.q) + static_cast<int64_t>(q_begin + token) * a.q_ts +
                     static_cast<int64_t>(head * G + g) * a.q_hs;
      float x[kSteps][8];  // loads that wait for no branch
#pragma unroll
      for (int s = 0; s < kSteps; ++s)
        load8<E>(row + 16 * (quad + 4 * (s / 2)) + 8 * (s % 2), x[s]);
#pragma unroll
      for (int s = 0; s < kSteps; ++s) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[s][i] = there ? x[s][i] : 0.f;
        Query part[kParts];
        split8<kParts>(x[s], part);
#pragma unroll
        for (int p = 0; p < kParts; ++p) qf[n][p][s] = part[p];
      }
    }
  };

  f32x4_t o[NC][D / 16];
  float m[NC], l[NC];
#pragma unroll
  for (int n = 0; n < NC; ++n) {
    m[n] = -INFINITY;
    l[n] = 0.f;
#pragma unroll
    for (int db = 0; db < D / 16; ++db) o[n][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }

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
    float sc[NC][8];
#pragma unroll
    for (int j = 0; j < 2; ++j) {
      f32x4_t s[NC];
#pragma unroll
      for (int n = 0; n < NC; ++n) s[n] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kSteps; ++i) {
        const Query kf =
            widen<Query, C>(kw[j][i / 2].w[2 * (i % 2)], kw[j][i / 2].w[2 * (i % 2) + 1]);
#pragma unroll
        for (int n = 0; n < NC; ++n)
#pragma unroll
          for (int q = 0; q < kParts; ++q)
            s[n] = mma(kf, qf[n][q][i], s[n]);
      }
      const float factor = scales[j] * a.scale_log2;
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          sc[n][4 * j + i] =
              (mask >> j & 1) && p + kHalf * j + i < limit[n] ? s[n][i] * factor : -INFINITY;
    }
    bf16x8_t pf[NC][kWeights];
#pragma unroll
    for (int n = 0; n < NC; ++n) {
      float tmax = sc[n][0];
#pragma unroll
      for (int i = 1; i < 8; ++i) tmax = fmaxf(tmax, sc[n][i]);
      tmax = fmaxf(tmax, lane_xor16(tmax, lane));
      tmax = fmaxf(tmax, lane_xor32(tmax, lane));
      if (__ballot(tmax > m[n] + kRescaleSlack) != 0) {
        const float mnew = fmaxf(m[n], tmax);
        const float alpha = mnew == -INFINITY ? 1.f : fast_exp2(m[n] - mnew);
        l[n] *= alpha;
#pragma unroll
        for (int db = 0; db < D / 16; ++db) o[n][db] *= alpha;
        m[n] = mnew;
      }
      const float base = m[n] == -INFINITY ? 0.f : m[n];
      float weight[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = fast_exp2(sc[n][i] - base);
        l[n] += e;
        // A half that is not there has a scale that is not its own.
        weight[i] = e * (mask >> (i / 4) & 1 ? scales[2 + i / 4] : 0.f);
      }
      split8<kWeights>(weight, pf[n]);
    }
#pragma unroll
    for (int db = 0; db < D / 16; ++db) {
      const bf16x8_t vf = widen_operand<C>(vw[db].x, vw[db].y);
#pragma unroll
      for (int n = 0; n < NC; ++n)
#pragma unroll
        for (int q = 0; q < kWeights; ++q)
          o[n][db] = mma(vf, pf[n][q], o[n][db]);
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

#pragma unroll
  for (int n = 0; n < NC; ++n) {
    l[n] += lane_xor16(l[n], lane);
    l[n] += lane_xor32(l[n], lane);
    if (!(l[n] == l[n])) m[n] = 0.f;  // NaN counts, whatever the maximum
    if (lane < kCols) {
      s_m[n * kCols + lane][wave] = m[n];
      s_l[n * kCols + lane][wave] = l[n];
    }
  }
  // The waves' sums into their own drained rings, acc[row][d] with four dims at
  // cell (d / 4) ^ (row % 16) of the row, joined by all threads: a thread's pair
  // of dims `dim`, of rows row_of(0), row_of(1), ...
  constexpr int kThreads = NW * kWave;
  constexpr int kStep = 2 * kThreads / D;  // rows that the threads cover at once
  constexpr int kPairs = NC * kCols / kStep;
  const int dim = 2 * (tid % (D / 2));
  auto row_of = [&](int j) { return j * kStep + tid / (D / 2); };
  {
    float* acc = reinterpret_cast<float*>(my_ring);
#pragma unroll
    for (int n = 0; n < NC; ++n)
#pragma unroll
      for (int db = 0; db < D / 16; ++db)
        if (n * kCols + col < rows)
          *reinterpret_cast<f32x4_t*>(acc + (n * kCols + col) * D +
                                      4 * ((db * 4 + quad) ^ col)) = o[n][db];
  }
  __syncthreads();
  Float2 sum[kPairs];
  float top[kPairs], total[kPairs];  // a row's maximum and sum
#pragma unroll
  for (int j = 0; j < kPairs; ++j) {
    const float* ms = s_m[row_of(j)];
    const float* lw = s_l[row_of(j)];
    top[j] = -INFINITY;
    total[j] = 0.f;
    sum[j] = Float2{0.f, 0.f};
    if (row_of(j) >= rows) continue;
    const int at = row_of(j) * D + 4 * ((dim / 4) ^ (row_of(j) % 16)) + dim % 4;
#pragma unroll
    for (int wv = 0; wv < NW; ++wv) top[j] = fmaxf(top[j], ms[wv]);
#pragma unroll
    for (int wv = 0; wv < NW; ++wv) {
      const Float2 y =
          *reinterpret_cast<const Float2*>(s_ring + wv * NS * kSlotBytes + at * 4);
      const float f = ms[wv] == -INFINITY ? 0.f : fast_exp2(ms[wv] - top[j]);
      total[j] = fmaf(f, lw[wv], total[j]);
      sum[j].x = fmaf(f, y.x, sum[j].x);
      sum[j].y = fmaf(f, y.y, sum[j].y);
    }
  }
  auto put = [&](int r, Float2 x, float ls) {
    const int token = token_of(row0 + r);
    const float inv = ls != 0.f ? 1.f / ls : 0.f;
    struct alignas(2 * sizeof(R)) Pair {
      R x, y;
    };
    *reinterpret_cast<Pair*>(static_cast<R*>(a.out) +
                             static_cast<int64_t>(q_begin + token) * a.o_ts +
                             static_cast<int64_t>(head * G + row0 + r - token * G) * a.o_hs +
                             dim) =
        Pair{E::store(x.x * inv), E::store(x.y * inv)};
  };
  if (nparts == 1) {
#pragma unroll
    for (int j = 0; j < kPairs; ++j)
      if (row_of(j) < rows) put(row_of(j), sum[j], total[j]);
    return;
  }

  int32_t* counter =
      a.counters + (static_cast<int64_t>(seq) * a.row_groups + group) * c.heads + head;
  // Row r of partition p.
  auto slot_of = [&](int p, int r) {
    return (static_cast<int64_t>(it.first_item + p) * c.heads + head) * a.head_rows + row0 + r;
  };
#pragma unroll
  for (int j = 0; j < kPairs; ++j)
    if (row_of(j) < rows) {
      store_coherent2(a.ws_acc + slot_of(it.part, row_of(j)) * D + dim, sum[j].x, sum[j].y);
      if (dim == 0) store_coherent2(a.ws_ml + slot_of(it.part, row_of(j)) * 2, top[j], total[j]);
    }
  wait_stores();
  __syncthreads();  // every thread's partials are at the coherent level
  if (tid == 0)
    s_arrived = __hip_atomic_fetch_add(counter, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s_arrived != nparts - 1) return;

  // What a merge takes is its loads' latency: 16 of a thread are in flight at once
  // (32 rows of 24 partitions, four layers, 8 / 16 / 24 / 32 / 64 loads: 120 / 117 /
  // 120 / 123 / 166 us; two levels of groups 124).
  if (rows <= kStep) {  // a row a thread
    const int r = row_of(0);
    constexpr int kBatch = 8;
    float mx = -INFINITY, ls = 0.f;
    Float2 x{0.f, 0.f};
    for (int p0 = 0; p0 < nparts && r < rows; p0 += kBatch) {
      Float2 ml[kBatch], y[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int64_t at = slot_of(min(p0 + b, nparts - 1), r);
        ml[b] = load_coherent2(a.ws_ml + at * 2);
        y[b] = load_coherent2(a.ws_acc + at * D + dim);
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (p0 + b >= nparts || ml[b].x == -INFINITY) continue;  // nothing was seen
        const float now = fmaxf(mx, ml[b].x);
        const float back = mx == -INFINITY ? 0.f : fast_exp2(mx - now);
        const float f = fast_exp2(ml[b].x - now);
        ls = fmaf(ls, back, f * ml[b].y);
        x.x = fmaf(x.x, back, f * y[b].x);
        x.y = fmaf(x.y, back, f * y[b].y);
        mx = now;
      }
    }
    if (r < rows) put(r, x, ls);
  } else if constexpr (kPairs > 1) {
    // Several rows a thread: the factors go through LDS, found by 16 lanes a row.
    constexpr int kChunk = 32;  // partitions at once there
    constexpr int kBatch = 16 / kPairs;
    static_assert(kThreads / 16 >= NC * kCols, "16 lanes for a row's factors");
    const int frow = tid / 16, sub = tid % 16;
    float(*s_f)[NC * kCols] = reinterpret_cast<float(*)[NC * kCols]>(s_ring);
    float mx = -INFINITY, ls = 0.f;
    Float2 x[kPairs] = {};
    for (int p0 = 0; p0 < nparts; p0 += kChunk) {
      const int n = min(kChunk, nparts - p0);
      Float2 y[kBatch][kPairs];
      auto load = [&](int q) __attribute__((always_inline)) {
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
#pragma unroll
          for (int j = 0; j < kPairs; ++j)
            y[b][j] = load_coherent2(
                a.ws_acc + slot_of(p0 + min(q + b, n - 1), min(row_of(j), rows - 1)) * D + dim);
      };
      Float2 ml[kChunk / 16];
#pragma unroll
      for (int i = 0; i < kChunk / 16; ++i)
        ml[i] = load_coherent2(
            a.ws_ml + slot_of(p0 + min(sub + 16 * i, n - 1), min(frow, rows - 1)) * 2);
      load(0);
      if (p0 > 0) __syncthreads();  // the last factors are read
      if (frow < NC * kCols) {
        float now = mx;
#pragma unroll
        for (int i = 0; i < kChunk / 16; ++i) now = fmaxf(now, max16(ml[i].x));
        float lsum = 0.f;
#pragma unroll
        for (int i = 0; i < kChunk / 16; ++i) {
          // Below zero: nothing was seen.
          const float f = ml[i].x == -INFINITY ? -1.f : fast_exp2(ml[i].x - now);
          lsum += f < 0.f || sub + 16 * i >= n ? 0.f : f * ml[i].y;
          s_f[sub + 16 * i][frow] = f;
        }
        const float back = mx == -INFINITY ? 0.f : fast_exp2(mx - now);
        ls = fmaf(ls, back, group_sum<16>(lsum));
        mx = now;
        if (sub == 0) {
          s_row[0][frow] = back;
          s_row[1][frow] = ls;
        }
      }
      __syncthreads();
#pragma unroll
      for (int j = 0; j < kPairs; ++j) {
        const float back = s_row[0][row_of(j)];
        x[j].x *= back;
        x[j].y *= back;
      }
      for (int q = 0; q < n; q += kBatch) {
        if (q > 0) load(q);
#pragma unroll
        for (int b = 0; b < kBatch; ++b)
#pragma unroll
          for (int j = 0; j < kPairs; ++j) {
            const float f = s_f[min(q + b, kChunk - 1)][row_of(j)];
            const bool weighs = q + b < n && f >= 0.f;
            x[j].x = weighs ? fmaf(f, y[b][j].x, x[j].x) : x[j].x;
            x[j].y = weighs ? fmaf(f, y[b][j].y, x[j].y) : x[j].y;
          }
      }
    }
#pragma unroll
    for (int j = 0; j < kPairs; ++j)
      if (row_of(j) < rows) put(row_of(j), x[j], s_row[1][row_of(j)]);
  }
  if (tid == 0) __hip_atomic_store(counter, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The lengths of requests as decode sequences (0: no rows), and the counters of
// their rows cleared.
__global__ __launch_bounds__(256) void few_rows_kernel(const int32_t* __restrict__ cu_q,
                                                       const int32_t* __restrict__ cu_k,
                                                       int num_seqs, int32_t* __restrict__ lens,
                                                       int32_t* __restrict__ counters,
                                                       int num_counters) {
  const int i = blockIdx.x * 256 + threadIdx.x;
  if (i < num_seqs) lens[i] = cu_q[i + 1] > cu_q[i] ? max(cu_k[i + 1] - cu_k[i], 0) : 0;
  if (i < num_counters) counters[i] = 0;
}

}  // namespace

bool quant_decode_mfma_takes(int32_t head_dim, int32_t block_size) {
  return (head_dim == 256 || head_dim == 128 || head_dim == 64) && block_size >= kHalf;
}

bool quant_mfma_aligned(const QuantCache& c) {
  const auto low = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | c.bs |
                   c.ts | c.hs;
  return low % 16 == 0 && c.ts < (int64_t(1) << 26);
}

int32_t quant_decode_row_groups(int32_t rows, int32_t head_dim) {
  if (head_dim == 256) return (rows - 1) / kCols + 1;
  return rows <= kCols ? 1 : (rows - 1) / (2 * kCols) + 1;
}

int32_t launch_quant_decode_mfma(QuantAttnArgs a, int32_t rows, int32_t dtype, int32_t code,
                                 hipStream_t stream) {
  a.head_rows = rows;
  a.row_groups = quant_decode_row_groups(rows, a.c.dim);
  // r * inverse >> 24 is r / group for r * group < 2^24, with no overflow for
  // r < 2^8.
  if (rows > 256) return fail(MI_ERR_UNSUPPORTED, "quantized decode: too many rows");
  a.group_inverse = ((1u << 24) + a.group - 1) / a.group;
  const int64_t grid = static_cast<int64_t>(a.max_items) * a.c.heads * a.row_groups;
  if (grid > INT_MAX)
    return fail(MI_ERR_UNSUPPORTED, "quantized attention: too many rows for one launch");
  // Many workgroups: two a CU with a slot a wave, where they fit the registers
  // that leaves them (four layers of 128 sequences of 500 tokens 144 us, 173 with
  // one of two slots; 64 of 1000 with heads of 64 77 / 80, float32 80 / 84. In
  // float32 heads of 128 spill: 64 of 1000 376 / 141).
  // Four of four waves where there are so many: their starts and ends overlap (128
  // sequences of 200 tokens 92 / 80 us, of 500 144 / 135, of 2000 403 / 412; at
  // three a CU, 96 of 200-400 87 / 77, but of 100-2500 238 / 248).
  const int64_t groups = static_cast<int64_t>(a.num_seqs) * a.c.heads * a.row_groups;
  const bool narrow = groups > device_cus(), small = groups >= 4 * device_cus();
  return with_types(dtype, code, [&](auto e, auto co) {
    using E = decltype(e);
    using C = decltype(co);
    auto go = [&](auto kernel, int waves = 8) {
      kernel<<<static_cast<uint32_t>(grid), kWave * waves, 0, stream>>>(a);
      return check_launch("quantized decode");
    };
    if (a.c.dim == 256) return go(quant_decode_kernel<E, C, 256, 1, 8, 1>);
    const bool wide = a.c.dim == 128;
    if (rows > kCols)
      return wide ? go(quant_decode_kernel<E, C, 128, 2, 8, 2>)
                  : go(quant_decode_kernel<E, C, 64, 2, 8, 2>);
    if (narrow && !wide)
      return small ? go(quant_decode_kernel<E, C, 64, 1, 4, 1>, 4)
                   : go(quant_decode_kernel<E, C, 64, 1, 8, 1>);
    if constexpr (!std::is_same<E, F32>::value)
      if (narrow)
        return small ? go(quant_decode_kernel<E, C, 128, 1, 4, 1>, 4)
                     : go(quant_decode_kernel<E, C, 128, 1, 8, 1>);
    return wide ? go(quant_decode_kernel<E, C, 128, 1, 8, 2>)
                : go(quant_decode_kernel<E, C, 64, 1, 8, 2>);
  });
}

int32_t launch_few_rows(const int32_t* cu_q, const int32_t* cu_k, int32_t num_seqs, int32_t* lens,
                        int32_t* counters, int32_t num_counters, hipStream_t stream) {
  const int n = std::max(num_seqs, num_counters);
  few_rows_kernel<<<(n - 1) / 256 + 1, 256, 0, stream>>>(cu_q, cu_k, num_seqs, lens, counters,
                                                         num_counters);
  return check_launch("quantized attention plan");
}

}  // namespace mi
