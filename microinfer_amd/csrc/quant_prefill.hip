// Varlen (chunked prefill, mixed) attention over an 8-bit K/V cache on MFMA:
// head_dim 64 or 128, any group of up to 128 query heads per KV head, blocks of
// at least 16, queries of any type.
//
// out = softmax(scale * q . (k * ks) + causal mask) (v * vs), with one ks and vs
// for each block and KV head. Bound by the matrix and vector units together.
//
//  * Workgroup = plan item (request, block of query rows, range of key tiles) x
//    KV head. The block's tokens times the group's heads are its rows, up to 128:
//    four waves of 32, so a key tile serves all heads of the group.
//  * A tile of 32 keys is widened to 16-bit floats (exactly) once for the four
//    waves: a thread loads 16 codes of K and of V and writes them, a tile later,
//    to the one of two LDS buffers that is not read. Rows of V that nothing may
//    see are written as zeros. K runs a tile ahead: the scores of a tile are
//    computed while the softmax of the one before is.
//  * S^T = K . Q^T on 32x32x16 MFMA: bf16 queries with codes as bf16, f16 with
//    codes as f16, f32 ones in three bf16 parts, which hold all of their bits.
//    The K scale meets the scores in float32. A lane owns 16 keys of one row, so
//    the softmax needs its neighbour only where a reference moves and for the
//    sum at the end.
//  * O^T += V^T . P^T on the same instruction, V^T by transposing LDS reads. A
//    weight e = 2^(score - m) meets V as e * vs * 2^(m - mo) in f16, of which mo
//    keeps the largest of the row between 2^10 and 2^15: rounding takes 2^-11 of a
//    weight (an eighth of what bf16 would, a quarter or less of the bf16 output's
//    own), and what f16 cannot hold is 2^-35 of the largest. f16 queries, whose
//    output is as fine, have two such parts; f32 ones three in bf16.
//  * Row blocks whose keys are split publish theirs; the last arrival merges
//    them in order.
#include <climits>

#include "quant_mfma.h"

namespace mi {
namespace {

constexpr int kKeys = 32;
constexpr int kRows = 32;  // of a wave
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kBlockRows = kRows * kWaves;
constexpr float kRescaleSlack = 15.f;
// A row's largest weight lies between 2^kTopWeight and 2^kMostWeight.
constexpr float kTopWeight = 10.f, kMostWeight = 15.f;

typedef short short4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ short4_t read_tr16(const uint16_t* lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16(
      (__attribute__((address_space(3))) short4_t*)(lds));
}

struct QuantPrefillArgs : QuantAttnArgs {
  const PrefillItem* items;
  const int32_t* count;
};

// LDS tiles are rows of D bf16, the 16-byte chunk c of key k at c ^ swz(k): K
// fragments (16 keys, one chunk) and V ones (4 keys, 4 chunks) are read without
// bank conflicts.
template <int D>
__device__ __forceinline__ int swz_k(int key) {
  return D == 128 ? key & 15 : (key >> 1) & 7;
}
template <int D>
__device__ __forceinline__ int swz_v(int key) {
  return D == 128 ? 4 * (key & 3) : 4 * ((key >> 1) & 1);
}

#ifndef VAR
#define VAR 0
#endif
// Workgroups of a CU, by the registers of the query's parts.
template <typename E>
constexpr int kResident = VAR == 1 && std::is_same<E, BF16>::value ? 3 : 2;
template <typename E>
constexpr bool kOverlap = !std::is_same<E, F32>::value && VAR != 1 && VAR != 2;

// How an element type's queries meet K (parts of the query), and its weights V.
template <typename E>
struct Meets {
  using Query = bf16x8_t;
  using Weight = f16x8_t;
  static constexpr int kQueries = 1, kWeights = 1;
};
template <>
struct Meets<F16> {
  using Query = f16x8_t;
  using Weight = f16x8_t;
  static constexpr int kQueries = 1, kWeights = 2;
};
template <>
struct Meets<F32> {
  using Query = bf16x8_t;
  using Weight = bf16x8_t;
  static constexpr int kQueries = 3, kWeights = 3;
};

__device__ __forceinline__ f32x16_t mma(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mma(f16x8_t a, f16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

template <typename V, typename C>
__device__ __forceinline__ V widen(uint32_t lo, uint32_t hi) {
  if constexpr (std::is_same<V, bf16x8_t>::value)
    return widen_operand<C>(lo, hi);
  else
    return widen_operand_f16<C>(lo, hi);
}

template <typename E, typename C, int D>
__global__ __launch_bounds__(kThreads, kResident<E>) void quant_prefill_kernel(
    const QuantPrefillArgs a) {
  using R = typename E::raw;
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  using ConstF32 = __attribute__((address_space(4))) const float;
  using Query = typename Meets<E>::Query;
  using Weight = typename Meets<E>::Weight;
  constexpr int kQueries = Meets<E>::kQueries, kWeights = Meets<E>::kWeights;
  constexpr int kTileElems = kKeys * D;
  constexpr int kAccFloats = D / 32 * 16;  // of a lane
  // A thread's 16 codes: with D = 128 of K and of V, with D = 64 of one of them.
  constexpr bool kBoth = D == 128;
  __shared__ __attribute__((aligned(16))) uint16_t s_k[2][kTileElems];
  __shared__ __attribute__((aligned(16))) uint16_t s_v[2][kTileElems];
  __shared__ int s_arrived;

  const QuantCache& c = a.c;
  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int half = lane / 32;
  const int col = lane % 32;
  const int head = blockIdx.x % c.heads;
  const int item = blockIdx.x / c.heads;
  if (item >= *(const ConstI32*)(a.count)) return;  // surplus (uniform)
  const ConstI32* it = (const ConstI32*)(a.items + item);
  const int req = it[0], rblock = it[1], part = it[4], nparts = it[5], slot = it[6];
  int t_begin = it[2];
  const int t_limit = it[3], counter = it[7];
  const ConstI32* cu_q = (const ConstI32*)(a.cu_q);
  const ConstI32* cu_k = (const ConstI32*)(a.cu_k);
  const int G = a.group;
  const int tokens = kBlockRows / G;  // of a row block
  const int q_begin = cu_q[req];
  const int q_len = cu_q[req + 1] - q_begin;
  const int ctx = cu_k[req + 1] - cu_k[req];
  const int tok0 = rblock * tokens;
  const int tok_last = min(q_len, tok0 + tokens) - 1;
  // Keys of the block: up to the causal limit of its last token.
  const int kv_end = max(0, min(ctx - q_len + tok_last + 1, a.t_width << c.log2_block));
  const int ntiles = min((kv_end + kKeys - 1) / kKeys, t_limit);
  t_begin = min(t_begin, ntiles);

  const int r = wave * kRows + col;
  const int token = tok0 + r / G, g = r % G;
  const bool row_ok = r < tokens * G && token < q_len;
  const int qpos = ctx - q_len + token;  // the row sees keys 0 .. qpos
  // Of the wave's rows: tiles below nint need no mask, from nend on they see
  // nothing.
  const int wave_tok0 = tok0 + wave * kRows / G;
  const int wave_tok1 = min(tok_last, tok0 + (wave * kRows + kRows - 1) / G);
  const bool wave_ok = wave * kRows < tokens * G && wave_tok0 < q_len;
  const int nint = min(kv_end / kKeys, max(ctx - q_len + wave_tok0 + 1, 0) / kKeys);
  const int nend =
      wave_ok ? min((max(ctx - q_len + wave_tok1 + 1, 0) + kKeys - 1) / kKeys, ntiles) : 0;

  // Staging: this thread's key of a tile, its 16 codes, and where they go.
  const bool is_v = !kBoth && wave >= 2;
  const int key = kBoth ? tid / 8 : tid % 128 / 4;
  const int chunk = 2 * (kBoth ? tid % 8 : tid % 4);  // of 8 codes
  const int wave_half = kBoth ? wave / 2 : wave % 2;  // of the tile, the wave's
  const int64_t lane_off = head * c.hs + key % 16 * c.ts + chunk * 8;
  const uint8_t* kc = c.k + lane_off;
  const uint8_t* vc = c.v + lane_off;
  const float* ks_head = c.ks + head * c.s_hs;
  const float* vs_head = c.vs + head * c.s_hs;
  const ConstI32* table = (const ConstI32*)(a.tables + req * a.t_stride);

  // What is known of a tile, from its ids (read a step before they are used)
  // to its scales.
  struct Ids {
    int id[2];
  };
  struct Page {
    int64_t at;  // byte offset of this wave's half
    int mask;    // bit h: half h is in a block of the pool
    float ks[2], vs[2];
  };
  auto load_ids = [&](int tile) __attribute__((always_inline)) {
    const int t0 = min(tile, ntiles - 1) * kKeys;
    const int e0 = t0 >> c.log2_block;
    // The second half's entry; past the keys, the first's again.
    const int e1 = t0 + 16 < kv_end ? (t0 + 16) >> c.log2_block : e0;
    return Ids{table[e0], table[e1]};
  };
  auto load_page = [&](int tile, const Ids& ids) __attribute__((always_inline)) {
    const bool ok0 = static_cast<uint32_t>(ids.id[0]) < static_cast<uint32_t>(c.num_blocks);
    const bool ok1 = static_cast<uint32_t>(ids.id[1]) < static_cast<uint32_t>(c.num_blocks);
    const uint32_t p0 = ok0 ? ids.id[0] : 0, p1 = ok1 ? ids.id[1] : 0;
    const int t0 = min(tile, ntiles - 1) * kKeys;
    Page p;
    p.mask = (ok0 ? 1 : 0) | (ok1 ? 2 : 0);
    p.at = (wave_half ? p1 : p0) * static_cast<uint64_t>(c.bs) +
           static_cast<uint32_t>((t0 + 16 * wave_half) & (c.block_size - 1)) *
               static_cast<uint64_t>(c.ts);
    p.ks[0] = ((const ConstF32*)ks_head)[p0 * c.s_bs];
    p.ks[1] = ((const ConstF32*)ks_head)[p1 * c.s_bs];
    p.vs[0] = ((const ConstF32*)vs_head)[p0 * c.s_bs];
    p.vs[1] = ((const ConstF32*)vs_head)[p1 * c.s_bs];
    return p;
  };
  auto load16 = [&](const uint8_t* base, const Page& p) __attribute__((always_inline)) {
    return *reinterpret_cast<const Word4*>(base + p.at);
  };
  // `first`: which of the two chunks goes first, for the banks.
  auto put = [&](auto lo, auto hi, uint16_t* row, int swz, int first)
      __attribute__((always_inline)) {
    using V = decltype(lo);
    *reinterpret_cast<V*>(row + ((chunk + first) ^ swz) * 8) = first ? hi : lo;
    *reinterpret_cast<V*>(row + ((chunk + 1 - first) ^ swz) * 8) = first ? lo : hi;
  };
  auto land_k = [&](const Word4& w, int buf) __attribute__((always_inline)) {
    put(widen<Query, C>(w.w[0], w.w[1]), widen<Query, C>(w.w[2], w.w[3]), s_k[buf] + key * D,
        swz_k<D>(key), 0);
  };
  // Keys that nothing may see may be NaN, which 0 times does not make 0.
  auto land_v = [&](Word4 w, int tile, const Page& p, int buf) __attribute__((always_inline)) {
    const bool there = tile * kKeys + key < kv_end && (p.mask >> wave_half & 1);
#pragma unroll
    for (int i = 0; i < 4; ++i) w.w[i] = there ? w.w[i] : 0;
    put(widen<Weight, C>(w.w[0], w.w[1]), widen<Weight, C>(w.w[2], w.w[3]), s_v[buf] + key * D,
        swz_v<D>(key), kBoth ? key & 1 : 0);
  };

  // Query operand: step s holds dims 16 s + 8 half .. + 7 of the lane's row. A
  // negative softmax scale goes into the query, so that the factors of the
  // scores are positive.
  Query qf[kQueries][D / 16];
  const float scale_log2 = fabsf(a.scale_log2);
  {
    const R* row = static_cast<const R*>(a.q) + static_cast<int64_t>(q_begin + token) * a.q_ts +
                   static_cast<int64_t>(head * G + g) * a.q_hs;
    const float sign = a.scale_log2 < 0.f ? -1.f : 1.f;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      float x[8] = {};
      if (row_ok) load8<E>(row + s * 16 + half * 8, x);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] *= sign;
      Query p[kQueries];
      split8<kQueries>(x, p);
#pragma unroll
      for (int n = 0; n < kQueries; ++n) qf[n][s] = p[n];
    }
  }

  // Fragment reads: K key `col`, chunk 2 s + half; V^T as four-by-four
  // transposes: lane (gq = lane / 16, sl = lane % 16) supplies the 8-byte row of
  // key 16 h + 8 j + (gq / 2) * 4 + sl / 4 at dims 32 db + (gq % 2) * 16 + 4 (sl % 4)
  // and receives keys 16 h + 8 j + 4 half .. + 3 of dim 32 db + col.
  int v_rd[D / 32];
  {
    const int gq = lane / 16, sl = lane % 16;
    const int vkey = gq / 2 * 4 + sl / 4;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
      v_rd[db] = vkey * D + ((4 * db + 2 * (gq % 2) + sl % 4 / 2) ^ swz_v<D>(vkey)) * 8 +
                 4 * (sl % 2);
  }

  f32x16_t o[D / 32];
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
  // Of the row, in the log2 domain: the references of l and of o, and the
  // sum of this lane's half of the keys.
  float m = -INFINITY, mo = -INFINITY, l = 0.f;

  // s[i]: key i / 4 * 8 + half * 4 + i % 4 of the row, in half i / 8 of the tile.
  auto scores = [&](int buf) __attribute__((always_inline)) {
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
      const Query kf = *reinterpret_cast<const Query*>(
          s_k[buf] + col * D + ((2 * x + half) ^ swz_k<D>(col)) * 8);
#pragma unroll
      for (int n = 0; n < kQueries; ++n) s = mma(kf, qf[n][x], s);
    }
    return s;
  };
  auto mask_scores = [&](int tile, const Page& p, f32x16_t& s) __attribute__((always_inline)) {
    const int last = min(qpos, kv_end - 1) - tile * kKeys - half * 4;
#pragma unroll
    for (int i = 0; i < 16; ++i)
      s[i] = i / 4 * 8 + i % 4 <= last && (p.mask >> (i / 8) & 1) ? s[i] : -INFINITY;
  };
  // Masked scores are -inf, which 0 would make NaN.
  auto factor_of = [&](float ks) __attribute__((always_inline)) {
    const float f = ks * scale_log2;
    return f == 0.f ? 0x1p-126f : f;
  };
  // Moves the references where the tile's scores lie too far above them.
  auto look = [&](const Page& p, const f32x16_t& s) __attribute__((always_inline)) {
    float high[2], weigh[2];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float x = s[8 * h];
#pragma unroll
      for (int i = 1; i < 8; ++i) x = fmaxf(x, s[8 * h + i]);
      high[h] = x * factor_of(p.ks[h]);
      weigh[h] = high[h] + __builtin_amdgcn_logf(p.vs[h]);
    }
    const float smax = fmaxf(high[0], high[1]), wmax = fmaxf(weigh[0], weigh[1]);
    if (__ballot(smax > m + kRescaleSlack || wmax > mo + kMostWeight) != 0) {
      const float mnew = fmaxf(m, fmaxf(smax, lane_xor32(smax, lane)));
      l *= mnew == -INFINITY ? 1.f : fast_exp2(m - mnew);
      m = mnew;
      const float monew = fmaxf(mo, fmaxf(wmax, lane_xor32(wmax, lane)) - kTopWeight);
      const float alpha = monew == -INFINITY ? 1.f : fast_exp2(mo - monew);
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
      mo = monew;
    }
  };
  auto weigh = [&](const Page& p, const f32x16_t& s, Weight (&pf)[2][kWeights])
      __attribute__((always_inline)) {
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const float factor = factor_of(p.ks[h]);
      // A half that is not there has a scale that is not its own.
      // Without a reference all scales were 0 or NaN so far, and so it stays.
      const float power = __builtin_amdgcn_logf(p.vs[h]) + (base - mo);
      float up = fast_exp2(power);
      up = mo > -INFINITY ? up : p.vs[h];
      up = p.mask >> h & 1 ? up : 0.f;
      float weight[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = fast_exp2(fmaf(s[8 * h + i], factor, -base));
        l += e;
        weight[i] = e * up;
      }
      split8<kWeights>(weight, pf[h]);
    }
  };
  // Slots 0 - 3 of a half's 8 are keys 16 h + 4 half .. + 3, the others eight
  // keys on.
  auto gather = [&](const Weight (&pf)[2][kWeights], int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint16_t* at = s_v[buf] + v_rd[db] + 16 * h * D;
        const short4_t both[2] = {read_tr16(at), read_tr16(at + 8 * D)};
        const Weight vf = __builtin_bit_cast(Weight, both);
#pragma unroll
        for (int n = 0; n < kWeights; ++n) o[db] = mma(vf, pf[h][n], o[db]);
      }
    }
  };

  // A bare barrier: this wave's LDS writes are done, its loads stay in flight.
  auto sync_lds = [&]() __attribute__((always_inline)) {
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
    __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
    __builtin_amdgcn_s_barrier();
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
  };
  // Step t: K of t + 2 and V of t + 1 go to LDS, K of t + 3 and V of t + 2 are
  // loaded, the scores of t + 1 and the rest of t computed. Tiles past the last
  // are the last once more.
  if (t_begin < ntiles) {
    Page p0 = load_page(t_begin, load_ids(t_begin));
    Page p1 = load_page(t_begin + 1, load_ids(t_begin + 1));
    Page p2 = load_page(t_begin + 2, load_ids(t_begin + 2));
    Ids ids = load_ids(t_begin + 3);
    Word4 k_reg, v_reg;
    if constexpr (kBoth) {
      const Word4 k0 = load16(kc, p0), v0 = load16(vc, p0), k1 = load16(kc, p1);
      k_reg = load16(kc, p2);
      v_reg = load16(vc, p1);
      land_k(k0, 0);
      land_v(v0, t_begin, p0, 0);
      land_k(k1, 1);
    } else if (is_v) {
      const Word4 v0 = load16(vc, p0);
      v_reg = load16(vc, p1);
      land_v(v0, t_begin, p0, 0);
    } else {
      const Word4 k0 = load16(kc, p0), k1 = load16(kc, p1);
      k_reg = load16(kc, p2);
      land_k(k0, 0);
      land_k(k1, 1);
    }
    sync_lds();
    f32x16_t s;
    if (t_begin < nend) s = scores(0);
    // K's first buffer is written next.
    sync_lds();
    for (int t = t_begin; t < ntiles; ++t) {
      const int even = (t - t_begin) & 1;
      const Page p3 = load_page(t + 3, ids);
      ids = load_ids(t + 4);
      if constexpr (kBoth) {
        land_k(k_reg, even);
        land_v(v_reg, t + 1, p1, even ^ 1);
        k_reg = load16(kc, p3);
        v_reg = load16(vc, p2);
      } else if (is_v) {
        land_v(v_reg, t + 1, p1, even ^ 1);
        v_reg = load16(vc, p2);
      } else {
        land_k(k_reg, even);
        k_reg = load16(kc, p3);
      }
      if (t < nend) {
        if (t >= nint || p0.mask != 3) mask_scores(t, p0, s);
        look(p0, s);
        Weight pf[2][kWeights];
        if constexpr (kOverlap<E>) {
          const f32x16_t ahead = scores(even ^ 1);
          weigh(p0, s, pf);
          gather(pf, even);
          s = ahead;
        } else {
          weigh(p0, s, pf);
          gather(pf, even);
          s = scores(even ^ 1);
        }
      }
      p0 = p1;
      p1 = p2;
      p2 = p3;
      sync_lds();
    }
  }

  l += lane_xor32(l, lane);  // commutative: both halves get the same sum
  if (nparts > 1) {
    // Region of (slot, head, wave): o as [i / 2][lane][2], the state as
    // [lane][4].
    auto region = [&](int p) {
      return (static_cast<int64_t>(slot + p) * c.heads + head) * kWaves + wave;
    };
    auto state = [&](int p) { return a.ws_ml + (region(p) * kWave + lane) * 4; };
    int32_t* ctr = a.counters + static_cast<int64_t>(counter) * c.heads + head;
    float* acc = a.ws_acc + region(part) * (kAccFloats * kWave) + 2 * lane;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 2)
        store_coherent2(acc + (db * 16 + i) * kWave, o[db][i], o[db][i + 1]);
    store_coherent2(state(part), m, l);
    store_coherent(state(part) + 2, mo);
    wait_stores();
    __syncthreads();  // every wave's partial is at the coherent level
    if (tid == 0)
      s_arrived = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_arrived != nparts - 1) return;  // uniform
    m = mo = -INFINITY;
    for (int p = 0; p < nparts; ++p) {
      m = fmaxf(m, load_coherent(state(p)));
      mo = fmaxf(mo, load_coherent(state(p) + 2));
    }
    // 0 times a NaN is NaN: that of a part in which nothing else was seen too.
    auto weight = [](float x, float top) { return x == -INFINITY ? 0.f : fast_exp2(x - top); };
    l = 0.f;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    for (int p = 0; p < nparts; ++p) {
      const Float2 ml = load_coherent2(state(p));
      l = fmaf(weight(ml.x, m), ml.y, l);
      const float f = weight(load_coherent(state(p) + 2), mo);
      const float* src = a.ws_acc + region(p) * (kAccFloats * kWave) + 2 * lane;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; i += 2) {
          const Float2 v = load_coherent2(src + (db * 16 + i) * kWave);
          o[db][i] = fmaf(f, v.x, o[db][i]);
          o[db][i + 1] = fmaf(f, v.y, o[db][i + 1]);
        }
    }
    if (tid == 0) __hip_atomic_store(ctr, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  if (!row_ok) return;
  // out = o 2^mo / (l 2^m), the power in two steps: it may be below 2^-126.
  const float inv = l != 0.f ? 1.f / l : 0.f;
  const float power = mo > -INFINITY ? fast_exp2(0.5f * (mo - m)) : 1.f;
  R* row = static_cast<R*>(a.out) + static_cast<int64_t>(q_begin + token) * a.o_ts +
           static_cast<int64_t>(head * G + g) * a.o_hs;
  // o[db][i]: dim 32 db + i / 4 * 8 + half * 4 + i % 4.
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      Pack<R, 4> v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v.v[j] = E::store(o[db][i + j] * power * inv * power);
      store_pack<R, 4>(row + db * 32 + i * 2 + half * 4, v);
    }
}

int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

// Workspace: [count][counters][items][m, l, mo][o].
struct Layout {
  int64_t counters, items, ml, acc, total;
  int32_t max_items;
};
Layout layout_of(int32_t num_rows, int32_t num_seqs, int32_t group, int32_t heads, int32_t dim) {
  Layout l{};
  l.max_items = prefill_items_max(num_rows, num_seqs, kBlockRows / group, heads);
  const int64_t regions = static_cast<int64_t>(prefill_items_slots(heads)) * heads * kWaves;
  l.counters = 256;
  l.items = l.counters + round256(int64_t(4) * prefill_counters(heads));
  l.ml = l.items + round256(l.max_items * static_cast<int64_t>(sizeof(PrefillItem)));
  l.acc = l.ml + round256(regions * 4 * kWave * 4);
  l.total = l.acc + regions * (dim / 2) * kWave * 4;
  return l;
}

}  // namespace

int64_t quant_prefill_workspace(int32_t num_rows, int32_t num_seqs, int32_t group, int32_t heads,
                                int32_t dim, int32_t block_size) {
  if (num_rows <= 0 || num_seqs <= 0 || group < 1 || group > kBlockRows || heads <= 0 ||
      (dim != 128 && dim != 64) || block_size < 16)
    return 0;
  const Layout l = layout_of(num_rows, num_seqs, group, heads, dim);
  return l.max_items == 0 ? 0 : l.total;
}

bool quant_prefill_mfma_supported(const QuantAttnArgs& a) {
  const QuantCache& c = a.c;
  const auto low = reinterpret_cast<uintptr_t>(c.k) | reinterpret_cast<uintptr_t>(c.v) | c.bs |
                   c.ts | c.hs;
  return low % 16 == 0 &&
         quant_prefill_workspace(a.num_rows, a.num_seqs, a.group, c.heads, c.dim, c.block_size) > 0;
}

int32_t launch_quant_prefill_plan(const int32_t* cu_q, const int32_t* cu_k, int32_t num_rows,
                                  int32_t num_seqs, int32_t group, int32_t heads, int32_t dim,
                                  void* workspace, hipStream_t stream) {
  const Layout l = layout_of(num_rows, num_seqs, group, heads, dim);
  char* ws = static_cast<char*>(workspace);
  return launch_prefill_items(cu_q, cu_k, num_rows, num_seqs, kBlockRows / group, heads, INT_MAX,
                              reinterpret_cast<PrefillItem*>(ws + l.items),
                              reinterpret_cast<int32_t*>(ws),
                              reinterpret_cast<int32_t*>(ws + l.counters), stream);
}

int32_t launch_quant_prefill_mfma(const QuantAttnArgs& args, int32_t dtype, int32_t code,
                                  void* workspace, hipStream_t stream) {
  QuantPrefillArgs a;
  static_cast<QuantAttnArgs&>(a) = args;
  const Layout l = layout_of(a.num_rows, a.num_seqs, a.group, a.c.heads, a.c.dim);
  char* ws = static_cast<char*>(workspace);
  a.items = reinterpret_cast<PrefillItem*>(ws + l.items);
  a.count = reinterpret_cast<int32_t*>(ws);
  a.counters = reinterpret_cast<int32_t*>(ws + l.counters);
  a.ws_ml = reinterpret_cast<float*>(ws + l.ml);
  a.ws_acc = reinterpret_cast<float*>(ws + l.acc);
  const int64_t grid = static_cast<int64_t>(l.max_items) * a.c.heads;
  if (grid > INT_MAX)
    return fail(MI_ERR_UNSUPPORTED, "quantized attention: too many rows for one launch");
  return with_types(dtype, code, [&](auto e, auto co) {
    using E = decltype(e);
    using C = decltype(co);
    auto go = [&](auto kernel) {
      kernel<<<static_cast<uint32_t>(grid), kThreads, 0, stream>>>(a);
      return check_launch("quantized prefill");
    };
    return a.c.dim == 128 ? go(quant_prefill_kernel<E, C, 128>)
                          : go(quant_prefill_kernel<E, C, 64>);
  });
}

}  // namespace mi
