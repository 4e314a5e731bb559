// Varlen (chunked prefill, mixed) attention over an 8-bit K/V cache on MFMA:
// head_dim 64 or 128, any group of up to 128 query heads per KV head, blocks of
// at least 16, queries of any type.
//
// out = softmax(scale * q . (k * ks) + causal mask) (v * vs), with one ks and vs
// for each block and KV head. Bound by the matrix and vector units together: of a
// SIMD's time the one is busy for 27 % and the other for 45 %, and they hardly
// overlap.
//
//  * Workgroup = plan item (request, block of query rows, range of key tiles) x
//    KV head. The block's tokens times the group's heads are its rows, up to 128:
//    four waves of 32, so a key tile serves all heads of the group.
//  * 64 keys (32 for f32 with D = 128) are a step: a thread loads its codes of K
//    and V, and a step later widens them to 16-bit floats (exactly) and writes
//    them to the one of two LDS buffers that is not read. Keys that nothing may
//    see have V rows of zeros. Where the halves of 16 keys lie, and their scales,
//    is looked up for 32 steps at once, a thread for a half.
//  * S^T = K . Q^T on 32x32x16 MFMA: bf16 queries with codes as bf16, f16 with
//    codes as f16, f32 ones in three bf16 parts, which hold all of their bits.
//    The K scale meets the scores in float32. A lane owns 16 keys of one row, so
//    the softmax needs its neighbour only where a reference moves and for the
//    sum at the end.
//  * O^T += V^T . P^T on the same instruction, V^T by transposing LDS reads. A
//    weight e = 2^(score - m) meets V as e * vs * 2^(m - mo) in f16, of which mo
//    keeps the largest of the row between 2^10 and 2^15: rounding takes 2^-11 of a
//    weight (an eighth of what bf16 would, and half a step of an f16 output), and
//    what f16 cannot hold is 2^-35 of the largest. Against float64 a bf16 output is
//    off by its own rounding (2^-9.2 root mean square), an f16 one by 2^-11.9, of
//    which its own makes 2^-12.2: a second part would take that away and a fifth
//    more time (six prompts 468 us for four layers, 386 without). The 16-bit cache's
//    kernel, whose weights are of the query's type, is off by 2^-8.8 and 2^-11.8
//    over the same values. f32 queries have three parts in bf16.
//  * Row blocks whose keys are split publish theirs; the last arrival merges
//    them in order.
//
// Four layers with their plan, captured, us (the 16-bit cache's kernel): 512 tokens
// on 7700, 32 / 8 heads of 128, bf16 392 (426; 681 TFLOP/s, 58 % of a large library
// product), six prompts of 40-1400 on up to 2000, 16 / 8 heads, f16 380 (307; 557
// TFLOP/s), 300 tokens on 2000 in f32 219 (394), 500 on 4000 with heads of 64 168.
// Not faster: scores of the next step beside the softmax, staging beside the
// scores, LDS reads issued in fixed groups ahead of their products, wave
// priorities, three workgroups a CU with steps of 32 keys.
#include <algorithm>
#include <climits>

#include "quant_mfma.h"

namespace mi {
namespace {

constexpr int kTile = 32;  // keys of an MFMA, and of the plan's tiles
constexpr int kRows = 32;  // of a wave
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kBlockRows = kRows * kWaves;
constexpr float kRescaleSlack = 15.f;
// A row's largest weight lies between 2^kTopWeight and 2^kMostWeight.
constexpr float kTopWeight = 10.f, kMostWeight = 15.f;
// V of zeros has the scale 2^-126. Where a row has seen little else, mo lies that far
// below the scores, and the factor 2^(m - mo) vs of another half, if only of keys that
// the row does not see, would be infinite, which 0 times is NaN. So m stays within
// kMostApart of mo, below the row's maximum by up to kMostAbove (l, a sum of so much
// larger terms, is far from its range's end), and the factor below 2^kMostUp. Only V
// beyond 2^62 of such a scale meets that last bound, in weights of less than 2^-111.
constexpr float kMostApart = 64.f, kMostAbove = 80.f, kMostUp = 126.f;

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

// How an element type's weights meet V, and in how many parts.
template <typename E>
using WeightOperand =
    typename std::conditional<std::is_same<E, F32>::value, bf16x8_t, f16x8_t>::type;
template <typename E>
constexpr int kWeightParts = std::is_same<E, F32>::value ? 3 : 1;

// What is known of 16 keys: the factor of their scores, the V scale and its
// logarithm, whether they are in a block of the pool.
struct alignas(16) Half {
  float factor, vs, log_vs;
  int ok;
};
// `ok` of a block whose K scale is NaN: its factor is a number, so that scores which
// a row does not see stay -infinity, and the scores that it sees become NaN.
constexpr int kOkNan = 2;
constexpr int kInfo = 256;  // halves looked up, a ring of two parts

__device__ __forceinline__ f32x16_t mma(bf16x8_t a, bf16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ f32x16_t mma(f16x8_t a, f16x8_t b, f32x16_t c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}

// Tiles of a step, by the registers of the query's parts.
template <typename E, int D>
constexpr int kTiles = std::is_same<E, F32>::value && D == 128 ? 1 : 2;

template <typename E, typename C, int D>
__global__ __launch_bounds__(kThreads, 2) void quant_prefill_kernel(
    const QuantPrefillArgs a) {
  using R = typename E::raw;
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  using ConstF32 = __attribute__((address_space(4))) const float;
  using Query = QueryOperand<E>;
  using Weight = WeightOperand<E>;
  constexpr int kQueries = kQueryParts<E>, kWeights = kWeightParts<E>;
  constexpr int NT = kTiles<E, D>;
  constexpr int kKeys = NT * kTile, kHalves = 2 * NT;
  constexpr int kAccFloats = D / 32 * 16;  // of a lane
  constexpr int kLoads = kKeys * D / 16 / kThreads;  // of 16 codes a thread, for K and for V
  constexpr int kSpread = kThreads * 16 / D;         // keys between them
  static_assert(kLoads * kSpread == kKeys, "every key is loaded");
  __shared__ __attribute__((aligned(16))) uint16_t s_k[2][kKeys * D];
  __shared__ __attribute__((aligned(16))) uint16_t s_v[2][kKeys * D];
  __shared__ int64_t s_at[kInfo];
  __shared__ Half s_half[kInfo];
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
  // Keys of the block: up to the causal limit of its last token; of the item.
  const int kv_end = max(0, min(ctx - q_len + tok_last + 1, a.t_width << c.log2_block));
  const int key0 = min(it[2] * kTile, kv_end);
  const int key_end = static_cast<int>(min(static_cast<int64_t>(t_limit) * kTile,
                                           static_cast<int64_t>(kv_end)));
  const int nsteps = key_end > key0 ? (key_end - key0 + kKeys - 1) / kKeys : 0;

  const int r = wave * kRows + col;
  const int token = tok0 + r / G, g = r % G;
  const bool row_ok = r < tokens * G && token < q_len;
  const int qpos = ctx - q_len + token;  // the row sees keys 0 .. qpos
  // Of the wave's rows: steps below nint need no mask, from nend on they see
  // nothing.
  const int wave_tok0 = tok0 + wave * kRows / G;
  const int wave_tok1 = min(tok_last, tok0 + (wave * kRows + kRows - 1) / G);
  const bool wave_ok = wave * kRows < tokens * G && wave_tok0 < q_len;
  const int nint = (min(key_end, ctx - q_len + wave_tok0 + 1) - key0) / kKeys;
  const int nend =
      wave_ok ? (min(key_end, ctx - q_len + wave_tok1 + 1) - key0 + kKeys - 1) / kKeys : 0;

  // Staging: a thread's first key of a step, its 16 codes, and where they go.
  const int key = tid * 16 / D;
  const int chunk = tid % (D / 16) * 2;  // of 8 codes
  const int64_t lane_off = head * c.hs + key % 16 * c.ts + chunk * 8;
  const uint8_t* kc = c.k + lane_off;
  const uint8_t* vc = c.v + lane_off;
  const int32_t* table = a.tables + req * a.t_stride;
  const float scale_log2 = fabsf(a.scale_log2);

  // Looks up half `h` of the item.
  auto look_up = [&](int h) {
    const int pos = key0 + 16 * h;
    Half x{0x1p-126f, 0.f, 0.f, 0};
    int64_t at = 1;  // not there: block 0 is read
    if (pos < key_end) {
      const int blk = table[pos >> c.log2_block];
      if (blk >= 0 && blk < c.num_blocks) {
        at = blk * c.bs + (pos & (c.block_size - 1)) * c.ts;
        const int64_t s = blk * c.s_bs + head * c.s_hs;
        x.factor = c.ks[s] * scale_log2;
        x.ok = x.factor == x.factor ? 1 : kOkNan;
        // Masked scores are -inf, which 0 or NaN would make NaN.
        if (!(x.factor > 0.f)) x.factor = 0x1p-126f;
        x.vs = c.vs[s];
        x.log_vs = __builtin_amdgcn_logf(x.vs);
      }
    }
    s_at[h % kInfo] = at;
    s_half[h % kInfo] = x;
  };
  Word4 k_reg[kLoads], v_reg[kLoads];
  bool there[kLoads];
  auto load_step = [&](int t) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int k = key + u * kSpread;
      const int64_t at = s_at[(t * kHalves + k / 16) % kInfo];
      there[u] = (at & 1) == 0 & key0 + t * kKeys + k < key_end;
      k_reg[u] = *reinterpret_cast<const Word4*>(kc + (at & ~int64_t(1)));
      v_reg[u] = *reinterpret_cast<const Word4*>(vc + (at & ~int64_t(1)));
    }
  };
  // The second of a thread's two chunks of V goes first for odd keys, for the banks.
  const int first = D == 128 ? key & 1 : 0;
  auto land_step = [&](int t, int buf) __attribute__((always_inline)) {
#pragma unroll
    for (int u = 0; u < kLoads; ++u) {
      const int k = key + u * kSpread;
      const Word4& w = k_reg[u];
      auto put = [&](auto x, uint16_t* row, int at) __attribute__((always_inline)) {
        *reinterpret_cast<decltype(x)*>(row + at * 8) = x;
      };
      put(widen<Query, C>(w.w[0], w.w[1]), s_k[buf] + k * D, chunk ^ swz_k<D>(k));
      put(widen<Query, C>(w.w[2], w.w[3]), s_k[buf] + k * D, (chunk + 1) ^ swz_k<D>(k));
      // Keys that nothing may see may be NaN, which 0 times does not make 0.
      Word4 v = v_reg[u];
      if (__ballot(!there[u]) != 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) v.w[i] = there[u] ? v.w[i] : 0;
      }
      put(widen<Weight, C>(first ? v.w[2] : v.w[0], first ? v.w[3] : v.w[1]), s_v[buf] + k * D,
          (chunk + first) ^ swz_v<D>(k));
      put(widen<Weight, C>(first ? v.w[0] : v.w[2], first ? v.w[1] : v.w[3]), s_v[buf] + k * D,
          (chunk + 1 - first) ^ swz_v<D>(k));
    }
  };

  // Query operand: step s holds dims 16 s + 8 half .. + 7 of the lane's row. A
  // negative softmax scale goes into the query, so that the factors of the
  // scores are positive.
  Query qf[kQueries][D / 16];
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

  // s[n][i]: key 32 n + i / 4 * 8 + half * 4 + i % 4 of the row, in half 2 n + i / 8.
  auto compute = [&](int t, int buf) __attribute__((always_inline)) {
    Half hf[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) hf[h] = s_half[(t * kHalves + h) % kInfo];
    f32x16_t s[NT];
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int i = 0; i < 16; ++i) s[n][i] = 0.f;
#pragma unroll
    for (int x = 0; x < D / 16; ++x)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        const int k = 32 * n + col;
        const Query kf = *reinterpret_cast<const Query*>(
            s_k[buf] + k * D + ((2 * x + half) ^ swz_k<D>(k)) * 8);
#pragma unroll
        for (int q = 0; q < kQueries; ++q) s[n] = mma(kf, qf[q][x], s[n]);
      }
    int all = 1;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) all &= hf[h].ok;  // not those of kOkNan
    if (t >= nint || !__builtin_amdgcn_readfirstlane(all)) {
      const int last = min(qpos, key_end - 1) - key0 - t * kKeys - half * 4;
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int ok = hf[2 * n + i / 8].ok;
          const float seen = ok == kOkNan ? NAN : s[n][i];
          s[n][i] = 32 * n + i / 4 * 8 + i % 4 <= last && ok ? seen : -INFINITY;
        }
    }
    // The references move where the step's scores lie too far above them.
    float smax = -INFINITY, wmax = -INFINITY;
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      float x = s[h / 2][8 * (h % 2)];
#pragma unroll
      for (int i = 1; i < 8; ++i) x = fmaxf(x, s[h / 2][8 * (h % 2) + i]);
      x *= hf[h].factor;
      smax = fmaxf(smax, x);
      wmax = fmaxf(wmax, x + hf[h].log_vs);
    }
    if (__ballot(smax > m + kRescaleSlack || wmax > mo + kMostWeight) != 0) {
      const float monew = fmaxf(mo, fmaxf(wmax, lane_xor32(wmax, lane)) - kTopWeight);
      const float alpha = monew == -INFINITY ? 1.f : fast_exp2(mo - monew);
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
      mo = monew;
      const float stop = fmaxf(smax, lane_xor32(smax, lane));
      const float mnew = fmaxf(fmaxf(m, stop - kMostAbove), fminf(stop, mo + kMostApart));
      l *= mnew == -INFINITY ? 1.f : fast_exp2(m - mnew);
      m = mnew;
    }
    const float base = m == -INFINITY ? 0.f : m;
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      // V's fragments come while the weights are computed. Slots 0 - 3 of a half's
      // 8 are keys 16 h + 4 half .. + 3, the others eight keys on.
      Weight vf[2][D / 32];
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int db = 0; db < D / 32; ++db) {
          const uint16_t* at = s_v[buf] + v_rd[db] + (32 * n + 16 * h) * D;
          const short4_t both[2] = {read_tr16(at), read_tr16(at + 8 * D)};
          vf[h][db] = __builtin_bit_cast(Weight, both);
        }
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const Half& x = hf[2 * n + h];
        // Without a reference all scales were 0 or NaN so far, and so it stays.
        const float rise = x.log_vs + (base - mo);
        float up = fast_exp2(rise > kMostUp ? kMostUp : rise);  // NaN stays
        up = mo > -INFINITY ? up : x.vs;
        up = x.ok ? up : 0.f;
        float weight[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float e = fast_exp2(fmaf(s[n][8 * h + i], x.factor, -base));
          l += e;
          weight[i] = e * up;
        }
        Weight pf[kWeights];
        split8<kWeights>(weight, pf);
#pragma unroll
        for (int db = 0; db < D / 32; ++db)
#pragma unroll
          for (int w = 0; w < kWeights; ++w) o[db] = mma(vf[h][db], pf[w], o[db]);
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
  if (nsteps > 0) {
    constexpr int kPart = kInfo / 2;
    if (tid < kInfo) look_up(tid);
    __syncthreads();
    load_step(0);
    land_step(0, 0);
    if (nsteps > 1) load_step(1);
    sync_lds();
    auto step = [&](int t, auto parity) __attribute__((always_inline)) {
      constexpr int kBuf = decltype(parity)::value;  // LDS addresses are immediates
      // The other buffer was last read before the barrier; so was the part of the
      // ring before this step's.
      if (t + 1 < nsteps) land_step(t + 1, kBuf ^ 1);
      if (t + 2 < nsteps) load_step(t + 2);
      if (t > 0 && t * kHalves % kPart == 0 && tid < kPart) look_up(t * kHalves + kPart + tid);
      if (t < nend) compute(t, kBuf);
      sync_lds();
    };
    for (int t = 0; t < nsteps; t += 2) {
      step(t, std::integral_constant<int, 0>());
      if (t + 1 < nsteps) step(t + 1, std::integral_constant<int, 1>());
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

// ---------------------------------------------------------------------------
// The plan: every (request, row block), cut along its keys into parts of at most
// `target` tiles, largest first. With equal parts a launch takes as many rounds
// of resident workgroups as they fill, so 552 of 63 tiles on 512 places take
// twice as long as 512 of 68: the target is chosen among kCandidates by that,
// with what a part costs by itself counted as kPartTiles.
// ---------------------------------------------------------------------------
constexpr int kPlanThreads = 256;
constexpr int kPlanWaves = kPlanThreads / kWave;
constexpr int kMaxPlanBlocks = 4096;
constexpr int kMaxPlanReqs = 2048;
constexpr int kMaxParts = 16;
constexpr int kMinPartTiles = 8;
constexpr int kPartTiles = 6;
constexpr int kCandidates = 16;   // targets of 4/8 .. 19/8 of an even share
constexpr int kSlots = 1024;      // partial slots (part x KV head)
constexpr int kResident = 2;      // workgroups of a CU
constexpr int kBuckets = 2 * kPlanThreads;  // sizes >= 511 share the first

__device__ __forceinline__ int parts_of(int tiles, int target) {
  return tiles > target ? min(kMaxParts, (tiles + target - 1) / target) : 1;
}

// Exclusive scan over the workgroup, and the total.
__device__ __forceinline__ int scan(int v, int* s_wave, int& total) {
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int incl = wave_inclusive_scan(v, lane);
  if (lane == kWave - 1) s_wave[wave] = incl;
  __syncthreads();
  int before = 0;
  total = 0;
#pragma unroll
  for (int w = 0; w < kPlanWaves; ++w) {
    before += w < wave ? s_wave[w] : 0;
    total += s_wave[w];
  }
  __syncthreads();
  return before + incl - v;
}

__global__ __launch_bounds__(kPlanThreads) void quant_prefill_plan_kernel(
    const int32_t* __restrict__ cu_q, const int32_t* __restrict__ cu_k, int num_seqs, int tokens,
    int places, int heads, int max_slots, int max_items, PrefillItem* __restrict__ items,
    int32_t* __restrict__ count, int32_t* __restrict__ counters, int num_counters) {
  __shared__ int s_first[kMaxPlanReqs + 1];  // request -> first row block
  __shared__ int s_tiles[kMaxPlanBlocks];
  __shared__ int16_t s_req[kMaxPlanBlocks];
  __shared__ int s_hist[kBuckets];
  __shared__ int s_wave[kPlanWaves];
  __shared__ int s_best[kPlanWaves][2];  // estimate, target
  const int tid = threadIdx.x;
  const int lane = tid % kWave, wave = tid / kWave;
  for (int i = tid; i < num_counters; i += kPlanThreads) counters[i] = 0;
  for (int i = tid; i < kBuckets; i += kPlanThreads) s_hist[i] = 0;
  // Row blocks, in the order of their requests.
  const int per = (num_seqs + kPlanThreads - 1) / kPlanThreads;
  const int r0 = min(num_seqs, tid * per), r1 = min(num_seqs, r0 + per);
  int run = 0;
  for (int r = r0; r < r1; ++r) {
    const int n = (max(cu_q[r + 1] - cu_q[r], 0) + tokens - 1) / tokens;
    s_first[r] = n;
    run += n;
  }
  int blocks;
  int first = scan(run, s_wave, blocks);
  for (int r = r0; r < r1; ++r) {
    const int n = s_first[r];
    s_first[r] = first;
    first += n;
  }
  if (tid == 0) s_first[num_seqs] = blocks;
  __syncthreads();
  blocks = min(blocks, min(max_items - max_slots, kMaxPlanBlocks));
  int sum = 0;
  for (int q = tid; q < blocks; q += kPlanThreads) {
    int lo = 0, hi = num_seqs - 1;  // the last request whose first block <= q
    while (lo < hi) {
      const int mid = (lo + hi + 1) / 2;
      if (s_first[mid] <= q) lo = mid; else hi = mid - 1;
    }
    const int q_len = cu_q[lo + 1] - cu_q[lo];
    const int64_t ctx = static_cast<int64_t>(cu_k[lo + 1]) - cu_k[lo];
    const int last = min(q_len, (q - s_first[lo] + 1) * tokens);
    const int keys = static_cast<int>(max(int64_t(0), min(ctx - q_len + last, int64_t(1) << 30)));
    s_tiles[q] = (keys + kTile - 1) / kTile;
    s_req[q] = static_cast<int16_t>(lo);
    sum += s_tiles[q];
  }
  int total;
  scan(sum, s_wave, total);
  const int64_t share = (static_cast<int64_t>(total) * heads + places - 1) / places;
  // Each wave tries every fourth target.
  int best = INT_MAX, best_target = INT_MAX / 2;
  for (int j = wave; j < kCandidates; j += kPlanWaves) {
    const int target = max(kMinPartTiles, static_cast<int>(
        min<int64_t>((share * (4 + j) + 7) / 8, INT_MAX / 4)));
    int n = 0, split = 0, longest = 0;
    for (int q = lane; q < blocks; q += kWave) {
      const int tiles = s_tiles[q], p = parts_of(tiles, target);
      n += p;
      split += p > 1 ? p : 0;
      longest = max(longest, (tiles + p - 1) / p);
    }
    n = wave_sum_int(n);
    split = wave_sum_int(split);
#pragma unroll
    for (int o = 1; o < kWave; o <<= 1) longest = max(longest, __shfl_xor(longest, o, kWave));
    if (split > max_slots) continue;
    // Rounds of average parts, and no less than the longest.
    const int64_t rounds = (static_cast<int64_t>(n) * heads + places - 1) / places;
    const int64_t mean = (static_cast<int64_t>(total) + max(n, 1) - 1) / max(n, 1);
    const int64_t estimate =
        max(rounds * (mean + kPartTiles), static_cast<int64_t>(longest) + kPartTiles);
    if (estimate < best) {
      best = static_cast<int>(min<int64_t>(estimate, INT_MAX - 1));
      best_target = target;
    }
  }
  if (lane == 0) {
    s_best[wave][0] = best;
    s_best[wave][1] = best_target;
  }
  __syncthreads();
  int target = s_best[0][1];
  best = s_best[0][0];
#pragma unroll
  for (int w = 1; w < kPlanWaves; ++w)
    // Of equal ones the larger parts.
    if (s_best[w][0] < best || (s_best[w][0] == best && s_best[w][1] > target)) {
      best = s_best[w][0];
      target = s_best[w][1];
    }
  // Part p of n covers tiles [p * tiles / n, (p + 1) * tiles / n).
  auto bucket_of = [](int size) { return kBuckets - 1 - min(size, kBuckets - 1); };
  int nsplit = 0, nslots = 0;
  for (int q = tid; q < blocks; q += kPlanThreads) {
    const int tiles = s_tiles[q], n = parts_of(tiles, target);
    for (int p = 0; p < n; ++p)
      atomicAdd(&s_hist[bucket_of((p + 1) * tiles / n - p * tiles / n)], 1);
    nsplit += n > 1;
    nslots += n > 1 ? n : 0;
  }
  int all;
  int unit = scan(nsplit, s_wave, all);
  int slot = scan(nslots, s_wave, all);
  const int h0 = s_hist[2 * tid], h1 = s_hist[2 * tid + 1];
  const int start = scan(h0 + h1, s_wave, all);
  s_hist[2 * tid] = start;
  s_hist[2 * tid + 1] = start + h0;
  if (tid == 0) count[0] = min(all, max_items);
  __syncthreads();
  for (int q = tid; q < blocks; q += kPlanThreads) {
    const int tiles = s_tiles[q], n = parts_of(tiles, target);
    for (int p = 0; p < n; ++p) {
      PrefillItem it;
      it.req = s_req[q];
      it.qblock = q - s_first[it.req];
      it.tile_begin = p * tiles / n;
      it.tile_end = (p + 1) * tiles / n;
      it.part = p;
      it.nparts = n;
      it.slot = n > 1 ? slot : 0;
      it.counter = n > 1 ? unit : 0;
      const int pos = atomicAdd(&s_hist[bucket_of(it.tile_end - it.tile_begin)], 1);
      if (pos < max_items) items[pos] = it;
    }
    if (n > 1) {
      slot += n;
      ++unit;
    }
  }
}

int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

// Workspace: [count][counters][items][m, l, mo][o].
struct Layout {
  int64_t counters, items, ml, acc, total;
  int32_t max_items, max_slots, num_counters;
};
// max_items 0: too many requests or row blocks.
Layout layout_of(int32_t num_rows, int32_t num_seqs, int32_t group, int32_t heads, int32_t dim) {
  Layout l{};
  const int tokens = kBlockRows / group;
  const int64_t blocks = (static_cast<int64_t>(num_rows) + tokens - 1) / tokens + num_seqs;
  if (num_seqs > kMaxPlanReqs || blocks > kMaxPlanBlocks) return l;
  l.max_slots = std::max(2, kSlots / heads);
  l.max_items = static_cast<int32_t>(blocks) + l.max_slots;
  l.num_counters = l.max_slots / 2 * heads;
  const int64_t regions = static_cast<int64_t>(l.max_slots) * heads * kWaves;
  l.counters = 256;
  l.items = l.counters + round256(int64_t(4) * l.num_counters);
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

int32_t launch_quant_prefill_plan(const int32_t* cu_q, const int32_t* cu_k, int32_t num_rows,
                                  int32_t num_seqs, int32_t group, int32_t heads, int32_t dim,
                                  void* workspace, hipStream_t stream) {
  const Layout l = layout_of(num_rows, num_seqs, group, heads, dim);
  char* ws = static_cast<char*>(workspace);
  quant_prefill_plan_kernel<<<1, kPlanThreads, 0, stream>>>(
      cu_q, cu_k, num_seqs, kBlockRows / group, kResident * device_cus(), heads, l.max_slots,
      l.max_items, reinterpret_cast<PrefillItem*>(ws + l.items), reinterpret_cast<int32_t*>(ws),
      reinterpret_cast<int32_t*>(ws + l.counters), l.num_counters);
  return check_launch("quantized prefill plan");
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
