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
//  * A tile of 32 keys is widened to bf16 (exactly) once for the four waves: a
//    thread loads 16 codes of K and of V a tile ahead, and writes them to one of
//    two LDS buffers while the other is computed on. Rows of V that nothing may
//    see are written as zeros.
//  * S^T = K . Q^T on v_mfma_f32_32x32x16_bf16, Q in as many bf16 parts as hold
//    all of its bits (1 for bf16, 2 for f16, 3 for f32); the K scale meets the
//    scores in float32. A lane owns 16 keys of one row, so the softmax needs its
//    neighbour only where the reference moves and for the sum at the end.
//  * O^T += V^T . P^T on the same instruction, V^T by transposing LDS reads; a
//    weight times the V scale goes in as two bf16 parts (three for f32).
//  * Row blocks whose keys are split publish (o, m, l); the last arrival merges
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

// Workgroups of a CU, by the registers of the query's parts.
template <typename E>
constexpr int kResident = std::is_same<E, BF16>::value ? 3 : 2;

template <typename E, typename C, int D>
__global__ __launch_bounds__(kThreads, kResident<E>) void quant_prefill_kernel(
    const QuantPrefillArgs a) {
  using R = typename E::raw;
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  using ConstF32 = __attribute__((address_space(4))) const float;
  constexpr int kParts = kQueryParts<E>;
  constexpr int kWeights = std::is_same<E, F32>::value ? 3 : 2;
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
  const int nend = wave_ok ? (max(ctx - q_len + wave_tok1 + 1, 0) + kKeys - 1) / kKeys : 0;

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

  struct Stage {
    Word4 k, v;
    float ks[2], vs[2];
    int mask;  // bit h: half h is in a block of the pool
    bool zero;  // this thread's key may not be seen
  };
  auto load_stage = [&](int tile, Stage& s) __attribute__((always_inline)) {
    const int t0 = tile * kKeys;
    const int e0 = t0 >> c.log2_block;
    // The second half's entry; past the keys, the first's again.
    const int e1 = t0 + 16 < kv_end ? (t0 + 16) >> c.log2_block : e0;
    const int id0 = table[e0], id1 = table[e1];
    const bool ok0 = id0 >= 0 && id0 < c.num_blocks;
    const bool ok1 = id1 >= 0 && id1 < c.num_blocks;
    const int64_t p0 = ok0 ? id0 : 0, p1 = ok1 ? id1 : 0;
    s.mask = (ok0 ? 1 : 0) | (ok1 ? 2 : 0);
    const int64_t at = (wave_half ? p1 : p0) * c.bs +
                       ((t0 + 16 * wave_half) & (c.block_size - 1)) * c.ts;
    s.zero = t0 + key >= kv_end || !(wave_half ? ok1 : ok0);
    if constexpr (kBoth) {
      s.k = *reinterpret_cast<const Word4*>(kc + at);
      s.v = *reinterpret_cast<const Word4*>(vc + at);
    } else {
      s.k = *reinterpret_cast<const Word4*>((is_v ? vc : kc) + at);
    }
    s.ks[0] = ((const ConstF32*)ks_head)[p0 * c.s_bs];
    s.ks[1] = ((const ConstF32*)ks_head)[p1 * c.s_bs];
    s.vs[0] = ((const ConstF32*)vs_head)[p0 * c.s_bs];
    s.vs[1] = ((const ConstF32*)vs_head)[p1 * c.s_bs];
  };
  auto put = [&](const Word4& w, uint16_t* row, int swz, int first) __attribute__((always_inline)) {
    const bf16x8_t lo = widen_operand<C>(w.w[0], w.w[1]);
    const bf16x8_t hi = widen_operand<C>(w.w[2], w.w[3]);
    // `first`: which of the two chunks goes first, for the banks.
    *reinterpret_cast<bf16x8_t*>(row + ((chunk + first) ^ swz) * 8) = first ? hi : lo;
    *reinterpret_cast<bf16x8_t*>(row + ((chunk + 1 - first) ^ swz) * 8) = first ? lo : hi;
  };
  auto land = [&](const Stage& s, int buf) __attribute__((always_inline)) {
    if constexpr (kBoth) {
      put(s.k, s_k[buf] + key * D, swz_k<D>(key), 0);
      put(s.zero ? Word4{} : s.v, s_v[buf] + key * D, swz_v<D>(key), key & 1);
    } else if (is_v) {
      put(s.zero ? Word4{} : s.k, s_v[buf] + key * D, swz_v<D>(key), 0);
    } else {
      put(s.k, s_k[buf] + key * D, swz_k<D>(key), 0);
    }
  };

  // Query operand: step s holds dims 16 s + 8 half .. + 7 of the lane's row. A
  // negative softmax scale goes into the query, so that the factors of the
  // scores are positive.
  bf16x8_t qf[kParts][D / 16];
  const float scale_log2 = fabsf(a.scale_log2);
  {
    const R* row = static_cast<const R*>(a.q) + static_cast<int64_t>(q_begin + token) * a.q_ts +
                   static_cast<int64_t>(head * G + g) * a.q_hs;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      float x[8] = {};
      if (row_ok) load8<E>(row + s * 16 + half * 8, x);
      if (a.scale_log2 < 0.f) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = -x[i];
      }
      bf16x8_t p[kParts];
      split8<kParts>(x, p);
#pragma unroll
      for (int n = 0; n < kParts; ++n) qf[n][s] = p[n];
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
  float m = -INFINITY, l = 0.f;  // of the row; its half's share of the sum

  auto compute = [&](int tile, const Stage& st, int buf) __attribute__((always_inline)) {
    const uint16_t* kbuf = s_k[buf];
    const uint16_t* vbuf = s_v[buf];
    f32x16_t s;
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] = 0.f;
#pragma unroll
    for (int x = 0; x < D / 16; ++x) {
      const bf16x8_t kf = *reinterpret_cast<const bf16x8_t*>(
          kbuf + col * D + ((2 * x + half) ^ swz_k<D>(col)) * 8);
#pragma unroll
      for (int n = 0; n < kParts; ++n)
        s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(kf, qf[n][x], s, 0, 0, 0);
    }
    // s[i]: key i / 4 * 8 + half * 4 + i % 4 of the row, in half i / 8.
    const float factor[2] = {st.ks[0] * scale_log2, st.ks[1] * scale_log2};
#pragma unroll
    for (int i = 0; i < 16; ++i) s[i] *= factor[i / 8];
    if (tile >= nint || st.mask != 3) {
      const int last = min(qpos, kv_end - 1) - tile * kKeys - half * 4;
#pragma unroll
      for (int i = 0; i < 16; ++i)
        s[i] = i / 4 * 8 + i % 4 <= last && (st.mask >> (i / 8) & 1) ? s[i] : -INFINITY;
    }
    float smax = s[0];
#pragma unroll
    for (int i = 1; i < 16; ++i) smax = fmaxf(smax, s[i]);
    if (__ballot(smax > m + kRescaleSlack) != 0) {
      const float mnew = fmaxf(m, fmaxf(smax, lane_xor32(smax, lane)));
      const float alpha = mnew == -INFINITY ? 1.f : fast_exp2(m - mnew);
      l *= alpha;
#pragma unroll
      for (int db = 0; db < D / 32; ++db)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[db][i] *= alpha;
      m = mnew;
    }
    const float base = m == -INFINITY ? 0.f : m;
    // A half that is not there has a scale that is not its own.
    const float vs[2] = {st.mask & 1 ? st.vs[0] : 0.f, st.mask & 2 ? st.vs[1] : 0.f};
    bf16x8_t pf[2][kWeights];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      float weight[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const float e = fast_exp2(s[8 * h + i] - base);
        l += e;
        weight[i] = e * vs[h];
      }
      split8<kWeights>(weight, pf[h]);
    }
    // Slots 0 - 3 of a half's 8 are keys 16 h + 4 half .. + 3, the others eight
    // keys on.
#pragma unroll
    for (int db = 0; db < D / 32; ++db) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const short4_t both[2] = {read_tr16(vbuf + v_rd[db] + 16 * h * D),
                                  read_tr16(vbuf + v_rd[db] + (16 * h + 8) * D)};
        const bf16x8_t vf = __builtin_bit_cast(bf16x8_t, both);
#pragma unroll
        for (int n = 0; n < kWeights; ++n)
          o[db] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(vf, pf[h][n], o[db], 0, 0, 0);
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
  if (t_begin < ntiles) {
    Stage cur, next;
    load_stage(t_begin, cur);
    land(cur, 0);
    if (t_begin + 1 < ntiles) load_stage(t_begin + 1, next);
    sync_lds();
    for (int t = t_begin; t < ntiles; ++t) {
      const int buf = (t - t_begin) & 1;
      // The other buffer was last read before the barrier.
      if (t + 1 < ntiles) land(next, buf ^ 1);
      Stage after = next;
      if (t + 2 < ntiles) load_stage(t + 2, after);
      if (t < nend) compute(t, cur, buf);
      cur = next;
      next = after;
      sync_lds();
    }
  }

  l += lane_xor32(l, lane);  // commutative: both halves get the same sum
  if (!(l == l)) m = 0.f;  // NaN counts, whatever the maximum
  if (nparts > 1) {
    // Region of (slot, head, wave): o as [i][lane], (m, l) as [lane].
    auto region = [&](int p) {
      return (static_cast<int64_t>(slot + p) * c.heads + head) * kWaves + wave;
    };
    int32_t* ctr = a.counters + static_cast<int64_t>(counter) * c.heads + head;
    float* acc = a.ws_acc + region(part) * (kAccFloats * kWave) + 2 * lane;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; i += 2)
        store_coherent2(acc + (db * 16 + i) * kWave, o[db][i], o[db][i + 1]);
    store_coherent2(a.ws_ml + (region(part) * kWave + lane) * 2, m, l);
    wait_stores();
    __syncthreads();  // every wave's partial is at the coherent level
    if (tid == 0)
      s_arrived = __hip_atomic_fetch_add(ctr, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __syncthreads();
    if (s_arrived != nparts - 1) return;  // uniform
    float mx = -INFINITY;
    for (int p = 0; p < nparts; ++p)
      mx = fmaxf(mx, load_coherent(a.ws_ml + (region(p) * kWave + lane) * 2));
    l = 0.f;
#pragma unroll
    for (int db = 0; db < D / 32; ++db)
#pragma unroll
      for (int i = 0; i < 16; ++i) o[db][i] = 0.f;
    for (int p = 0; p < nparts; ++p) {
      const Float2 ml = load_coherent2(a.ws_ml + (region(p) * kWave + lane) * 2);
      const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - mx);
      l = fmaf(f, ml.y, l);
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
  const float inv = l != 0.f ? 1.f / l : 0.f;
  R* row = static_cast<R*>(a.out) + static_cast<int64_t>(q_begin + token) * a.o_ts +
           static_cast<int64_t>(head * G + g) * a.o_hs;
  // o[db][i]: dim 32 db + i / 4 * 8 + half * 4 + i % 4.
#pragma unroll
  for (int db = 0; db < D / 32; ++db)
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      Pack<R, 4> v;
#pragma unroll
      for (int j = 0; j < 4; ++j) v.v[j] = E::store(o[db][i + j] * inv);
      store_pack<R, 4>(row + db * 32 + i * 2 + half * 4, v);
    }
}

int64_t round256(int64_t x) { return (x + 255) / 256 * 256; }

// Workspace: [count][counters][items][m, l][o].
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
  l.acc = l.ml + round256(regions * 2 * kWave * 4);
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
