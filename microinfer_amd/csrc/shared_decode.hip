// Decode attention of sequences that share their first pages (forks of one
// prompt, a common system prompt), gfx950.
//
// A group's shared pages are read once for all of its sequences: the query
// rows of up to 64 / G sequences (G query heads each) meet a K/V row together,
// as MFMA columns that the decode of single sequences would leave empty. With
// the rest of each context as a work item of its own, an item is
//   (query rows of one KV head, contiguous positions of one block table)
// whether it is a piece of a shared prefix (up to 64 rows) or of one
// sequence's own pages (G rows). Each item leaves its unnormalised sums
// acc = sum 2^(s - m) v, l = sum 2^(s - m) and m of every row, and a second
// launch joins the pieces of each row,
//   out = sum_i 2^(m_i - M) acc_i / sum_i 2^(m_i - M) l_i, M = max m_i.
// Whole pages are shared only, so an item has no mask but the end of its last
// tile.
//
// The plan (items, rows, pieces) is made on the device from the lengths, the
// groups and their shared pages, once for all layers of a step.
#include <algorithm>

#include "paged_attention.h"
#include "mi_fork.h"

namespace mi {
namespace {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef short short4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

template <typename E>
struct SharedMfma;
template <>
struct SharedMfma<BF16> {
  using vec8 = bf16x8_t;
  static __device__ __forceinline__ f32x4_t qk(vec8 a, vec8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t pv(short4_t a, short4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t round(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<__bf16>(x));
  }
};
template <>
struct SharedMfma<F16> {
  using vec8 = f16x8_t;
  static __device__ __forceinline__ f32x4_t qk(vec8 a, vec8 b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_t pv(short4_t a, short4_t b, f32x4_t c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4_t, a),
                                                 __builtin_bit_cast(f16x4_t, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint16_t round(float x) {
    return __builtin_bit_cast(uint16_t, static_cast<_Float16>(x));
  }
};

constexpr int kD = 128;         // head_dim
constexpr int kTile = 16;       // positions per tile
constexpr int kMaxRows = 64;    // query rows of an item
constexpr int kMaxGroup = 16;   // query heads per KV head
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;
constexpr int kSlots = 4;       // ring slots of a wave
constexpr int kRowBytes = kD * 2;
constexpr int kHalfBytes = kTile * kRowBytes;
constexpr int kSlotBytes = 2 * kHalfBytes;  // K then V of a tile
constexpr int kLoadBytes = kWave * 16;
constexpr int kLoadsPerHalf = kHalfBytes / kLoadBytes;
constexpr int kLoadsPerTile = 2 * kLoadsPerHalf;
constexpr int kAccStride = kD + 4;  // floats: rows of a wave's sums, 4 banks apart
constexpr int kRegionBytes = std::max(kSlots * kSlotBytes, kMaxRows * kAccStride * 4);
constexpr int kRescaleSlack = 15;
static_assert((kSlots - 1) * kLoadsPerTile <= 63, "vmcnt immediate");

// A piece of work, for every KV head: the rows of sequences [seq, seq + seqs)
// over positions [begin, end) of sequence seq's table. Its row r is partial
// row first_row + r.
struct alignas(32) SharedItem {
  int32_t seq, seqs, begin, end, first_row, unused[3];
};
// Where a sequence's pieces are: parts p of its group's prefix at row
// prefix_row + p * prefix_step + g, of its own pages at own_row + p G + g.
struct alignas(32) SharedSeq {
  int32_t prefix_row, prefix_step, prefix_parts, own_row, own_parts, unused[3];
};
struct alignas(32) SharedHead {
  int32_t items, unused[7];
};

constexpr int kPlanThreads = 256;
// About this many workgroups a launch.
constexpr int kTargetGroups = 512;
constexpr int kPartUnit = 64;  // a tile for every wave
constexpr int kMinPart = 128;
constexpr int kMaxPositions = 1 << 30;  // of a block table: sums of two stay int32

struct SharedSizes {
  int32_t max_items, max_rows;
  int64_t plan_bytes, workspace_bytes;
};
SharedSizes shared_sizes(int32_t num_seqs, int32_t num_kv_heads, int32_t group) {
  const int64_t target = (kTargetGroups + num_kv_heads - 1) / num_kv_heads;
  SharedSizes z;
  // A part is at least the step's positions / target long, and every tile of
  // a group (two sequences or more) and every sequence may end in a short one.
  z.max_items = static_cast<int32_t>(target + num_seqs + num_seqs / 2 + 1);
  z.max_rows = static_cast<int32_t>(target * (kMaxRows + group) + 2 * int64_t(num_seqs) * group);
  z.plan_bytes = 32 * (1 + int64_t(z.max_items) + num_seqs);
  z.workspace_bytes = int64_t(z.max_rows) * num_kv_heads * (kD + 2) * 4;
  return z;
}

struct PlanArgs {
  const int32_t* ctx;
  const int32_t* starts;
  const int32_t* shared;
  int32_t num_seqs, num_groups, num_kv_heads, group, lb, width;
  SharedHead* head;
  SharedItem* items;
  SharedSeq* seqs;
  int32_t max_items, max_rows;
};

__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(const PlanArgs a) {
  __shared__ int s_ctx[kMaxPlanSeqs];
  __shared__ int s_group[kMaxPlanSeqs];
  __shared__ int s_least[kMaxPlanSeqs];  // of a group's first sequence: shared whole pages
  __shared__ unsigned long long s_work;
  __shared__ int s_scan[kPlanThreads / kWave][4];
  const int t = threadIdx.x;
  const int per_tile = kMaxRows / a.group;  // sequences
  if (t == 0) s_work = 0;
  for (int s = t; s < a.num_seqs; s += kPlanThreads) {
    s_ctx[s] = min(max(a.ctx[s], 0), a.width << a.lb);
    // The last group that starts at or before s, if s lies in it.
    int lo = -1, hi = a.num_groups - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (a.starts[mid] <= s) lo = mid; else hi = mid - 1;
    }
    s_group[s] = lo >= 0 && a.starts[lo] <= s && s < a.starts[lo + 1] ? lo : -1;
    s_least[s] = a.width;
  }
  __syncthreads();
  for (int s = t; s < a.num_seqs; s += kPlanThreads)
    if (s_group[s] >= 0)
      atomicMin(&s_least[max(a.starts[s_group[s]], 0)], s_ctx[s] >> a.lb);
  __syncthreads();

  // Positions of s's group that all its sequences share, s's first in the
  // group and the group's end.
  auto shared_of = [&](int s, int* first, int* last) {
    const int g = s_group[s];
    *first = s;
    *last = s + 1;
    if (g < 0) return 0;
    *first = max(a.starts[g], 0);
    *last = min(a.starts[g + 1], a.num_seqs);
    if (*last - *first < 2) return 0;
    return min(max(a.shared[g], 0), s_least[*first]) << a.lb;
  };
  auto tile_seqs = [&](int s, int first, int last, int shared) {
    return shared > 0 && (s - first) % per_tile == 0 ? min(per_tile, last - s) : 0;
  };

  unsigned long long work = 0;
  for (int s = t; s < a.num_seqs; s += kPlanThreads) {
    int first, last;
    const int shared = shared_of(s, &first, &last);
    work += max(s_ctx[s] - shared, 0);
    if (tile_seqs(s, first, last, shared) > 0) work += shared;
  }
  atomicAdd(&s_work, work);
  __syncthreads();
  const int target = (kTargetGroups + a.num_kv_heads - 1) / a.num_kv_heads;
  const int unit = max(kPartUnit, 1 << a.lb);
  const unsigned long long want = (s_work + target - 1) / target;
  const int part = static_cast<int>(
      min((max(want, static_cast<unsigned long long>(kMinPart)) + unit - 1) / unit * unit,
          static_cast<unsigned long long>(kMaxPositions)));

  // Each thread's run of sequences: prefix items and rows, own items and rows
  // before it.
  const int per = (a.num_seqs + kPlanThreads - 1) / kPlanThreads;
  const int s0 = min(t * per, a.num_seqs), s1 = min(s0 + per, a.num_seqs);
  int mine[4] = {0, 0, 0, 0};
  for (int s = s0; s < s1; ++s) {
    int first, last;
    const int shared = shared_of(s, &first, &last);
    const int tile = tile_seqs(s, first, last, shared);
    if (tile > 0) {
      const int parts = (shared + part - 1) / part;
      mine[0] += parts;
      mine[1] += parts * tile * a.group;
    }
    const int own = (max(s_ctx[s] - shared, 0) + part - 1) / part;
    mine[2] += own;
    mine[3] += own * a.group;
  }
  const int lane = t % kWave, wave = t / kWave;
  int before[4], total[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int upto = wave_inclusive_scan(mine[i], lane);
    before[i] = upto - mine[i];
    if (lane == kWave - 1) s_scan[wave][i] = upto;
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    total[i] = 0;
#pragma unroll
    for (int w = 0; w < kPlanThreads / kWave; ++w) {
      if (w < wave) before[i] += s_scan[w][i];
      total[i] += s_scan[w][i];
    }
  }
  if (t == 0) a.head->items = min(total[0] + total[2], a.max_items);
  // Prefix items first (they have more rows); own rows behind prefix rows.
  int item = before[0], row = before[1], own_item = total[0] + before[2],
      own_row = total[1] + before[3];
  auto put = [&](int at, int seq, int seqs, int begin, int end, int first_row) {
    if (at >= a.max_items || first_row + seqs * a.group > a.max_rows) return;
    SharedItem it{};
    it.seq = seq;
    it.seqs = seqs;
    it.begin = begin;
    it.end = end;
    it.first_row = first_row;
    a.items[at] = it;
  };
  for (int s = s0; s < s1; ++s) {
    int first, last;
    const int shared = shared_of(s, &first, &last);
    const int tile = tile_seqs(s, first, last, shared);
    if (tile > 0) {
      for (int p = 0; p < shared; p += part) {
        put(item++, s, tile, p, min(p + part, shared), row);
        row += tile * a.group;
      }
    }
    a.seqs[s].own_row = own_row;
    const int ctx = s_ctx[s];
    int own = 0;
    for (int p = shared; p < ctx; p += part) {
      put(own_item++, s, 1, p, min(p + part, ctx), own_row);
      own_row += a.group;
      ++own;
    }
    a.seqs[s].own_parts = own;
    if (shared == 0) a.seqs[s].prefix_parts = 0;
  }
  // The prefix pieces of every sequence of a tile, by the thread that has it.
  item = before[0];
  row = before[1];
  for (int s = s0; s < s1; ++s) {
    int first, last;
    const int shared = shared_of(s, &first, &last);
    const int tile = tile_seqs(s, first, last, shared);
    const int parts = (shared + part - 1) / part;
    for (int i = 0; i < tile; ++i) {
      a.seqs[s + i].prefix_row = row + i * a.group;
      a.seqs[s + i].prefix_step = tile * a.group;
      a.seqs[s + i].prefix_parts = parts;
    }
    if (tile > 0) row += parts * tile * a.group;
  }
}

struct SharedArgs {
  const void* q;
  int64_t q_ts, q_hs;
  const void* kc;
  const void* vc;
  int64_t c_bs, c_ts, c_hs;
  const int32_t* tables;
  int64_t t_stride;
  int32_t t_width;
  void* out;
  int64_t o_ts, o_hs;
  float* ws_acc;  // [max_rows, Hkv, D]
  float* ws_ml;   // [max_rows, Hkv, 2]
  const SharedHead* head;
  const SharedItem* items;
  const SharedSeq* seqs;
  int32_t max_items, max_rows;
  int32_t num_seqs, num_kv_heads, group, block_size, lb, num_blocks;
  float scale_log2;
};

// LDS rows are 256 bytes; 16-byte chunk c of row r sits at c ^ swz(r), so that
// neither the K fragment reads nor the transposing V reads conflict.
__device__ __forceinline__ int swz_k(int r) { return r & 15; }
__device__ __forceinline__ int swz_v(int r) { return 2 * (r & 7); }

// One item with up to 16 MT query rows. Wave w takes tiles w, w + kWaves, ...
// of the positions, all rows of each, so a K/V row is read by one wave only.
template <typename E, int MT>
__device__ __forceinline__ void run_item(const SharedArgs& a, const SharedItem& it, int kv_head,
                                         char* s_ring, float (*s_m)[kMaxRows],
                                         float (*s_l)[kMaxRows]) {
  using M = SharedMfma<E>;
  using vec8 = typename M::vec8;
  using R = uint16_t;
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  const int tid = threadIdx.x;
  const int lane = tid % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(tid / kWave);
  const int G = a.group;
  const int rows = it.seqs * G;
  const int col = lane % 16;   // MFMA column: query row of a 16-row tile
  const int quad = lane / 16;  // MFMA row group: positions 4 quad .. + 3
  const int lb = a.lb;
  const int ntiles = (it.end - it.begin + kTile - 1) / kTile;
  const ConstI32* table = (const ConstI32*)(a.tables + it.seq * a.t_stride);
  const R* kc = static_cast<const R*>(a.kc) + kv_head * a.c_hs;
  const R* vc = static_cast<const R*>(a.vc) + kv_head * a.c_hs;
  const int c_ts = static_cast<int>(a.c_ts);
  uint32_t off_k[kLoadsPerHalf], off_v[kLoadsPerHalf];
#pragma unroll
  for (int u = 0; u < kLoadsPerHalf; ++u) {
    const int row = 4 * u + lane / 16;
    off_k[u] = static_cast<uint32_t>((row * c_ts + ((lane % 16) ^ swz_k(row)) * 8) * 2);
    off_v[u] = static_cast<uint32_t>((row * c_ts + ((lane % 16) ^ swz_v(row)) * 8) * 2);
  }
  char* ring = s_ring + wave * kRegionBytes;

  // Issues tile k's loads into ring slot `slot`; false for an invalid block id
  // (block 0 is read and masked).
  auto issue = [&](int slot, int k) -> bool {
    const int p0 = it.begin + k * kTile;
    const int blk = table[p0 >> lb];
    const bool ok = blk >= 0 && blk < a.num_blocks;
    const int64_t base = ok ? static_cast<int64_t>(blk) * a.c_bs +
                                  static_cast<int64_t>(p0 & (a.block_size - 1)) * a.c_ts
                            : 0;
    char* dst = ring + slot * kSlotBytes;
#pragma unroll
    for (int u = 0; u < kLoadsPerHalf; ++u) {
      lds_load16_sbase(kc + base, off_k[u], dst + u * kLoadBytes);
      lds_load16_sbase(vc + base, off_v[u], dst + kHalfBytes + u * kLoadBytes);
    }
    return ok;
  };

  f32x4_t o[MT][kD / 16];
  float m[MT], l[MT];
#pragma unroll
  for (int t = 0; t < MT; ++t) {
#pragma unroll
    for (int db = 0; db < kD / 16; ++db) o[t][db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m[t] = -INFINITY;
    l[t] = 0.f;
  }
  bool ok_slot[kSlots];
#pragma unroll
  for (int j = 0; j < kSlots; ++j) ok_slot[j] = false;
  if (wave < ntiles) {
    ok_slot[0] = issue(0, wave);
    // Query fragments (B operand): dims 32 ks + 8 quad .. + 7 of row 16 t + col.
    vec8 qf[MT][kD / 32];
#pragma unroll
    for (int t = 0; t < MT; ++t) {
      const int r = 16 * t + col;
      const int i = r / G;
      const R* qrow = static_cast<const R*>(a.q) + (it.seq + i) * a.q_ts +
                      (kv_head * G + (r - i * G)) * a.q_hs;
#pragma unroll
      for (int ks = 0; ks < kD / 32; ++ks) {
        Pack<R, 8> p = zero_pack<R, 8>();
        if (r < rows) p = load_pack<R, 8>(qrow + ks * 32 + quad * 8);
        qf[t][ks] = __builtin_bit_cast(vec8, p);
      }
    }
    // All in flight is waited for once, so that the loop's waits are its own.
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
    __atomic_signal_fence(__ATOMIC_SEQ_CST);
#pragma unroll
    for (int j = 1; j < kSlots; ++j)
      if (wave + j * kWaves < ntiles) ok_slot[j] = issue(j, wave + j * kWaves);
    int k = wave, slot = 0;
    while (true) {
      const int younger = min(kSlots - 1, (ntiles - 1 - k) / kWaves);
      if (younger == 0)
        __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
      else if (younger == 1)
        __builtin_amdgcn_s_waitcnt(vmcnt_only(kLoadsPerTile));
      else if (younger == 2)
        __builtin_amdgcn_s_waitcnt(vmcnt_only(2 * kLoadsPerTile));
      else
        __builtin_amdgcn_s_waitcnt(vmcnt_only(3 * kLoadsPerTile));
      __atomic_signal_fence(__ATOMIC_SEQ_CST);
      char* cur = ring + slot * kSlotBytes;
      bool ok = ok_slot[0];
#pragma unroll
      for (int j = 1; j < kSlots; ++j)
        if (slot == j) ok = ok_slot[j];
      const int p0 = it.begin + k * kTile;
      if (!ok || p0 + kTile > it.end) {
        // Masked rows may hold anything, and 0 * NaN is NaN: zero their V.
        const int r = lane / 4;
        if (!ok || p0 + r >= it.end) {
          char* row = cur + kHalfBytes + r * kRowBytes + (lane % 4) * 64;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<Pack<uint32_t, 4>*>(row + c * 16) = zero_pack<uint32_t, 4>();
        }
      }
      vec8 kf[kD / 32];
#pragma unroll
      for (int ks = 0; ks < kD / 32; ++ks) {
        const int chunk = (4 * ks + quad) ^ swz_k(col);
        kf[ks] = __builtin_bit_cast(
            vec8, *reinterpret_cast<const Pack<R, 8>*>(cur + col * kRowBytes + chunk * 16));
      }
      short4_t vf[kD / 16];
      {
        const int vrow = 4 * quad + col / 4;
        const char* vbase = cur + kHalfBytes + vrow * kRowBytes + 8 * (col & 1);
#pragma unroll
        for (int db = 0; db < kD / 16; ++db) {
          const int chunk = (2 * db + ((col % 4) >> 1)) ^ swz_v(vrow);
          vf[db] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) short4_t*)(vbase + chunk * 16));
        }
      }
#pragma unroll
      for (int t = 0; t < MT; ++t) {
        f32x4_t s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int ks = 0; ks < kD / 32; ++ks) s = M::qk(kf[ks], qf[t][ks], s);
        float sc[4];
        float tmax = -INFINITY;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[i] = ok && p0 + 4 * quad + i < it.end ? s[i] * a.scale_log2 : -INFINITY;
          tmax = fmaxf(tmax, sc[i]);
        }
        tmax = fmaxf(tmax, lane_xor16(tmax, lane));
        tmax = fmaxf(tmax, lane_xor32(tmax, lane));
        if (__ballot(tmax > m[t] + kRescaleSlack) != 0) {
          const float mnew = fmaxf(m[t], tmax);
          const float alpha = mnew == -INFINITY ? 1.f : fast_exp2(m[t] - mnew);
          l[t] *= alpha;
#pragma unroll
          for (int db = 0; db < kD / 16; ++db) o[t][db] *= alpha;
          m[t] = mnew;
        }
        const float neg_m = m[t] == -INFINITY ? 0.f : -m[t];
        // The weights round to the cache's type for the product; their sum
        // adds the rounded values.
        Pack<R, 4> pk;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          pk.v[i] = M::round(fast_exp2(sc[i] + neg_m));
          l[t] += E::load(pk.v[i]);
        }
        const short4_t pf = __builtin_bit_cast(short4_t, pk);
#pragma unroll
        for (int db = 0; db < kD / 16; ++db) o[t][db] = M::pv(vf[db], pf, o[t][db]);
      }
      if (k + kWaves >= ntiles) break;
      if (k + kSlots * kWaves < ntiles) {
        // This slot's fragment reads have returned; refill it.
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        __atomic_signal_fence(__ATOMIC_SEQ_CST);
        const bool next = issue(slot, k + kSlots * kWaves);
#pragma unroll
        for (int j = 0; j < kSlots; ++j)
          if (slot == j) ok_slot[j] = next;
      }
      k += kWaves;
      slot = slot + 1 == kSlots ? 0 : slot + 1;
    }
  }
  // No load is in flight and this wave's fragments are read: its region takes
  // its sums.
  __builtin_amdgcn_s_waitcnt(0x0070);
  __atomic_signal_fence(__ATOMIC_SEQ_CST);
  float* acc = reinterpret_cast<float*>(ring);
#pragma unroll
  for (int t = 0; t < MT; ++t) {
    l[t] += lane_xor16(l[t], lane);
    l[t] += lane_xor32(l[t], lane);
    const int r = 16 * t + col;
#pragma unroll
    for (int db = 0; db < kD / 16; ++db)
      *reinterpret_cast<f32x4_t*>(acc + r * kAccStride + db * 16 + 4 * quad) = o[t][db];
    if (quad == 0) {
      s_m[wave][r] = m[t];
      s_l[wave][r] = l[t];
    }
  }
  __syncthreads();
  const int d = tid % kD;
  for (int r = tid / kD; r < rows; r += kThreads / kD) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, s_m[w][r]);
    float ls = 0.f, os = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = s_m[w][r];
      const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - mx);
      ls = fmaf(f, s_l[w][r], ls);
      os = fmaf(f,
                reinterpret_cast<const float*>(s_ring + w * kRegionBytes)[r * kAccStride + d], os);
    }
    const int64_t at = static_cast<int64_t>(it.first_row + r) * a.num_kv_heads + kv_head;
    a.ws_acc[at * kD + d] = os;
    if (d == 0) {
      a.ws_ml[at * 2] = mx;
      a.ws_ml[at * 2 + 1] = ls;
    }
  }
}

template <typename E>
__global__ __launch_bounds__(kThreads) void shared_decode_kernel(const SharedArgs a) {
  __shared__ __attribute__((aligned(16))) char s_ring[kWaves * kRegionBytes];
  __shared__ float s_m[kWaves][kMaxRows];
  __shared__ float s_l[kWaves][kMaxRows];
  typedef int32_t int8v __attribute__((ext_vector_type(8)));
  using ConstItem = __attribute__((address_space(4))) const int8v;
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  const int kv_head = blockIdx.x % a.num_kv_heads;
  const int w = blockIdx.x / a.num_kv_heads;
  if (w >= ((const ConstI32*)(a.head))[0]) return;
  const SharedItem it = __builtin_bit_cast(SharedItem, ((ConstItem*)(a.items))[w]);
  // A foreign plan can give wrong attention, never an access out of bounds.
  if (it.seq < 0 || it.seqs < 1 || it.seqs > kMaxRows / a.group ||
      it.seq > a.num_seqs - it.seqs || it.begin < 0 || it.begin % kTile != 0 ||
      it.end <= it.begin || it.end > a.t_width << a.lb || it.first_row < 0 ||
      it.first_row > a.max_rows - it.seqs * a.group)
    return;
  const int rows = it.seqs * a.group;
  if (rows <= 16)
    run_item<E, 1>(a, it, kv_head, s_ring, s_m, s_l);
  else if (rows <= 32)
    run_item<E, 2>(a, it, kv_head, s_ring, s_m, s_l);
  else
    run_item<E, 4>(a, it, kv_head, s_ring, s_m, s_l);
}

constexpr int kJoinThreads = 256;

// out of one sequence and KV head from its pieces, in their order.
template <typename E>
__global__ __launch_bounds__(kJoinThreads) void shared_join_kernel(const SharedArgs a) {
  const int kv_head = blockIdx.x % a.num_kv_heads;
  const int seq = blockIdx.x / a.num_kv_heads;
  const SharedSeq q = a.seqs[seq];
  const int G = a.group;
  // As above: a foreign plan's pieces stay inside the workspace, and are no
  // more than a plan can have.
  const int prefix_parts = min(max(q.prefix_parts, 0), a.max_items);
  const int parts = prefix_parts + min(max(q.own_parts, 0), a.max_items);
  auto row_of = [&](int p) {
    const int64_t row = p < prefix_parts
                            ? q.prefix_row + static_cast<int64_t>(p) * q.prefix_step
                            : q.own_row + static_cast<int64_t>(p - prefix_parts) * G;
    return min(max(row, int64_t(0)), static_cast<int64_t>(a.max_rows - G));
  };
  constexpr int kBatch = 8;
  for (int e = threadIdx.x; e < G * kD; e += kJoinThreads) {
    const int h = e / kD, d = e % kD;
    float mx = -INFINITY, ls = 0.f, os = 0.f;
    for (int p0 = 0; p0 < parts; p0 += kBatch) {
      float mb[kBatch], lb[kBatch], ob[kBatch];
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        const int64_t at =
            (row_of(min(p0 + b, parts - 1)) + h) * a.num_kv_heads + kv_head;
        mb[b] = a.ws_ml[at * 2];
        lb[b] = a.ws_ml[at * 2 + 1];
        ob[b] = a.ws_acc[at * kD + d];
      }
#pragma unroll
      for (int b = 0; b < kBatch; ++b) {
        if (p0 + b >= parts || mb[b] == -INFINITY) continue;
        const float mnew = fmaxf(mx, mb[b]);
        const float fo = mx == -INFINITY ? 0.f : fast_exp2(mx - mnew);
        const float fb = fast_exp2(mb[b] - mnew);
        ls = fmaf(ls, fo, lb[b] * fb);
        os = fmaf(os, fo, ob[b] * fb);
        mx = mnew;
      }
    }
    const float inv = ls > 0.f ? 1.f / ls : 0.f;  // no position: zeros
    static_cast<uint16_t*>(a.out)[seq * a.o_ts + (kv_head * G + h) * a.o_hs + d] =
        E::store(os * inv);
  }
}

// Arguments that plan, sizes and call share; MI_OK if there is a kernel.
int32_t check_shape(const char* what, int32_t num_seqs, int32_t num_q_heads,
                    int32_t num_kv_heads, int32_t head_dim, int32_t block_size, int32_t width,
                    int32_t dtype) {
  const std::string name(what);
  if (!valid_dtype(dtype)) return fail(MI_ERR_INVALID_ARGUMENT, name + ": bad dtype");
  if (num_seqs < 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 || width < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, name + ": invalid sizes");
  if (num_q_heads % num_kv_heads)
    return fail(MI_ERR_INVALID_ARGUMENT,
                name + ": num_q_heads must be a multiple of num_kv_heads");
  if (!is_pow2(block_size))
    return fail(MI_ERR_INVALID_ARGUMENT, name + ": block_size must be a power of two");
  if (dtype == MI_DTYPE_F32 || head_dim != kD || num_q_heads / num_kv_heads > kMaxGroup ||
      block_size < kTile)
    return fail(MI_ERR_UNSUPPORTED,
                name + ": bf16/f16 with head_dim 128, at most 16 query heads per KV head and "
                       "blocks of at least 16 only");
  if (num_seqs > kMaxPlanSeqs)
    return fail(MI_ERR_UNSUPPORTED, name + ": more than 4096 sequences");
  if (static_cast<int64_t>(width) * block_size > kMaxPositions)
    return fail(MI_ERR_UNSUPPORTED, name + ": block tables of more than 2^30 positions");
  // The launch's threads are counted in 32 bits.
  if ((num_seqs + num_seqs / 2 + kTargetGroups + 1ll) * num_kv_heads > (1 << 23))
    return fail(MI_ERR_UNSUPPORTED, name + ": too many sequences times KV heads");
  return MI_OK;
}

bool off_grid(const void* p, uint64_t bytes) {
  return reinterpret_cast<uintptr_t>(p) % bytes != 0;
}

}  // namespace
}  // namespace mi

extern "C" int64_t mi_shared_decode_plan_bytes(int32_t num_seqs, int32_t num_q_heads,
                                               int32_t num_kv_heads) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads) return 0;
  return mi::shared_sizes(num_seqs, num_kv_heads, num_q_heads / num_kv_heads).plan_bytes;
}

extern "C" int64_t mi_shared_decode_workspace_bytes(int32_t num_seqs, int32_t num_q_heads,
                                                    int32_t num_kv_heads) {
  if (num_seqs <= 0 || num_kv_heads <= 0 || num_q_heads < num_kv_heads) return 0;
  return mi::shared_sizes(num_seqs, num_kv_heads, num_q_heads / num_kv_heads).workspace_bytes;
}

extern "C" int32_t mi_shared_decode_plan(const int32_t* context_lens, int32_t num_seqs,
                                         const int32_t* group_starts,
                                         const int32_t* shared_blocks, int32_t num_groups,
                                         int32_t num_q_heads, int32_t num_kv_heads,
                                         int32_t head_dim, int32_t block_size,
                                         int32_t block_table_width, int32_t dtype, void* plan,
                                         int64_t plan_bytes, void* stream) {
  using namespace mi;
  clear_error();
  const char* what = "mi_shared_decode_plan";
  const int32_t st = check_shape(what, num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                                 block_table_width, dtype);
  if (st != MI_OK) return st;
  if (num_groups < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_shared_decode_plan: negative num_groups");
  if (num_seqs == 0) return MI_OK;
  if (!context_lens || (num_groups > 0 && (!group_starts || !shared_blocks)))
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_shared_decode_plan: null pointer");
  if (off_grid(context_lens, 4) || off_grid(group_starts, 4) || off_grid(shared_blocks, 4))
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_shared_decode_plan: misaligned pointer");
  const int32_t group = num_q_heads / num_kv_heads;
  const SharedSizes z = shared_sizes(num_seqs, num_kv_heads, group);
  if (!plan || off_grid(plan, 32) || plan_bytes < z.plan_bytes)
    return fail(MI_ERR_WORKSPACE, "mi_shared_decode_plan: plan must be 32-byte aligned and at "
                                  "least mi_shared_decode_plan_bytes() long");
  PlanArgs a;
  a.ctx = context_lens;
  a.starts = group_starts;
  a.shared = shared_blocks;
  a.num_seqs = num_seqs;
  a.num_groups = num_groups;
  a.num_kv_heads = num_kv_heads;
  a.group = group;
  a.lb = ilog2(block_size);
  a.width = block_table_width;
  a.head = static_cast<SharedHead*>(plan);
  a.items = reinterpret_cast<SharedItem*>(a.head + 1);
  a.seqs = reinterpret_cast<SharedSeq*>(a.items + z.max_items);
  a.max_items = z.max_items;
  a.max_rows = z.max_rows;
  shared_plan_kernel<<<1, kPlanThreads, 0, static_cast<hipStream_t>(stream)>>>(a);
  return check_launch(what);
}

extern "C" int32_t mi_shared_decode(
    const void* query, int64_t q_token_stride, int64_t q_head_stride, const void* key_cache,
    const void* value_cache, int64_t cache_block_stride, int64_t cache_token_stride,
    int64_t cache_head_stride, const int32_t* block_tables, int64_t block_table_stride,
    int32_t block_table_width, const void* plan, int64_t plan_bytes, void* out,
    int64_t out_token_stride, int64_t out_head_stride, void* workspace, int64_t workspace_bytes,
    int32_t num_seqs, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
    int32_t block_size, int32_t num_blocks, float scale, int32_t dtype, void* stream) {
  using namespace mi;
  clear_error();
  const char* what = "mi_shared_decode";
  int32_t st = check_shape(what, num_seqs, num_q_heads, num_kv_heads, head_dim, block_size,
                           block_table_width, dtype);
  if (st != MI_OK) return st;
  if (num_blocks <= 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_shared_decode: invalid sizes");
  if (num_seqs == 0) return MI_OK;
  if (!query || !key_cache || !value_cache || !block_tables || !out)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_shared_decode: null pointer");
  if (off_grid(query, 16) || off_grid(key_cache, 16) || off_grid(value_cache, 16) ||
      off_grid(out, 2) || off_grid(block_tables, 4) || q_token_stride % 8 || q_head_stride % 8 ||
      cache_block_stride % 8 || cache_token_stride % 8 || cache_head_stride % 8)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_shared_decode: misaligned pointers or strides");
  if (cache_token_stride < 0 || cache_token_stride * kTile >= (int64_t(1) << 30))
    return fail(MI_ERR_UNSUPPORTED, "mi_shared_decode: token stride outside 2^26 elements");
  const int32_t group = num_q_heads / num_kv_heads;
  const SharedSizes z = shared_sizes(num_seqs, num_kv_heads, group);
  if (!plan || off_grid(plan, 32) || plan_bytes < z.plan_bytes)
    return fail(MI_ERR_WORKSPACE, "mi_shared_decode: plan must be 32-byte aligned and at least "
                                  "mi_shared_decode_plan_bytes() long");
  if (!workspace || off_grid(workspace, 16) || workspace_bytes < z.workspace_bytes)
    return fail(MI_ERR_WORKSPACE, "mi_shared_decode: workspace must be 16-byte aligned and at "
                                  "least mi_shared_decode_workspace_bytes() long");
  SharedArgs a;
  a.q = query;
  a.q_ts = q_token_stride;
  a.q_hs = q_head_stride;
  a.kc = key_cache;
  a.vc = value_cache;
  a.c_bs = cache_block_stride;
  a.c_ts = cache_token_stride;
  a.c_hs = cache_head_stride;
  a.tables = block_tables;
  a.t_stride = block_table_stride;
  a.t_width = block_table_width;
  a.out = out;
  a.o_ts = out_token_stride;
  a.o_hs = out_head_stride;
  a.ws_acc = static_cast<float*>(workspace);
  a.ws_ml = a.ws_acc + static_cast<int64_t>(z.max_rows) * num_kv_heads * kD;
  a.head = static_cast<const SharedHead*>(plan);
  a.items = reinterpret_cast<const SharedItem*>(a.head + 1);
  a.seqs = reinterpret_cast<const SharedSeq*>(a.items + z.max_items);
  a.max_items = z.max_items;
  a.max_rows = z.max_rows;
  a.num_seqs = num_seqs;
  a.num_kv_heads = num_kv_heads;
  a.group = group;
  a.block_size = block_size;
  a.lb = ilog2(block_size);
  a.num_blocks = num_blocks;
  a.scale_log2 = scale * 1.4426950408889634f;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const uint32_t blocks = static_cast<uint32_t>(z.max_items) * num_kv_heads;
  const uint32_t joins = static_cast<uint32_t>(num_seqs) * num_kv_heads;
  if (dtype == MI_DTYPE_BF16) {
    shared_decode_kernel<BF16><<<blocks, kThreads, 0, s>>>(a);
    shared_join_kernel<BF16><<<joins, kJoinThreads, 0, s>>>(a);
  } else {
    shared_decode_kernel<F16><<<blocks, kThreads, 0, s>>>(a);
    shared_join_kernel<F16><<<joins, kJoinThreads, 0, s>>>(a);
  }
  return check_launch(what);
}
