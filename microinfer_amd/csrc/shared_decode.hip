// Decode attention of sequences that share their first pages (forks of one
// prompt, a common system prompt), gfx950.
//
// A group's shared pages are read once for the query rows of up to 64 / G of its
// sequences (G query heads each), which meet a K/V row together, as MFMA columns
// that the decode of single sequences would leave empty; further 64 rows find the
// pages in the L2, where a KV head's workgroups lie on one XCD (64 sequences
// behind 3500 tokens issue loads of 156 MB a layer and read 117, of 114
// distinct). With
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
//
// Bound by latency below some 50 MB of K/V, by memory above. Measured per layer
// (block 16, 8 KV heads, bf16, captured; the plan's eighth of 6-10 us and the
// join's 2.5-4 us included), us here / each sequence reading its own context:
//   4 sequences, 500 shared tokens, 16 query heads         9.5 /  8.8
//   16 with 12000 shared, up to 500 own, 32 query heads   26.5 / 66.8
//   6 groups of 7, 300-3000 shared, 5-300 own             23.3 / 38.6
//   64 with 3500 shared, 20-700 own, 32 query heads       33.5 / 62.5
//   8 with 32000 shared, 10-100 own, 32 query heads       39.2 / 84.0
//   2 with 8000 shared                                    15.6 / 16.0
// The long prefixes reach 3.4 TB/s of distinct rows: of the 16 sequences'
// launch (20 us, 11.6 at the rate of a large read) 4 us pass before the first
// tiles are there and 1.5 at the end; between, a workgroup takes 1.2 us for
// a stage of 64 positions, and two on a CU take turns: each of the four row
// waves reads every tile, 160 KB of LDS traffic a stage. Moved by 3 % at most,
// either way: stages begun one earlier (two in flight, a barrier more), half
// the vector instructions (row sums by dot products, a maximum joined only
// when it moves, block ids from registers), 16 waves on 128 KiB, one workgroup
// per CU (10.1, 26.5, 25.5, 36.5).
#include <algorithm>
#include <type_traits>

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
constexpr int kFewRows = 16;    // up to here the waves split the positions, not the rows
constexpr int kMaxGroup = 16;   // query heads per KV head
constexpr int kWaves = 8;
constexpr int kThreads = kWaves * kWave;
constexpr int kRowBytes = kD * 2;
constexpr int kHalfBytes = kTile * kRowBytes;  // K (or V) of a tile
constexpr int kTileBytes = 2 * kHalfBytes;     // K then V
constexpr int kLoadBytes = kWave * 16;
constexpr int kLoadsPerHalf = kHalfBytes / kLoadBytes;
constexpr int kLoadsPerTile = 2 * kLoadsPerHalf;
// 64 KiB of tiles per workgroup, two workgroups per CU: a tile per wave (few
// rows), or two stages of four tiles (many).
constexpr int kRingBytes = kWaves * kTileBytes;
constexpr int kStageTiles = 4;
constexpr int kStageBytes = kStageTiles * kTileBytes;
constexpr int kRowWaves = kMaxRows / kTile;       // waves that split the rows
constexpr int kKeyWaves = kWaves / kRowWaves;     // and the tiles of a stage
constexpr int kWaveTiles = kStageTiles / kKeyWaves;
constexpr int kAccStride = kD + 4;  // floats: rows of a wave's sums, 4 banks apart
// Weights go up to 2^kMostWeight (fp16 ends at 2^16) before a row's reference
// moves.
constexpr int kMostWeight = 15;
static_assert(2 * kStageBytes == kRingBytes, "two stages");
static_assert(kStageTiles * 2 == kWaves, "a stage is one half-tile per wave");
static_assert(kKeyWaves == 2 && kWaveTiles == 2, "two key waves, 32 positions each");
static_assert(kFewRows * kD * 4 <= kTileBytes, "a wave's sums fit its tile");
static_assert(kRowWaves * kTile * kAccStride * 4 <= kRingBytes, "half the waves' sums fit");

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
constexpr int kMaxGroups = 4096;
// About this many workgroups a launch, two per CU: the 64 sequences above take
// 34 us with 512, 35.7 with 384, 40 with 256, the 8 sequences 39.2, 37.1, 37.6.
constexpr int kTargetGroups = 512;
constexpr int kPartUnit = 64;  // positions: a stage
// Every piece of a prefix leaves 64 rows for the join, so the longest context
// is cut into about kMostParts pieces, unless they would be shorter than
// kMinPart or longer than kMaxMinPart. 16 pieces and 512 positions: the 16
// sequences 25.7 us, the 64 33.6; 24 and 384: 26.9, 34.5; 32 and 256: 29.4,
// 34.5; 64 and 192: 29.2, 34.0.
constexpr int kMinPart = 128;
constexpr int kMaxMinPart = 512;
constexpr int kMostParts = 16;
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

// Own items in the order of their length, longest first, in this many classes:
// a long one that starts last would end long after the others.
constexpr int kClasses = 16;

__global__ __launch_bounds__(kPlanThreads) void shared_plan_kernel(const PlanArgs a) {
  __shared__ int s_starts[kMaxGroups + 1];
  __shared__ int s_shared[kMaxGroups];
  __shared__ int s_ctx[kMaxPlanSeqs];
  __shared__ int s_group[kMaxPlanSeqs];
  // Of a group's first sequence: the whole pages that all its contexts have.
  __shared__ int s_least[kMaxPlanSeqs];
  __shared__ unsigned long long s_work;
  __shared__ int s_longest;
  __shared__ int s_scan[kPlanThreads / kWave][4];
  __shared__ int s_class[kClasses];  // items of a class, then where its next one goes
  const int t = threadIdx.x;
  const int per_tile = kMaxRows / a.group;  // sequences
  if (t == 0) {
    s_work = 0;
    s_longest = 0;
  }
  if (t < kClasses) s_class[t] = 0;
  for (int s = t; s < a.num_seqs; s += kPlanThreads) {
    s_ctx[s] = min(max(a.ctx[s], 0), a.width << a.lb);
    s_least[s] = a.width;
  }
  for (int g = t; g < a.num_groups; g += kPlanThreads) s_shared[g] = a.shared[g];
  if (a.num_groups > 0)
    for (int g = t; g <= a.num_groups; g += kPlanThreads) s_starts[g] = a.starts[g];
  __syncthreads();
  for (int s = t; s < a.num_seqs; s += kPlanThreads) {
    // The last group that starts at or before s, if s lies in it.
    int lo = -1, hi = a.num_groups - 1;
    while (lo < hi) {
      const int mid = (lo + hi + 1) >> 1;
      if (s_starts[mid] <= s) lo = mid; else hi = mid - 1;
    }
    const bool in = lo >= 0 && s_starts[lo] <= s && s < s_starts[lo + 1];
    s_group[s] = in ? lo : -1;
    if (in) atomicMin(&s_least[max(s_starts[lo], 0)], s_ctx[s] >> a.lb);
  }
  __syncthreads();

  // Positions of s's group that all its sequences share; s's first in the
  // group and the group's end.
  auto shared_of = [&](int s, int* first, int* last) {
    const int g = s_group[s];
    *first = s;
    *last = s + 1;
    if (g < 0) return 0;
    *first = max(s_starts[g], 0);
    *last = min(s_starts[g + 1], a.num_seqs);
    if (*last - *first < 2) return 0;
    return min(max(s_shared[g], 0), s_least[*first]) << a.lb;
  };
  // Sequences of the row tile that begins with s (0: none does).
  auto tile_seqs = [&](int s, int first, int last, int shared) {
    return shared > 0 && (s - first) % per_tile == 0 ? min(per_tile, last - s) : 0;
  };

  unsigned long long work = 0;
  int longest = 0;
  for (int s = t; s < a.num_seqs; s += kPlanThreads) {
    int first, last;
    const int shared = shared_of(s, &first, &last);
    work += max(s_ctx[s] - shared, 0);
    longest = max(longest, max(s_ctx[s] - shared, shared));
    if (tile_seqs(s, first, last, shared) > 0) work += shared;
  }
  // Summed in the wave first: lanes' atomics on one word take 70 ns each. The
  // halves' sums fit 32 bits (16 sequences of 2^31 positions a lane at most).
  const int low = wave_sum_int(static_cast<int>(work & 0xffff));
  const int high = wave_sum_int(static_cast<int>(work >> 16));
#pragma unroll
  for (int i = 1; i < kWave; i *= 2) longest = max(longest, __shfl_xor(longest, i));
  if (t % kWave == 0) {
    atomicAdd(&s_work, (static_cast<unsigned long long>(high) << 16) + low);
    atomicMax(&s_longest, longest);
  }
  __syncthreads();
  const int target = (kTargetGroups + a.num_kv_heads - 1) / a.num_kv_heads;
  const int unit = max(kPartUnit, 1 << a.lb);  // a power of two
  // Rounded up; positions of 2^31 in all are divided in 32 bits, which takes
  // half a microsecond less.
  const unsigned long long all = s_work + target - 1;
  const unsigned long long want =
      all >> 32 == 0 ? static_cast<uint32_t>(all) / static_cast<uint32_t>(target) : all / target;
  const int least = min(max(s_longest / kMostParts, kMinPart), kMaxMinPart);
  const int most = static_cast<int>(min(want, static_cast<unsigned long long>(kMaxPositions)));
  const int part = (max(most, least) + unit - 1) & ~(unit - 1);
  // 0 for the longest items.
  const float per_class = kClasses / static_cast<float>(part);
  auto class_of = [&](int positions) {
    return max(kClasses - 1 - static_cast<int>((positions - 1) * per_class), 0);
  };

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
    const int own = max(s_ctx[s] - shared, 0);
    const int full = own / part, rest = own - full * part;
    if (full > 0) atomicAdd(&s_class[0], full);
    if (rest > 0) atomicAdd(&s_class[class_of(rest)], 1);
    mine[2] += full + (rest > 0);
    mine[3] += (full + (rest > 0)) * a.group;
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
  int class_begin = total[0];
  if (t < kClasses)
    for (int i = 0; i < t; ++i) class_begin += s_class[i];
  __syncthreads();
  if (t < kClasses) s_class[t] = class_begin;
  if (t == 0) a.head->items = min(total[0] + total[2], a.max_items);
  __syncthreads();

  // Prefix items first (they have more rows); own rows behind prefix rows.
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
  int item = before[0], row = before[1], own_row = total[1] + before[3];
  for (int s = s0; s < s1; ++s) {
    int first, last;
    const int shared = shared_of(s, &first, &last);
    const int tile = tile_seqs(s, first, last, shared);
    // The prefix pieces of every sequence of a tile, by the thread that has it.
    for (int i = 0; i < tile; ++i) {
      a.seqs[s + i].prefix_row = row + i * a.group;
      a.seqs[s + i].prefix_step = tile * a.group;
      a.seqs[s + i].prefix_parts = (shared + part - 1) / part;
    }
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
      const int end = min(p + part, ctx);
      put(atomicAdd(&s_class[class_of(end - p)], 1), s, 1, p, end, own_row);
      own_row += a.group;
      ++own;
    }
    a.seqs[s].own_parts = own;
    if (shared == 0) a.seqs[s].prefix_parts = 0;
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

struct Lds {
  __attribute__((aligned(16))) char ring[kRingBytes];
  __attribute__((aligned(16))) char q[kFewRows * kRowBytes];
  float m[kWaves][kFewRows], l[kWaves][kFewRows];
};

// What the loops below share: the lane's place in the MFMA tiles, its offsets
// in the direct loads of a half-tile (load u puts lane i's 16 bytes at LDS row
// 4 u + i / 16), and the block table.
template <typename E>
struct ItemLoop {
  using R = uint16_t;
  using M = SharedMfma<E>;
  using vec8 = typename M::vec8;
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  const SharedArgs& a;
  const SharedItem& it;
  const int kv_head, lane, wave, col, quad, rows;
  const ConstI32* table;
  const R* kc;
  const R* vc;

  __device__ __forceinline__ ItemLoop(const SharedArgs& args, const SharedItem& item, int head)
      : a(args), it(item), kv_head(head), lane(threadIdx.x % kWave),
        wave(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave)), col(lane % 16),
        quad(lane / 16), rows(item.seqs * args.group),
        table((const ConstI32*)(args.tables + item.seq * args.t_stride)),
        kc(static_cast<const R*>(args.kc) + head * args.c_hs),
        vc(static_cast<const R*>(args.vc) + head * args.c_hs) {}

  // Byte offset of load u of a half-tile, swizzled as K (or V) rows are.
  __device__ __forceinline__ uint32_t load_offset(int u, bool v) const {
    const int row = 4 * u + lane / 16;
    const int swz = v ? swz_v(row) : swz_k(row);
    return static_cast<uint32_t>((row * static_cast<int>(a.c_ts) + ((lane % 16) ^ swz) * 8) * 2);
  }
  // Block id of position p, clamped to the item's last position. The loops load
  // it (a scalar load) a turn before they need it.
  __device__ __forceinline__ int block_at(int p) const {
    return table[min(p, it.end - 1) >> a.lb];
  }
  // Element offset of the tile at position p, in block blk; an invalid id reads
  // block 0 (and is masked).
  __device__ __forceinline__ int64_t tile_base(int p, int blk, bool* ok) const {
    *ok = blk >= 0 && blk < a.num_blocks;
    return *ok ? static_cast<int64_t>(blk) * a.c_bs +
                     static_cast<int64_t>(p & (a.block_size - 1)) * a.c_ts
               : 0;
  }
  // Query row r (clamped to the item's) of this KV head.
  __device__ __forceinline__ const R* query_row(int r) const {
    r = min(r, rows - 1);
    const int i = r / a.group;
    return static_cast<const R*>(a.q) + (it.seq + i) * a.q_ts +
           (kv_head * a.group + (r - i * a.group)) * a.q_hs;
  }
  // Query fragments (B operand): dims 32 ks + 8 quad .. + 7 of row `col` of a
  // 16-row LDS tile laid out as K rows are; K fragments (A operand) alike.
  __device__ __forceinline__ void row_fragments(const char* tile, vec8 (&f)[kD / 32]) const {
#pragma unroll
    for (int ks = 0; ks < kD / 32; ++ks) {
      const int chunk = (4 * ks + quad) ^ swz_k(col);
      f[ks] = __builtin_bit_cast(
          vec8, *reinterpret_cast<const Pack<R, 8>*>(tile + col * kRowBytes + chunk * 16));
    }
  }
  // V^T fragments: dim 16 db + col of positions 4 quad .. + 3.
  __device__ __forceinline__ void v_fragments(const char* tile, short4_t (&f)[kD / 16]) const {
    const int row = 4 * quad + col / 4;
    const char* base = tile + row * kRowBytes + 8 * (col & 1);
#pragma unroll
    for (int db = 0; db < kD / 16; ++db) {
      const int chunk = (2 * db + ((col % 4) >> 1)) ^ swz_v(row);
      f[db] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
          (__attribute__((address_space(3))) short4_t*)(base + chunk * 16));
    }
  }
};

// A weight in the cache's type: what it rounds to, and what that leaves out,
// rounded again.
struct Weight {
  uint16_t high, low;
};

// The running softmax of one query row per lane (shared by the lanes of equal
// `col`), with the row's sums over 128 dims in o. The reference m is near the
// maximum; fp16 keeps it 2^10 below, so that only weights under 2^-35 of a
// wave's largest vanish (bf16 has float32's range).
template <typename E>
struct RowState {
  static constexpr float kBelow = std::is_same<E, F16>::value ? 10.f : 0.f;
  f32x4_t o[kD / 16];
  float m = -INFINITY, l = 0.f;
  __device__ __forceinline__ RowState() {
#pragma unroll
    for (int db = 0; db < kD / 16; ++db) o[db] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  }
  // Moves the references when some row's new scores lie too far above.
  __device__ __forceinline__ void see(float tmax, int lane) {
    tmax = fmaxf(tmax, lane_xor16(tmax, lane));
    tmax = fmaxf(tmax, lane_xor32(tmax, lane));
    if (__ballot(tmax > m + kMostWeight) == 0) return;
    const float mnew = fmaxf(m, tmax - kBelow);
    const float alpha = mnew == -INFINITY ? 1.f : fast_exp2(m - mnew);
    l *= alpha;
#pragma unroll
    for (int db = 0; db < kD / 16; ++db) o[db] *= alpha;
    m = mnew;
  }
  // The weight of a score in two halves, which meet V one after the other: to
  // 2^-16 of it in bf16, 2^-22 in fp16. One half alone leaves an output 2^-8 or
  // 2^-11 of the values off, as much again as its own rounding (16 sequences
  // behind 12000 tokens in bf16: 0.00231 of the outputs' size from 64 bits, 0.00166
  // with both, which is their rounding alone; 26.5 us either way).
  __device__ __forceinline__ Weight weigh(float score) {
    const float p = fast_exp2(score - (m == -INFINITY ? 0.f : m));
    l += p;
    Weight w;
    w.high = SharedMfma<E>::round(p);
    w.low = SharedMfma<E>::round(p - E::load(w.high));
    return w;
  }
  __device__ __forceinline__ void close(int lane) {
    l += lane_xor16(l, lane);
    l += lane_xor32(l, lane);
  }
};

// Where a few-rows wave keeps float c of row r of its sums: 16-byte chunks
// permuted within the row, or all rows' chunks would share banks.
__device__ __forceinline__ int sum_at(int r, int c) { return r * kD + (c ^ ((r & 7) * 4)); }

// Up to 16 query rows: wave w takes tiles w, w + kWaves, ... of the positions,
// and the waves' sums are joined through LDS.
template <typename E>
__device__ __forceinline__ void run_few_rows(const SharedArgs& a, const SharedItem& it,
                                             int kv_head, Lds& s) {
  using Loop = ItemLoop<E>;
  using M = SharedMfma<E>;
  using R = uint16_t;
  const Loop x(a, it, kv_head);
  const int lane = x.lane, wave = x.wave, col = x.col, quad = x.quad;
  const int ntiles = (it.end - it.begin + kTile - 1) / kTile;
  uint32_t off_k[kLoadsPerHalf], off_v[kLoadsPerHalf];
#pragma unroll
  for (int u = 0; u < kLoadsPerHalf; ++u) {
    off_k[u] = x.load_offset(u, false);
    off_v[u] = x.load_offset(u, true);
  }
  char* tile = s.ring + wave * kTileBytes;
  auto block_of = [&](int k) { return x.block_at(it.begin + k * kTile); };
  auto issue = [&](int k, int blk) -> bool {
    bool ok;
    const int64_t base = x.tile_base(it.begin + k * kTile, blk, &ok);
#pragma unroll
    for (int u = 0; u < kLoadsPerHalf; ++u) {
      lds_load16_sbase(x.kc + base, off_k[u], tile + u * kLoadBytes);
      lds_load16_sbase(x.vc + base, off_v[u], tile + kHalfBytes + u * kLoadBytes);
    }
    return ok;
  };
  const int blk0 = block_of(wave);
  int blk_next = block_of(wave + kWaves);
  if (wave < kLoadsPerHalf) {
    // A quarter of the query rows each.
    const int r = 4 * wave + lane / 16;
    lds_load16(x.query_row(r) + ((lane % 16) ^ swz_k(r)) * 8, s.q + wave * kLoadBytes);
  }
  bool ok = false;
  if (wave < ntiles) {
    ok = issue(wave, blk0);
    __builtin_amdgcn_s_waitcnt(vmcnt_only(kLoadsPerTile));
  } else {
    __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
  }
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  RowState<E> row;
  if (wave < ntiles) {
    typename M::vec8 qf[kD / 32];
    x.row_fragments(s.q, qf);
    for (int k = wave;; k += kWaves) {
      __builtin_amdgcn_s_waitcnt(vmcnt_only(0));
      asm volatile("" ::: "memory");
      const int p0 = it.begin + k * kTile;
      if (!ok || p0 + kTile > it.end) {
        // Masked rows may hold anything, and 0 * NaN is NaN: zero their V.
        const int r = lane / 4;
        if (!ok || p0 + r >= it.end) {
          char* v = tile + kHalfBytes + r * kRowBytes + (lane % 4) * 64;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            *reinterpret_cast<Pack<uint32_t, 4>*>(v + c * 16) = zero_pack<uint32_t, 4>();
        }
      }
      typename M::vec8 kf[kD / 32];
      x.row_fragments(tile, kf);
      short4_t vf[kD / 16];
      x.v_fragments(tile + kHalfBytes, vf);
      f32x4_t sc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < kD / 32; ++ks) sc = M::qk(kf[ks], qf[ks], sc);
      const bool cur_ok = ok;
      if (k + kWaves < ntiles) {
        // The tile's fragments are in registers: refill it.
        __builtin_amdgcn_s_waitcnt(0xC07F);  // lgkmcnt(0)
        asm volatile("" ::: "memory");
        ok = issue(k + kWaves, blk_next);
        blk_next = block_of(k + 2 * kWaves);
      }
      float tmax = -INFINITY;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        sc[i] = cur_ok && p0 + 4 * quad + i < it.end ? sc[i] * a.scale_log2 : -INFINITY;
        tmax = fmaxf(tmax, sc[i]);
      }
      row.see(tmax, lane);
      Pack<R, 4> high, low;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Weight w = row.weigh(sc[i]);
        high.v[i] = w.high;
        low.v[i] = w.low;
      }
      const short4_t pf = __builtin_bit_cast(short4_t, high);
      const short4_t pl = __builtin_bit_cast(short4_t, low);
#pragma unroll
      for (int db = 0; db < kD / 16; ++db) row.o[db] = M::pv(vf[db], pf, row.o[db]);
#pragma unroll
      for (int db = 0; db < kD / 16; ++db) row.o[db] = M::pv(vf[db], pl, row.o[db]);
      if (k + kWaves >= ntiles) break;
    }
  }
  // No load of this wave is in flight and its fragments are read: its tile
  // takes its sums.
  __builtin_amdgcn_s_waitcnt(0x0070);
  asm volatile("" ::: "memory");
  row.close(lane);
  float* acc = reinterpret_cast<float*>(tile);
#pragma unroll
  for (int db = 0; db < kD / 16; ++db)
    *reinterpret_cast<f32x4_t*>(acc + sum_at(col, db * 16 + 4 * quad)) = row.o[db];
  if (quad == 0) {
    s.m[wave][col] = row.m;
    s.l[wave][col] = row.l;
  }
  __syncthreads();
  const int d = threadIdx.x % kD;
  for (int r = threadIdx.x / kD; r < x.rows; r += kThreads / kD) {
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) mx = fmaxf(mx, s.m[w][r]);
    float ls = 0.f, os = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float mw = s.m[w][r];
      const float f = mw == -INFINITY ? 0.f : fast_exp2(mw - mx);
      ls = fmaf(f, s.l[w][r], ls);
      os = fmaf(f, reinterpret_cast<const float*>(s.ring + w * kTileBytes)[sum_at(r, d)], os);
    }
    const int64_t at = static_cast<int64_t>(it.first_row + r) * a.num_kv_heads + kv_head;
    a.ws_acc[at * kD + d] = os;
    if (d == 0) {
      a.ws_ml[at * 2] = mx;
      a.ws_ml[at * 2 + 1] = ls;
    }
  }
}

// More query rows: the workgroup walks the positions in stages of 64 that all
// its waves load; wave w has rows 16 (w % 4) .. + 15 and 32 of the positions
// of each stage, the first for waves 0-3, the second for waves 4-7, whose sums
// are joined at the end.
template <typename E>
__device__ __forceinline__ void run_many_rows(const SharedArgs& a, const SharedItem& it,
                                              int kv_head, Lds& s) {
  using Loop = ItemLoop<E>;
  using M = SharedMfma<E>;
  using vec8 = typename M::vec8;
  using R = uint16_t;
  const Loop x(a, it, kv_head);
  const int lane = x.lane, wave = x.wave, col = x.col, quad = x.quad;
  const int row_wave = wave % kRowWaves, key_wave = wave / kRowWaves;
  constexpr int kStage = kStageTiles * kTile;
  const int nstages = (it.end - it.begin + kStage - 1) / kStage;
  // Wave w loads K (even w) or V (odd) of tile w / 2, one of the two that it
  // computes with.
  const bool loads_v = wave & 1;
  const R* half = loads_v ? x.vc : x.kc;
  uint32_t off[kLoadsPerHalf];
#pragma unroll
  for (int u = 0; u < kLoadsPerHalf; ++u) off[u] = x.load_offset(u, loads_v);
  // First position of this wave's two tiles in stage k.
  auto begin_of = [&](int k) { return it.begin + k * kStage + key_wave * kWaveTiles * kTile; };
  struct Blocks {
    int id[kWaveTiles];
  };
  auto blocks_of = [&](int k) {
    Blocks b;
#pragma unroll
    for (int j = 0; j < kWaveTiles; ++j) b.id[j] = x.block_at(begin_of(k) + j * kTile);
    return b;
  };
  // Issues this wave's part of stage k; which of its two tiles are valid. A
  // tile past the end reads the last one.
  const int last_tile = (it.end - 1) & ~(kTile - 1);
  auto issue = [&](int k, const Blocks& blocks) -> int {
    bool ok[kWaveTiles];
    int64_t base[kWaveTiles];
#pragma unroll
    for (int j = 0; j < kWaveTiles; ++j)
      base[j] = x.tile_base(min(begin_of(k) + j * kTile, last_tile), blocks.id[j], &ok[j]);
    const int64_t mine = wave / 2 % kWaveTiles ? base[1] : base[0];
    char* dst = s.ring + (k & 1) * kStageBytes + wave * kHalfBytes;
#pragma unroll
    for (int u = 0; u < kLoadsPerHalf; ++u)
      lds_load16_sbase(half + mine, off[u], dst + u * kLoadBytes);
    return (ok[0] ? 1 : 0) | (ok[1] ? 2 : 0);
  };
  // The wave's query rows wait in the second stage's buffer, which is filled
  // when the first stage is read.
  char* q_tile = s.ring + kStageBytes + wave * kHalfBytes;
#pragma unroll
  for (int u = 0; u < kLoadsPerHalf; ++u) {
    const int r = 4 * u + lane / 16;
    lds_load16(x.query_row(kTile * row_wave + r) + ((lane % 16) ^ swz_k(r)) * 8,
               q_tile + u * kLoadBytes);
  }
  const Blocks first = blocks_of(0);
  Blocks next = blocks_of(1);
  int ok = issue(0, first);
  __builtin_amdgcn_s_waitcnt(vmcnt_only(kLoadsPerHalf));
  asm volatile("" ::: "memory");
  vec8 qf[kD / 32];
  x.row_fragments(q_tile, qf);
  const bool active = kTile * row_wave < x.rows;
  RowState<E> row;
  for (int k = 0; k < nstages; ++k) {
    // Stage k's loads of this wave are done, its earlier reads too; behind the
    // barrier those of every wave are.
    __builtin_amdgcn_s_waitcnt(0x0070);  // vmcnt(0) lgkmcnt(0)
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    const int now = ok;
    if (k + 1 < nstages) ok = issue(k + 1, next);
    next = blocks_of(k + 2);
    const int p0 = begin_of(k);
    if (!active || p0 >= it.end) continue;
    const char* stage = s.ring + (k & 1) * kStageBytes + key_wave * kWaveTiles * kTileBytes;
    f32x4_t sc[kWaveTiles];
    short4_t vf[kWaveTiles][kD / 16];
#pragma unroll
    for (int j = 0; j < kWaveTiles; ++j) {
      vec8 kf[kD / 32];
      x.row_fragments(stage + j * kTileBytes, kf);
      x.v_fragments(stage + j * kTileBytes + kHalfBytes, vf[j]);
      sc[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int ks = 0; ks < kD / 32; ++ks) sc[j] = M::qk(kf[ks], qf[ks], sc[j]);
    }
    float tmax = -INFINITY;
    if (now == 3 && p0 + kWaveTiles * kTile <= it.end) {
#pragma unroll
      for (int j = 0; j < kWaveTiles; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          sc[j][i] *= a.scale_log2;
          tmax = fmaxf(tmax, sc[j][i]);
        }
    } else {
      // Masked positions: no score, and zeros for whatever their V rows hold
      // (0 * NaN is NaN).
#pragma unroll
      for (int j = 0; j < kWaveTiles; ++j) {
        short4_t keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const bool in = (now >> j & 1) && p0 + j * kTile + 4 * quad + i < it.end;
          sc[j][i] = in ? sc[j][i] * a.scale_log2 : -INFINITY;
          tmax = fmaxf(tmax, sc[j][i]);
          keep[i] = in ? -1 : 0;
        }
#pragma unroll
        for (int db = 0; db < kD / 16; ++db) vf[j][db] &= keep;
      }
    }
    row.see(tmax, lane);
    // The contraction runs over k = 8 quad + 4 j + i: position 4 quad + i of
    // tile j, for the weights as for V.
    Pack<R, 8> high, low;
#pragma unroll
    for (int j = 0; j < kWaveTiles; ++j)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Weight w = row.weigh(sc[j][i]);
        high.v[4 * j + i] = w.high;
        low.v[4 * j + i] = w.low;
      }
    const vec8 pf = __builtin_bit_cast(vec8, high);
    const vec8 pl = __builtin_bit_cast(vec8, low);
#pragma unroll
    for (int db = 0; db < kD / 16; ++db) {
      const vec8 v8 = __builtin_bit_cast(
          vec8, __builtin_shufflevector(vf[0][db], vf[1][db], 0, 1, 2, 3, 4, 5, 6, 7));
      row.o[db] = M::qk(v8, pf, row.o[db]);
      row.o[db] = M::qk(v8, pl, row.o[db]);
    }
  }
  row.close(lane);
  // Every wave has read its last stage, no load is in flight: the second key
  // waves' sums go through the ring.
  __syncthreads();
  float* acc = reinterpret_cast<float*>(s.ring) + (row_wave * kTile + col) * kAccStride + 4 * quad;
  if (key_wave == 1 && active) {
#pragma unroll
    for (int db = 0; db < kD / 16; ++db) *reinterpret_cast<f32x4_t*>(acc + db * 16) = row.o[db];
    if (quad == 0) {
      s.m[row_wave][col] = row.m;
      s.l[row_wave][col] = row.l;
    }
  }
  __syncthreads();
  const int r = kTile * row_wave + col;
  if (key_wave == 1 || r >= x.rows) return;
  const float m1 = s.m[row_wave][col];
  const float m = fmaxf(row.m, m1);
  const float f0 = row.m == -INFINITY ? 0.f : fast_exp2(row.m - m);
  const float f1 = m1 == -INFINITY ? 0.f : fast_exp2(m1 - m);
  const int64_t at = static_cast<int64_t>(it.first_row + r) * a.num_kv_heads + kv_head;
#pragma unroll
  for (int db = 0; db < kD / 16; ++db) {
    const f32x4_t other = *reinterpret_cast<const f32x4_t*>(acc + db * 16);
    f32x4_t sum;
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[i] = fmaf(row.o[db][i], f0, other[i] * f1);
    *reinterpret_cast<f32x4_t*>(a.ws_acc + at * kD + db * 16 + 4 * quad) = sum;
  }
  if (quad == 0) {
    a.ws_ml[at * 2] = m;
    a.ws_ml[at * 2 + 1] = fmaf(row.l, f0, s.l[row_wave][col] * f1);
  }
}

template <typename E>
__global__ __launch_bounds__(kThreads, 4) void shared_decode_kernel(const SharedArgs a) {
  __shared__ Lds s;
  typedef int32_t int8v __attribute__((ext_vector_type(8)));
  using ConstItem = __attribute__((address_space(4))) const int8v;
  using ConstI32 = __attribute__((address_space(4))) const int32_t;
  const int kv_head = blockIdx.x % a.num_kv_heads;
  const int w = blockIdx.x / a.num_kv_heads;
  const SharedItem it = __builtin_bit_cast(SharedItem, ((ConstItem*)(a.items))[w]);
  if (w >= ((const ConstI32*)(a.head))[0]) return;
  // A foreign plan can give wrong attention, never an access out of bounds.
  if (it.seq < 0 || it.seqs < 1 || it.seqs > kMaxRows / a.group ||
      it.seq > a.num_seqs - it.seqs || it.begin < 0 || it.begin % kTile != 0 ||
      it.end <= it.begin || it.end > a.t_width << a.lb || it.first_row < 0 ||
      it.first_row > a.max_rows - it.seqs * a.group)
    return;
  if (it.seqs * a.group <= kFewRows)
    run_few_rows<E>(a, it, kv_head, s);
  else
    run_many_rows<E>(a, it, kv_head, s);
}

// A workgroup of two waves per query row, 16 pieces in flight: 4 us for the 7 MB
// of the 16 sequences' pieces, 2.6 for none.
constexpr int kJoinThreads = 128;
constexpr int kJoinLanes = kD / 4;  // a float4 each
constexpr int kJoinWays = kJoinThreads / kJoinLanes;
constexpr int kJoinBatch = 4;

// (m, l, o) += 2^(..) of another piece; pieces of no weight add nothing. The
// maximum passes over NaN scores, so a piece of them alone has none, and NaN for
// its sums, which have to reach the output.
__device__ __forceinline__ void join_piece(float& m, float& l, f32x4_t& o, float mb, float lb,
                                           f32x4_t ob) {
  if (mb == -INFINITY && lb == 0.f) return;
  const float mnew = fmaxf(m, mb);
  const float fo = m == -INFINITY ? 0.f : fast_exp2(m - mnew);
  const float fb = fast_exp2(mb - mnew);
  l = fmaf(l, fo, lb * fb);
  o = o * fo + ob * fb;
  m = mnew;
}

// One query row of one sequence from its pieces: way w of 4 joins pieces w, w
// + 4, ... (four at a time), then the ways are joined in order.
template <typename E>
__global__ __launch_bounds__(kJoinThreads) void shared_join_kernel(const SharedArgs a) {
  __shared__ f32x4_t s_o[kJoinWays][kJoinLanes];
  __shared__ float s_m[kJoinWays], s_l[kJoinWays];
  const int hq = a.num_kv_heads * a.group;
  const int head = blockIdx.x % hq;
  const int seq = blockIdx.x / hq;
  const int kv_head = head / a.group;
  const int g = head - kv_head * a.group;
  const SharedSeq q = a.seqs[seq];
  const int lane = threadIdx.x % kJoinLanes;
  const int way = threadIdx.x / kJoinLanes;
  // As above: a foreign plan's pieces stay inside the workspace, and are no
  // more than a plan can have.
  const int prefix_parts = min(max(q.prefix_parts, 0), a.max_items);
  const int parts = prefix_parts + min(max(q.own_parts, 0), a.max_items);
  float m = -INFINITY, l = 0.f;
  f32x4_t o = {0.f, 0.f, 0.f, 0.f};
  for (int p0 = way; p0 < parts; p0 += kJoinBatch * kJoinWays) {
    float mb[kJoinBatch], lb[kJoinBatch];
    f32x4_t ob[kJoinBatch];
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b) {
      const int p = min(p0 + b * kJoinWays, parts - 1);
      int64_t row = p < prefix_parts
                        ? q.prefix_row + static_cast<int64_t>(p) * q.prefix_step
                        : q.own_row + static_cast<int64_t>(p - prefix_parts) * a.group;
      row = min(max(row + g, int64_t(0)), static_cast<int64_t>(a.max_rows - 1));
      const int64_t at = row * a.num_kv_heads + kv_head;
      const Float2 ml = *reinterpret_cast<const Float2*>(a.ws_ml + at * 2);
      mb[b] = ml.x;
      lb[b] = ml.y;
      ob[b] = *reinterpret_cast<const f32x4_t*>(a.ws_acc + at * kD + lane * 4);
    }
#pragma unroll
    for (int b = 0; b < kJoinBatch; ++b)
      if (p0 + b * kJoinWays < parts) join_piece(m, l, o, mb[b], lb[b], ob[b]);
  }
  s_o[way][lane] = o;
  if (lane == 0) {
    s_m[way] = m;
    s_l[way] = l;
  }
  __syncthreads();
  if (way != 0) return;
#pragma unroll
  for (int w = 1; w < kJoinWays; ++w) join_piece(m, l, o, s_m[w], s_l[w], s_o[w][lane]);
  const float inv = l == 0.f ? 0.f : 1.f / l;  // no position: zeros
  Pack<uint16_t, 4> out;
#pragma unroll
  for (int i = 0; i < 4; ++i) out.v[i] = E::store(o[i] * inv);
  store_pack<uint16_t, 4>(
      static_cast<uint16_t*>(a.out) + seq * a.o_ts + head * a.o_hs + lane * 4, out);
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
  if ((num_seqs + num_seqs / 2 + kTargetGroups + 1ll) * num_q_heads > (1 << 23))
    return fail(MI_ERR_UNSUPPORTED, name + ": too many sequences times query heads");
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
  if (num_groups > kMaxGroups)
    return fail(MI_ERR_UNSUPPORTED, "mi_shared_decode_plan: more than 4096 groups");
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
  // Tables of no columns (no sequence has a context) are never read.
  if (!query || !key_cache || !value_cache || !out || (!block_tables && block_table_width > 0))
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_shared_decode: null pointer");
  if (off_grid(query, 16) || off_grid(key_cache, 16) || off_grid(value_cache, 16) ||
      off_grid(out, 16) || off_grid(block_tables, 4) || q_token_stride % 8 || q_head_stride % 8 ||
      out_token_stride % 8 || out_head_stride % 8 || cache_block_stride % 8 ||
      cache_token_stride % 8 || cache_head_stride % 8)
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
  const uint32_t joins = static_cast<uint32_t>(num_seqs) * num_q_heads;
  if (dtype == MI_DTYPE_BF16) {
    shared_decode_kernel<BF16><<<blocks, kThreads, 0, s>>>(a);
    shared_join_kernel<BF16><<<joins, kJoinThreads, 0, s>>>(a);
  } else {
    shared_decode_kernel<F16><<<blocks, kThreads, 0, s>>>(a);
    shared_join_kernel<F16><<<joins, kJoinThreads, 0, s>>>(a);
  }
  return check_launch(what);
}
