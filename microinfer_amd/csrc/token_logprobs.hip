// Log probabilities of given tokens, entropy and the best alternatives of each
// row of logits: one pass over the logits, one launch.
//
// With x the row, c = log2(e) / temperature and any reference r,
//   S = sum 2^((x_v - r) c),  E = sum 2^((x_v - r) c) (x_v - r) c,
//   ln p[v] = ln 2 ((x_v - r) c - log2 S),  entropy = ln 2 (log2 S - E / S).
// The sums do not need r to be the maximum, only near it: a wave keeps its
// first tile's maximum and moves it when a later value lies more than
// 2^kSlack above, which hardly ever happens, and sums of another reference
// scale by 2^((r - r') c). The difference is taken before the product, so rows
// whose maximum is the type's lowest value stay right.
//
// The alternatives come out of the same registers. A row's values order as
// 64-bit words (order key of the value, then the lower index). Each wave keeps
// a list of candidates of its own in LDS: after the first tile each finds the
// key that a quarter of num_top of its lanes' maxima reach, and as at least
// num_top values are no smaller than the least of these four, only values from
// that floor on can matter (about num_top / 4 of a wave's 2048 ordinary
// values). From then on, without barriers, the floor follows the lanes' maxima.
// At the end the highest of the waves' floors holds for the workgroup; what
// lies above it, some tens of words, is ranked. A tile with too many values at
// its floor (equal or masked ones) leaves those out, and if they are needed
// they are taken in order of their index by a scan at the end. Tiles with a
// NaN compare order keys instead of values.
//
// Few rows are split over many workgroups: each publishes (maximum, S, E) and
// its own best words, and the last to arrive at the row's counter joins them.
//
// Bound by memory for many rows (about ten operations an element, one of them
// an exp2 at a quarter of the rate): 3000 rows of 151936 in bf16 with entropy
// 164-172 us, 5.3-5.5 TB/s, a large read's rate; with 20 alternatives 195. By
// latency for few: 64 rows 11.6 us with entropy, 19.2 with 20 alternatives as
// well (3.5 at the rate of a read); one row 5.3, and 9.3 with 5 alternatives.
// 333 float32 rows of 32003 values in unaligned rows, 8 alternatives: 18.5-20.4
// (7.6); 3000 of 151936 in float32 302, 332 with 20 alternatives (323). The
// lists suit rows whose first tile tells what is large: with 20 alternatives and
// entropy 64 rows take 20 us, also with nine values in ten masked, but 91 with the
// first 8192 masked and 142 rising; 3000 rows 194, 498 and 5919 (each tile of a
// rising row overflows the lists).
#include <algorithm>

#include "mi_common.h"
#include "mi_fork.h"

namespace mi {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxTop = 32;
constexpr int kListCap = 2048;  // words of the LDS list
// Parts of a row: every part's best words fit the list when they are joined.
constexpr int kMaxParts = kListCap / kMaxTop;
// Sums taken relative to a value up to 2^kSlack too small: no overflow near,
// and (x - r) c of at most 10 rounds to 2^-21 when it is scaled.
constexpr float kSlack = 10.f;
constexpr float kLowest = -3.4028234663852886e38f;
// log2(e) / temperature is finite from here on: the smallest normal number.
constexpr float kLeastTemperature = 1.1754943508222875e-38f;
constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct LogprobArgs {
  const void* logits;
  int64_t row_stride;
  int32_t vocab, parts, part_packs;  // part_packs: 16-byte packs of a part
  const float* temperatures;
  const int64_t* tokens;
  int64_t token_stride;
  int32_t given;
  float* logprobs;
  float* entropy;
  int64_t* top_tokens;
  float* top_logprobs;
  int32_t top;
  char* workspace;  // [rows, parts] records of part_bytes
  int32_t part_bytes;
  int32_t* counters;
};

constexpr uint32_t kNanKey = 0xffffffffu;
constexpr uint32_t kInfKey = 0xff800000u;      // of +inf
constexpr uint32_t kMinusInfKey = 0x007fffffu;  // of -inf, the least

// Unsigned order of float values: NaN above everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float v) {
  uint32_t b = __float_as_uint(v);
  if (v != v) return kNanKey;
  if ((b << 1) == 0) b = 0;
  return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}
// Larger for larger values, then for lower indices; never 0 or ~0.
__device__ __forceinline__ uint64_t make_word(float v, uint32_t index) {
  return (static_cast<uint64_t>(order_key(v)) << 32) | (0x7fffffffu - index);
}
__device__ __forceinline__ uint32_t word_index(uint64_t w) {
  return 0x7fffffffu - static_cast<uint32_t>(w);
}

// The largest t with at least n lanes' keys >= t, in the upper BITS bits: the
// n-th largest key of the wave, its lower bits cleared (n <= 64).
template <int BITS>
__device__ __forceinline__ uint32_t nth_key(uint32_t key, int n) {
  uint32_t t = 0;
#pragma unroll
  for (int b = 31; b >= 32 - BITS; --b) {
    const uint32_t trial = t | (1u << b);
    if (__popcll(__ballot(key >= trial)) >= n) t = trial;
  }
  return t;
}

// Bits of an order key that can differ between values of the type; the lower
// ones are all zeros, or all ones for negative values.
template <typename E>
struct KeyBits;
template <>
struct KeyBits<F32> {
  static constexpr int value = 32;
};
template <>
struct KeyBits<F16> {
  static constexpr int value = 19;
};
template <>
struct KeyBits<BF16> {
  static constexpr int value = 16;
};

// nth_key of values of the type, at least -inf's.
template <typename E>
__device__ __forceinline__ uint32_t nth_value_key(uint32_t key, int n) {
  constexpr int kBits = KeyBits<E>::value;
  uint32_t t = nth_key<kBits>(key, n);
  if (kBits < 32 && !(t & 0x80000000u)) t |= 0xffffffffu >> (kBits & 31);
  return t > kInfKey ? kNanKey : max(t, kMinusInfKey);
}

// The n-th largest word of the wave, or a word below it and above the next
// smaller value's words.
template <typename E>
__device__ __forceinline__ uint64_t nth_word(uint64_t word, int n) {
  const uint32_t key = static_cast<uint32_t>(word >> 32);
  const uint32_t hi = nth_key<KeyBits<E>::value>(key, n);
  const int equal = __popcll(__ballot(key >> (32 - KeyBits<E>::value) ==
                                      hi >> (32 - KeyBits<E>::value)));
  uint32_t lo = 0;
  if (equal > 4) {
    // Ties: the lower indices among them.
    constexpr uint32_t kLow = 0xffffffffu >> (KeyBits<E>::value - 1) >> 1;
    const int above = __popcll(__ballot(key > (hi | kLow)));
    const uint32_t full = hi & 0x80000000u ? hi : hi | kLow;
    lo = nth_key<32>(key == full ? static_cast<uint32_t>(word) : 0u, n - above);
    return (static_cast<uint64_t>(full) << 32) | lo;
  }
  return static_cast<uint64_t>(hi) << 32;
}

constexpr int kWaveCap = kListCap / kWaves;
constexpr int kTilePasses = 4;  // packs per thread and tile
constexpr int kScanLanes = 32;
// Parts' words that are ranked as they are, without a floor first: 24 of 333
// rows 19.4 us, 20.2 with one; but 50 of 64 rows 16.7, 16.4, 200 22.4, 19.3.
constexpr int kFewWords = 32;
constexpr int kKeptWords = 256;  // what compress() leaves at most: kMaxTop per list slice

// LDS of a launch: with the lists of the alternatives, or without.
template <bool TOP>
struct Shared {
  float wave_ref[kWaves], wave_sum[kWaves], wave_ent[kWaves];
  int32_t arrived;
};
template <>
struct Shared<true> : Shared<false> {
  // The waves' lists; joining parts, the row's.
  uint64_t list[kListCap + 8];
  uint64_t kept[kMaxTop];  // the best words, largest first
  // Packs of lanes whose values are looked through, and whose they are; once the
  // tiles are done, the workgroup's list.
  union {
    __attribute__((aligned(16))) char scan[kWaves][kScanLanes * kTilePasses * 16];
    uint64_t best[kWaves * kKeptWords + 8];
  };
  uint8_t scan_lane[kWaves][kScanLanes];
  uint32_t wave_key[kWaves];    // what each wave contributes to the shared floor
  uint32_t wave_first[kWaves];  // the num_top-th key of each wave's first tile
  uint32_t wave_floor[kWaves];
  int32_t wave_open[kWaves];  // values equal to the wave's floor are left out
  int32_t count;              // words in the workgroup's list
  int32_t fill[kWaves];
};
using Lists = Shared<true>;

// Each wave shares the key that top / kWaves of its lanes reach; the least of
// these is reached by top values of the workgroup. Waves read it as it comes:
// the keys only rise, so an old one is a floor too.
__device__ __forceinline__ void share(Lists& s, int wave, uint32_t key) {
  __hip_atomic_store(&s.wave_key[wave], key, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_WORKGROUP);
}
__device__ __forceinline__ uint32_t shared_floor(Lists& s) {
  uint32_t key = kNanKey;
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    key = min(key, __hip_atomic_load(&s.wave_key[w], __ATOMIC_RELAXED,
                                     __HIP_MEMORY_SCOPE_WORKGROUP));
  return __builtin_amdgcn_readfirstlane(key);
}

// The `top` largest of list[0, n) into kept[0, top), largest first, zeros
// behind them: each word's rank is the number of larger ones. All threads,
// after a barrier; eight words behind the last are overwritten.
__device__ void rank_words(Lists& s, uint64_t* list, int n, int top) {
  const int t = threadIdx.x;
  if (t < 8) list[n + t] = 0;
  if (t < top) s.kept[t] = 0;
  __syncthreads();
  for (int at = t; at < n; at += kThreads) {
    const uint64_t w = list[at];
    int rank = 0;
    for (int j = 0; j < n; j += 8) {
#pragma unroll
      for (int k = 0; k < 8; ++k) rank += list[j + k] > w;
    }
    if (rank < top) s.kept[rank] = w;
  }
  __syncthreads();
}

// Appends the first `want` indices of [lo, hi) whose value has key `key` to
// best. All threads.
template <typename E>
__device__ void fill_equal(Lists& s, const typename E::raw* row, int lo, int hi, uint32_t key,
                           int want) {
  const int t = threadIdx.x;
  const int lane = t % kWave, wave = t / kWave;
  int found = 0;
  const int start = s.count;
  __syncthreads();
  for (int at = lo; at < hi && found < want; at += kThreads) {
    const int v = at + t;
    const bool hit = v < hi && order_key(E::load(row[v])) == key;
    const uint64_t hits = __ballot(hit);
    if (lane == 0) s.fill[wave] = __popcll(hits);
    __syncthreads();
    int before = found, all = found;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      if (w < wave) before += s.fill[w];
      all += s.fill[w];
    }
    before += __popcll(hits & ((1ull << lane) - 1));
    if (hit && before < want) s.best[start + before] = make_word(key_value(key), v);
    found = all;
    __syncthreads();
  }
  if (t == 0) s.count = start + min(found, want);
  __syncthreads();
}

// A wave's candidates.
struct Candidates {
  uint64_t* list;      // kWaveCap words
  int count = 0;       // wave-uniform, as all of this
  int raised_at = 0;   // the count when the floor was last looked at
  bool first = true;   // no floor yet
  bool open = false;   // values equal to the floor are not in the list
  uint32_t floor = 0;  // key

  // Keeps about the `top` largest words (at most `top` words a lane's slice
  // holds), and raises the floor to the least of `top` of them.
  __device__ void compress(int top) {
    const int lane = threadIdx.x % kWave;
    uint64_t mine[kWaveCap / kWave];
    uint64_t best = 0;
#pragma unroll
    for (int i = 0; i < kWaveCap / kWave; ++i) {
      const int at = i * kWave + lane;
      mine[i] = at < count ? list[at] : 0;
      best = mine[i] > best ? mine[i] : best;
    }
    const uint32_t hi = nth_key<32>(static_cast<uint32_t>(best >> 32), top);
    const uint32_t key = static_cast<uint32_t>(best >> 32);
    const uint32_t lo = nth_key<32>(key == hi ? static_cast<uint32_t>(best) : 0u,
                                    top - __popcll(__ballot(key > hi)));
    const uint64_t least = (static_cast<uint64_t>(hi) << 32) | lo;
    count = 0;
#pragma unroll
    for (int i = 0; i < kWaveCap / kWave; ++i) {
      const bool keep = mine[i] != 0 && mine[i] >= least;
      const uint64_t hits = __ballot(keep);
      if (keep) list[count + __popcll(hits & ((1ull << lane) - 1))] = mine[i];
      count += __popcll(hits);
    }
    raise(hi);
    raised_at = count;
  }

  // A floor that `top` values of the list reach.
  __device__ void raise(uint32_t key) {
    if (key <= floor) return;
    floor = key;
    open = false;
  }

  // Leaves out of the list what is not above `key`, the new floor.
  __device__ void reopen(uint32_t key) {
    const int lane = threadIdx.x % kWave;
    int kept = 0;
    for (int i = 0; i < count; i += kWave) {
      const uint64_t w = i + lane < count ? list[i + lane] : 0;
      const bool keep = static_cast<uint32_t>(w >> 32) > key;
      const uint64_t hits = __ballot(keep);
      if (keep) list[kept + __popcll(hits & ((1ull << lane) - 1))] = w;
      kept += __popcll(hits);
    }
    raised_at = count = kept;
    floor = key;
    open = true;
  }
};

__device__ __forceinline__ void store_agent(uint64_t* p, uint64_t v) {
  __hip_atomic_store(p, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ uint64_t load_agent(const uint64_t* p) {
  return __hip_atomic_load(const_cast<uint64_t*>(p), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// Adds sums of reference r to those of reference `to`: NaN sums stay NaN.
__device__ __forceinline__ void add_sums(float r, float sum, float ent, float to, float c,
                                         float& S, float& E) {
  const float d = (r - to) * c;
  const float f = fast_exp2(d);
  S += sum * f;
  if (!(f == 0.f)) E += f * fmaf(sum, d, ent);
}

// What a row's outputs need once its sums and best words are known. All
// threads.
template <typename E, bool TOP>
__device__ void write_row(const LogprobArgs& a, const Shared<TOP>& s, int row,
                          const typename E::raw* logits, float r, float temperature, float S,
                          float ent) {
  const float log_sum = log2f(S);
  // In nats from the start: (x - r) c overflows where x is float32's lowest value.
  auto logprob = [&](float x) { return (x - r) / temperature - kLn2 * log_sum; };
  for (int i = threadIdx.x; i < a.given; i += kThreads) {
    const int64_t token = a.tokens[row * a.token_stride + i];
    float lp = NAN;
    if (token >= 0 && token < a.vocab) lp = logprob(E::load(logits[token]));
    a.logprobs[static_cast<int64_t>(row) * a.given + i] = lp;
  }
  if (a.entropy != nullptr && threadIdx.x == 0) a.entropy[row] = kLn2 * (log_sum - ent / S);
  if constexpr (TOP) {
    if (threadIdx.x < a.top) {
      const uint64_t w = s.kept[threadIdx.x];
      const int64_t at = static_cast<int64_t>(row) * a.top + threadIdx.x;
      a.top_tokens[at] = word_index(w);
      a.top_logprobs[at] = logprob(key_value(static_cast<uint32_t>(w >> 32)));
    }
  }
}

// NP packs of VEC elements per thread make a tile.
template <typename E, bool TOP, bool ENT>
__global__ __launch_bounds__(kThreads, 4) void logprob_kernel(const LogprobArgs a) {
  using R = typename E::raw;
  constexpr int VEC = 16 / sizeof(R);
  constexpr int NP = kTilePasses;
  constexpr int kTilePacks = kThreads * NP;
  __shared__ Shared<TOP> s;
  const int row = blockIdx.x / a.parts;
  const int part = blockIdx.x - row * a.parts;
  const int t = threadIdx.x;
  const int lane = t % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const R* logits = static_cast<const R*>(a.logits) + row * a.row_stride;
  float temperature = a.temperatures == nullptr ? 1.f : a.temperatures[row];
  if (!(temperature >= kLeastTemperature && temperature < INFINITY)) temperature = NAN;
  const float c = kLog2E / temperature;
  // Packs lie on the 16-byte grid; the row's first and last may be partial.
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(logits) & 15u) / sizeof(R));
  const R* grid = logits - lead;
  const int pack_begin = part * a.part_packs;
  const int pack_end = min((lead + a.vocab + VEC - 1) / VEC, pack_begin + a.part_packs);
  const int v_begin = max(0, pack_begin * VEC - lead);

  float ref = -INFINITY;   // wave-uniform reference of the sums; -inf: none yet
  float sum = 0.f, ent = 0.f, top_value = -INFINITY;
  Candidates cand;
  if constexpr (TOP) cand.list = s.list + wave * kWaveCap;
  uint32_t lane_key = 0;  // of the lane's largest value
  const int quarter = (a.top + kWaves - 1) / kWaves;

  // Pack u of this thread in the tile that begins at pack p0, -inf outside the
  // row.
  auto load_tile = [&](int p0, int u) {
    const int p = p0 + u * kThreads + t;
    const int v0 = p * VEC - lead;
    Pack<R, VEC> x;
    if (p < pack_end && v0 >= 0 && v0 + VEC <= a.vocab) {
      x = load_pack<R, VEC>(grid + static_cast<int64_t>(p) * VEC);
    } else {
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        x.v[j] = E::store(-INFINITY);
        if (p < pack_end && v0 + j >= 0 && v0 + j < a.vocab) x.v[j] = logits[v0 + j];
      }
    }
    return x;
  };

  for (int p0 = pack_begin; p0 < pack_end; p0 += kTilePacks) {
    Pack<R, VEC> x[NP];
    const int wave_begin = p0 + wave * kWave;
    const int wave_end = wave_begin + (NP - 1) * kThreads + kWave;
    if (wave_begin * VEC >= lead && wave_end <= pack_end && wave_end * VEC - lead <= a.vocab) {
      // All of the wave's packs are whole: its loads go out together.
#pragma unroll
      for (int u = 0; u < NP; ++u) {
        const int64_t pack = wave_begin + u * kThreads + lane;
        x[u] = load_pack<R, VEC>(grid + pack * VEC);
      }
    } else {
#pragma unroll
      for (int u = 0; u < NP; ++u) x[u] = load_tile(p0, u);
    }
    float tile_max = -INFINITY;
#pragma unroll
    for (int u = 0; u < NP; ++u) {
#pragma unroll
      for (int j = 0; j < VEC; ++j) tile_max = fmaxf(tile_max, E::load(x[u].v[j]));
    }
    top_value = fmaxf(top_value, tile_max);
    // The reference: the first tile's maximum, moved when it lies too low.
    if (__ballot(ref == -INFINITY || (tile_max - ref) * c > kSlack) != 0) {
      const float to = fmaxf(fmaxf(xor_max<1, kWave>(tile_max), ref), kLowest);
      if (ref != -INFINITY) {
        float S = 0.f, N = 0.f;
        add_sums(ref, sum, ent, to, c, S, N);
        sum = S;
        ent = N;
      }
      ref = to;
    }
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      // A pack at a time, unpacked again: what the registers of the list's code
      // leave room for.
      if constexpr (TOP) {
        __builtin_amdgcn_sched_barrier(0);
        pin(x[u]);
      }
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = (E::load(x[u].v[j]) - ref) * c;
        const float p = fast_exp2(d);
        sum += p;
        if (ENT) ent = fmaf(p, fmaxf(d, -200.f), ent);  // 2^-200 is 0: 0 ln 0 = 0
      }
    }
    if constexpr (TOP) {
      // Both sums are done here: else the entropy's is put off past the branches
      // below, with every weight kept for it (76 registers, 128 and spills).
      asm volatile("" : "+v"(sum), "+v"(ent));
      // The tile's keys again, for the paths that hardly a tile takes.
      auto each_key = [&](auto&& f) {
#pragma unroll 1
        for (int u = 0; u < NP; ++u) {
          const Pack<R, VEC> y = load_tile(p0, u);
#pragma unroll
          for (int j = 0; j < VEC; ++j) f(order_key(E::load(y.v[j])));
        }
      };
      // The key of the lane's largest value in this tile, and so far.
      uint32_t tile_key = order_key(tile_max);
      if (__ballot(sum != sum) != 0) each_key([&](uint32_t k) { tile_key = max(tile_key, k); });
      lane_key = max(lane_key, tile_key);
      const bool was_first = cand.first;
      if (was_first) {
        cand.first = false;
        const uint32_t part_key = nth_value_key<E>(lane_key, quarter);
        // A wave may be alone in a short tile.
        const bool is_short = p0 + kTilePacks > pack_end;
        const uint32_t all_key = is_short ? nth_value_key<E>(lane_key, a.top) : 0;
        if (lane == 0) {
          share(s, wave, part_key);
          s.wave_first[wave] = all_key;
        }
        // Every wave of the workgroup is here, or none: an aligned row's last part
        // can be empty.
        __syncthreads();
        cand.floor = shared_floor(s);
        if (is_short) {
#pragma unroll
          for (int w = 0; w < kWaves; ++w) cand.floor = max(cand.floor, s.wave_first[w]);
          cand.floor = __builtin_amdgcn_readfirstlane(cand.floor);
        }
      }
      // Puts the tile's values of keys from `least` on behind the list; how many
      // it then has, stored or not. The lanes that have such values put their
      // packs into LDS, 32 at a time, where all lanes look through them.
      auto gather = [&](uint32_t least) -> int {
        int n = cand.count;
        if (least == 0) return n;  // above NaN: nothing
        uint64_t lanes = __ballot(tile_key >= least);
        while (lanes != 0) {
          const int rank = __popcll(lanes & ((1ull << lane) - 1));
          const bool puts = (lanes >> lane & 1) && rank < kScanLanes;
          const uint64_t put = __ballot(puts);
          if (puts) {
#pragma unroll
            for (int u = 0; u < NP; ++u)
              store_pack<R, VEC>(reinterpret_cast<R*>(s.scan[wave]) + (rank * NP + u) * VEC, x[u]);
            s.scan_lane[wave][rank] = static_cast<uint8_t>(lane);
          }
          __builtin_amdgcn_wave_barrier();
          const int values = __popcll(put) * NP * VEC;
          for (int e0 = 0; e0 < values; e0 += kWave) {
            const int e = e0 + lane;  // NP VEC is a multiple of 16, so is `values`
            bool hit = e < values;
            float v = 0.f;
            int at_v = 0;
            if (hit) {
              v = E::load(reinterpret_cast<const R*>(s.scan[wave])[e]);
              const int u = e / VEC % NP;
              const int p = p0 + u * kThreads + wave * kWave + s.scan_lane[wave][e / (NP * VEC)];
              at_v = p * VEC - lead + e % VEC;
              hit = order_key(v) >= least && p < pack_end && at_v >= 0 && at_v < a.vocab;
            }
            const uint64_t hits = __ballot(hit);
            const int at = n + __popcll(hits & ((1ull << lane) - 1));
            if (hit && at < kWaveCap) cand.list[at] = make_word(v, at_v);
            n += __popcll(hits);
          }
          __builtin_amdgcn_wave_barrier();
          lanes &= ~put;
        }
        return n;
      };
      const int before = cand.count;
      int n = gather(cand.floor + (was_first ? 0 : 1));
      for (int attempt = 1; n > kWaveCap; ++attempt) {
        if (attempt == 1 && was_first) {
          cand.open = true;  // too many values equal to the floor: leave them out
        } else if (attempt == 1) {
          cand.compress(a.top);
        } else {
          // Many large values in few lanes: the tile's own top-th largest key.
          uint32_t key = 0;
          for (int b = 31; b >= 0; --b) {
            const uint32_t trial = key | (1u << b);
            int mine = 0;
            each_key([&](uint32_t k) { mine += k >= trial; });
            if (wave_sum_int(mine) >= a.top) key = trial;
          }
          cand.reopen(key);
        }
        n = gather(cand.floor + 1);
      }
      cand.count = n;
      if (was_first) {
        cand.raised_at = n;
      } else if (n != before && n > cand.raised_at + a.top / 2) {
        if (lane == 0) share(s, wave, nth_value_key<E>(lane_key, quarter));
        // Another wave may be ahead, so its values equal to the floor may come
        // later in the row: only what is below it cannot matter.
        cand.raise(max(nth_value_key<E>(lane_key, a.top), shared_floor(s) - 1));
        cand.raised_at = n;
      }
    }
  }

  if constexpr (TOP) {
    if (cand.count > kKeptWords) cand.compress(a.top);
  }
  // The workgroup's sums, relative to its maximum (of the wave's reference
  // where every value is below it).
  const float wave_max = fmaxf(xor_max<1, kWave>(top_value), kLowest);
  {
    float S = 0.f, N = 0.f;
    add_sums(ref == -INFINITY ? kLowest : ref, group_sum<kWave>(sum), group_sum<kWave>(ent),
             wave_max, c, S, N);
    if constexpr (TOP) {
      if (t == 0) s.count = 0;
      if (lane == 0) {
        s.wave_floor[wave] = cand.floor;
        s.wave_open[wave] = cand.open;
      }
    }
    if (lane == 0) {
      s.wave_ref[wave] = wave_max;
      s.wave_sum[wave] = S;
      s.wave_ent[wave] = N;
    }
  }
  __syncthreads();
  float r = kLowest, S = 0.f, N = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) r = fmaxf(r, s.wave_ref[w]);
#pragma unroll
  for (int w = 0; w < kWaves; ++w)
    add_sums(s.wave_ref[w], s.wave_sum[w], s.wave_ent[w], r, c, S, N);
  if constexpr (TOP) {
    // What lies above the highest floor, or at it.
    uint32_t floor = 0;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) floor = max(floor, s.wave_floor[w]);
    bool open = false;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) open = open || (s.wave_open[w] && s.wave_floor[w] == floor);
    for (int i = lane; i < cand.count; i += kWave) {
      const uint64_t w = cand.list[i];
      const uint32_t key = static_cast<uint32_t>(w >> 32);
      if (key > floor || (key == floor && !open)) s.best[atomicAdd(&s.count, 1)] = w;
    }
    __syncthreads();
    if (open && s.count < a.top)
      fill_equal<E>(s, logits, v_begin, min(a.vocab, pack_end * VEC - lead), floor,
                    a.top - s.count);
    const int n = s.count;
    rank_words(s, s.best, n, a.top);
  }
  if (a.parts == 1) {
    write_row<E, TOP>(a, s, row, logits, r, temperature, S, N);
    return;
  }

  // Publish, count in; the last part of the row joins all of them.
  char* records = a.workspace + static_cast<int64_t>(row) * a.parts * a.part_bytes;
  uint64_t* mine = reinterpret_cast<uint64_t*>(records + part * a.part_bytes);
  if (t == 0) {
    store_agent(mine, __builtin_bit_cast(uint64_t, Float2{r, S}));
    store_agent(mine + 1, __builtin_bit_cast(uint64_t, Float2{N, 0.f}));
  }
  if constexpr (TOP) {
    if (t < a.top) store_agent(mine + 2 + t, s.kept[t]);
  }
  wait_stores();
  __syncthreads();
  if (t == 0)
    s.arrived = __hip_atomic_fetch_add(a.counters + row, 1, __ATOMIC_RELAXED,
                                       __HIP_MEMORY_SCOPE_AGENT);
  __syncthreads();
  if (s.arrived != a.parts - 1) return;
  if (t == 0)
    __hip_atomic_store(a.counters + row, 0, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  // A lane per part (at most 64), every wave the same sums in the same order.
  Float2 rs{kLowest, 0.f}, nn{0.f, 0.f};
  if (lane < a.parts) {
    const uint64_t* rec = reinterpret_cast<const uint64_t*>(records + lane * a.part_bytes);
    rs = __builtin_bit_cast(Float2, load_agent(rec));
    nn = __builtin_bit_cast(Float2, load_agent(rec + 1));
  }
  if constexpr (TOP) {
    auto word_of = [&](int q, int i) {
      return load_agent(reinterpret_cast<const uint64_t*>(records + q * a.part_bytes) + 2 + i);
    };
    const int words = a.parts * a.top;
    int n = words;
    if (words <= kFewWords) {
      if (t < words) s.list[t] = word_of(t / a.top, t % a.top);
    } else {
      // Every part's words are sorted, so the best 64 / parts of each are a good
      // sample: the top-th largest of those is a floor.
      const int deep = lane / a.parts;
      uint64_t probe = 0;
      if (deep < a.top) probe = word_of(lane - deep * a.parts, deep);
      // Fewer words than that in the sample: no floor but zero's, of no word.
      uint64_t floor = 1;
      if (__popcll(__ballot(probe != 0)) >= a.top) floor = nth_word<E>(probe, a.top);
      if (t == 0) s.count = 0;
      __syncthreads();
#pragma unroll 2
      for (int at = t; at < words; at += kThreads) {
        const uint64_t w = word_of(at / a.top, at % a.top);
        if (w >= floor) s.list[atomicAdd(&s.count, 1)] = w;
      }
      __syncthreads();
      n = s.count;
    }
    rank_words(s, s.list, n, a.top);
  }
  const float all = xor_max<1, kWave>(rs.x);
  S = N = 0.f;
  add_sums(rs.x, rs.y, nn.x, all, c, S, N);
  write_row<E, TOP>(a, s, row, logits, all, temperature, group_sum<kWave>(S),
               group_sum<kWave>(N));
}
static_assert(kMaxParts <= kWave, "a lane per part");
static_assert(kMaxTop * (kWaveCap / kWave) <= kKeptWords, "compressed lists fit");
static_assert(kMaxTop <= kKeptWords, "and a scan's words");

// Four workgroups a CU: 64 rows with 20 alternatives take 30.6 us with 512,
// 19.1 with 700, 19.2 with 1024, 19.5 with 2048.
constexpr int kWantParts = 1024;
// A part less where rounding up ends past five a CU, some of which would start
// when others end: 1000 rows with 20 alternatives 91.6 us with two parts, 81.3
// with one; 900 of 65536 values with 5 43.1, 33.5; 700 rows 68.1, 69.2. 300
// rows keep four parts, 1200 workgroups: 38.7, 40.9 with three.
constexpr int kMostGroups = 1280;

// Packs of a part of a row, a whole number of tiles: about kWantParts
// workgroups in all, at most kMaxParts in a row. From the sizes alone, so a
// workspace fits every call; every alignment of a row fits.
struct RowSplit {
  int32_t parts, part_packs;
};
RowSplit split_row(int32_t rows, int32_t vocab, int32_t dtype) {
  const int vec = dtype == MI_DTYPE_F32 ? 4 : 8;
  const int64_t packs = (static_cast<int64_t>(vocab) + 2 * vec - 2) / vec;
  const int64_t tile = kThreads * kTilePasses;
  const int64_t tiles = (packs + tile - 1) / tile;
  int64_t want = (kWantParts + int64_t(rows) - 1) / rows;
  if (want > 1 && want * rows > kMostGroups) --want;
  want = std::min<int64_t>(want, kMaxParts);
  const int64_t each = (tiles + want - 1) / want;
  return {static_cast<int32_t>((tiles + each - 1) / each), static_cast<int32_t>(each * tile)};
}

constexpr int kPartBytes = 16;  // (maximum, S), (E, -); then the words

template <typename E, bool TOP, bool ENT>
int32_t launch_logprobs(const LogprobArgs& a, int32_t rows, hipStream_t stream) {
  const uint32_t blocks = static_cast<uint32_t>(rows) * static_cast<uint32_t>(a.parts);
  logprob_kernel<E, TOP, ENT><<<blocks, kThreads, 0, stream>>>(a);
  return check_launch("mi_token_logprobs");
}

template <typename E>
int32_t dispatch_logprobs(const LogprobArgs& a, int32_t rows, hipStream_t stream) {
  if (a.top > 0)
    return a.entropy != nullptr ? launch_logprobs<E, true, true>(a, rows, stream)
                                : launch_logprobs<E, true, false>(a, rows, stream);
  return a.entropy != nullptr ? launch_logprobs<E, false, true>(a, rows, stream)
                              : launch_logprobs<E, false, false>(a, rows, stream);
}

}  // namespace
}  // namespace mi

extern "C" int64_t mi_token_logprobs_workspace_bytes(int32_t num_rows, int32_t vocab_size,
                                                     int32_t num_top, int32_t dtype) {
  using namespace mi;
  if (num_rows <= 0 || vocab_size <= 0 || num_top < 0 || !valid_dtype(dtype)) return 0;
  const int32_t parts = split_row(num_rows, vocab_size, dtype).parts;
  return parts == 1 ? 0
                    : static_cast<int64_t>(num_rows) * parts * (kPartBytes + 8 * int64_t(num_top));
}

extern "C" int32_t mi_token_logprobs(const void* logits, int64_t row_stride, int32_t num_rows,
                                     int32_t vocab_size, int32_t dtype,
                                     const float* temperatures, const int64_t* tokens,
                                     int64_t token_stride, int32_t num_given, float* logprobs,
                                     float* entropy, int64_t* top_tokens, float* top_logprobs,
                                     int32_t num_top, void* workspace, int64_t workspace_bytes,
                                     int32_t* counters, void* stream) {
  using namespace mi;
  clear_error();
  if (!valid_dtype(dtype)) return fail(MI_ERR_INVALID_ARGUMENT, "mi_token_logprobs: bad dtype");
  if (num_rows < 0 || vocab_size <= 0 || num_given < 0 || num_top < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_token_logprobs: invalid sizes");
  if (num_top > kMaxTop || num_top > vocab_size)
    return fail(MI_ERR_INVALID_ARGUMENT,
                "mi_token_logprobs: num_top is at most 32 and at most vocab_size");
  if (vocab_size > (1 << 30) || num_given > 65536)
    return fail(MI_ERR_UNSUPPORTED, "mi_token_logprobs: vocab_size above 2^30 or num_given "
                                    "above 65536");
  if (num_rows == 0) return MI_OK;
  if (!logits || (num_given > 0 && (!tokens || !logprobs)) ||
      (num_top > 0 && (!top_tokens || !top_logprobs)))
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_token_logprobs: null pointer");
  if (num_rows > 1 && (row_stride < vocab_size || (num_given > 0 && token_stride < num_given)))
    return fail(MI_ERR_INVALID_ARGUMENT,
                "mi_token_logprobs: row_stride must be >= vocab_size, token_stride >= num_given");
  const auto off = [](const void* p, uint64_t bytes) {
    return reinterpret_cast<uintptr_t>(p) % bytes != 0;
  };
  if (off(logits, dtype_size(dtype)) || off(temperatures, 4) || off(tokens, 8) ||
      off(logprobs, 4) || off(entropy, 4) || off(top_tokens, 8) || off(top_logprobs, 4))
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_token_logprobs: misaligned pointer");
  const int64_t need = mi_token_logprobs_workspace_bytes(num_rows, vocab_size, num_top, dtype);
  if (need > 0 && (!workspace || off(workspace, 16) || workspace_bytes < need))
    return fail(MI_ERR_WORKSPACE,
                "mi_token_logprobs: workspace must be 16-byte aligned and at least "
                "mi_token_logprobs_workspace_bytes() long");
  if (need > 0 && (!counters || off(counters, 4)))
    return fail(MI_ERR_WORKSPACE, "mi_token_logprobs: counters (num_rows zeros) are missing");
  if (static_cast<int64_t>(num_rows) * split_row(num_rows, vocab_size, dtype).parts >
      0xffffffffll / kThreads)
    return fail(MI_ERR_UNSUPPORTED, "mi_token_logprobs: too many rows for one launch");
  LogprobArgs a;
  a.logits = logits;
  a.row_stride = num_rows > 1 ? row_stride : 0;
  a.vocab = vocab_size;
  const RowSplit split = split_row(num_rows, vocab_size, dtype);
  a.parts = split.parts;
  a.part_packs = split.part_packs;
  a.temperatures = temperatures;
  a.tokens = tokens;
  a.token_stride = token_stride;
  a.given = num_given;
  a.logprobs = logprobs;
  a.entropy = entropy;
  a.top_tokens = top_tokens;
  a.top_logprobs = top_logprobs;
  a.top = num_top;
  a.workspace = static_cast<char*>(workspace);
  a.part_bytes = kPartBytes + 8 * num_top;
  a.counters = counters;
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (dtype == MI_DTYPE_BF16) return dispatch_logprobs<BF16>(a, num_rows, s);
  if (dtype == MI_DTYPE_F16) return dispatch_logprobs<F16>(a, num_rows, s);
  return dispatch_logprobs<F32>(a, num_rows, s);
}
