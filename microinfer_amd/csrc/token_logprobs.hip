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
// 64-bit words (order key of the value, then the lower index). After its first
// tile a wave knows the num_top-th largest of its 64 lanes' maxima: at least
// num_top values are no smaller than that threshold, so only values above it
// can matter and go to a small list in LDS, and values equal to it fill up
// from the lowest index if the list is short. That fill-up is what rows of
// equal or masked values run on; NaN, infinities and lists that overflow take
// num_top rounds of a maximum over the tile instead.
//
// Few rows are split over many workgroups: each publishes (maximum, S, E) and
// its own best words, and the last to arrive at the row's counter joins them.
//
// Bound by memory for many rows (about ten operations an element, one of them
// an exp2 at a quarter of the rate), by latency for few.
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

// Unsigned order of float values: NaN above everything, -0 equal to +0.
__device__ __forceinline__ uint32_t order_key(float v) {
  uint32_t b = __float_as_uint(v);
  if (v != v) return 0xffffffffu;
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

__device__ __forceinline__ uint64_t shfl_xor_word(uint64_t v, int mask) {
  const uint32_t lo = __shfl_xor(static_cast<uint32_t>(v), mask, kWave);
  const uint32_t hi = __shfl_xor(static_cast<uint32_t>(v >> 32), mask, kWave);
  return (static_cast<uint64_t>(hi) << 32) | lo;
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

// Bits of a float32 that can differ between values of the type.
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

struct Shared {
  uint64_t list[kListCap];
  uint64_t kept[kMaxTop];  // select()'s result, largest first
  uint64_t wave_word[kWaves];
  uint32_t wave_key[kWaves];
  float wave_ref[kWaves], wave_sum[kWaves], wave_ent[kWaves];
  int32_t count;  // words in the list
  int32_t bad;    // a sum is NaN
  int32_t fill[kWaves];
  int32_t arrived;
};

// The `top` largest of list[0, n) into kept[0, top), largest first, zeros
// behind them. All threads; the list is spoilt.
__device__ void select_words(Shared& s, int n, int top) {
  const int t = threadIdx.x;
  const int lane = t % kWave, wave = t / kWave;
  __syncthreads();
  uint64_t mine[kListCap / kThreads];
  uint64_t best = 0;
#pragma unroll
  for (int i = 0; i < kListCap / kThreads; ++i) {
    const int at = i * kThreads + t;
    mine[i] = at < n ? s.list[at] : 0;
    best = mine[i] > best ? mine[i] : best;
  }
  if (t < top) s.kept[t] = 0;
  uint32_t hi = 0, lo = 0;
  if (n > kWave) {
    // A word that at least `top` words are no smaller than: the top-th largest
    // of a wave's lanes' maxima, the best wave's.
    hi = nth_key<32>(static_cast<uint32_t>(best >> 32), top);
    const uint32_t above = static_cast<uint32_t>(best >> 32);
    const int more = __popcll(__ballot(above > hi));
    lo = nth_key<32>(above == hi ? static_cast<uint32_t>(best) : 0, top - more);
  }
  const uint64_t floor_word = (static_cast<uint64_t>(hi) << 32) | lo;
  if (lane == 0) s.wave_word[wave] = floor_word;
  if (t == 0) s.count = 0;
  __syncthreads();
  uint64_t least = 1;  // zeros are no words
#pragma unroll
  for (int w = 0; w < kWaves; ++w) least = s.wave_word[w] > least ? s.wave_word[w] : least;
#pragma unroll
  for (int i = 0; i < kListCap / kThreads; ++i)
    if (mine[i] >= least) s.list[atomicAdd(&s.count, 1)] = mine[i];
  __syncthreads();
  // Each word's rank is the number of larger ones; words are distinct.
  const int m = s.count;
  for (int at = t; at < m; at += kThreads) {
    const uint64_t w = s.list[at];
    int rank = 0;
    for (int j = 0; j < m && rank < top; ++j) rank += s.list[j] > w;
    if (rank < top) s.kept[rank] = w;
  }
  __syncthreads();
}

// Appends the first `want` indices of [lo, hi) whose value has key `key` to the
// list. All threads.
template <typename E>
__device__ void fill_equal(Shared& s, const typename E::raw* row, int lo, int hi, uint32_t key,
                           int want) {
  const int t = threadIdx.x;
  const int lane = t % kWave, wave = t / kWave;
  int found = 0;
  const int start = s.count;
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
    if (hit && before < want) s.list[start + before] = make_word(key_value(key), v);
    found = all;
    __syncthreads();
  }
  if (t == 0) s.count = start + min(found, want);
  __syncthreads();
}

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
template <typename E>
__device__ void write_row(const LogprobArgs& a, const Shared& s, int row,
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
  if (threadIdx.x < a.top) {
    const uint64_t w = s.kept[threadIdx.x];
    const int64_t at = static_cast<int64_t>(row) * a.top + threadIdx.x;
    a.top_tokens[at] = word_index(w);
    a.top_logprobs[at] = logprob(key_value(static_cast<uint32_t>(w >> 32)));
  }
}

// NP packs of VEC elements per thread make a tile.
template <typename E, int NP, bool TOP, bool ENT>
__global__ __launch_bounds__(kThreads) void logprob_kernel(const LogprobArgs a) {
  using R = typename E::raw;
  constexpr int VEC = 16 / sizeof(R);
  constexpr int kTilePacks = kThreads * NP;
  __shared__ Shared s;
  const int row = blockIdx.x / a.parts;
  const int part = blockIdx.x - row * a.parts;
  const int t = threadIdx.x;
  const int lane = t % kWave;
  const int wave = __builtin_amdgcn_readfirstlane(t / kWave);
  const R* logits = static_cast<const R*>(a.logits) + row * a.row_stride;
  float temperature = a.temperatures == nullptr ? 1.f : a.temperatures[row];
  if (!(temperature > 0.f && temperature < INFINITY)) temperature = NAN;
  const float c = kLog2E / temperature;
  // Packs lie on the 16-byte grid; the row's first and last may be partial.
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(logits) & 15u) / sizeof(R));
  const R* grid = logits - lead;
  const int pack_begin = part * a.part_packs;
  const int pack_end = min((lead + a.vocab + VEC - 1) / VEC, pack_begin + a.part_packs);
  const int v_begin = max(0, pack_begin * VEC - lead);

  if (TOP && t == 0) {
    s.count = 0;
    s.bad = 0;
  }
  float ref = -INFINITY;   // wave-uniform reference of the sums; -inf: none yet
  float sum = 0.f, ent = 0.f, top_value = -INFINITY;
  bool first = true;       // no threshold yet
  bool complete = false;   // the list holds every value seen
  uint32_t floor_key = 0;  // values of larger keys are in the list
  float floor_value = -INFINITY;

  for (int p0 = pack_begin; p0 < pack_end; p0 += kTilePacks) {
    Pack<R, VEC> x[NP];
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      const int p = p0 + u * kThreads + t;
      const int v0 = p * VEC - lead;
      if (p < pack_end && v0 >= 0 && v0 + VEC <= a.vocab) {
        x[u] = load_pack<R, VEC>(grid + static_cast<int64_t>(p) * VEC);
      } else {
#pragma unroll
        for (int j = 0; j < VEC; ++j) {
          x[u].v[j] = E::store(-INFINITY);
          if (p < pack_end && v0 + j >= 0 && v0 + j < a.vocab) x[u].v[j] = logits[v0 + j];
        }
      }
    }
    float pack_max[NP];
    float tile_max = -INFINITY;
#pragma unroll
    for (int u = 0; u < NP; ++u) {
      pack_max[u] = E::load(x[u].v[0]);
#pragma unroll
      for (int j = 1; j < VEC; ++j) pack_max[u] = fmaxf(pack_max[u], E::load(x[u].v[j]));
      tile_max = fmaxf(tile_max, pack_max[u]);
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
#pragma unroll
      for (int j = 0; j < VEC; ++j) {
        const float d = (E::load(x[u].v[j]) - ref) * c;
        const float p = fast_exp2(d);
        sum += p;
        if (ENT) ent = fmaf(p, fmaxf(d, -200.f), ent);  // 2^-200 is 0: 0 ln 0 = 0
      }
    }
    if constexpr (TOP) {
      const int before = first ? 0 : s.count;
      if (first) {
        constexpr int kBits = KeyBits<E>::value;
        uint32_t key = nth_key<kBits>(order_key(tile_max), a.top);
        if (!(key & 0x80000000u)) key |= (kBits == 32 ? 0u : 0xffffffffu >> kBits);
        if (lane == 0) s.wave_key[wave] = key;
      }
      if (sum != sum) s.bad = 1;
      __syncthreads();
      if (first) {
#pragma unroll
        for (int w = 0; w < kWaves; ++w) floor_key = max(floor_key, s.wave_key[w]);
        floor_key = max(floor_key, order_key(-INFINITY));
        floor_value = key_value(floor_key);
      }
      const bool was_first = first;
      first = false;
      const bool bad = s.bad != 0;
      if (!bad) {
#pragma unroll
        for (int u = 0; u < NP; ++u) {
          if (pack_max[u] > floor_value) {
            const int v0 = (p0 + u * kThreads + t) * VEC - lead;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const float v = E::load(x[u].v[j]);
              if (v > floor_value) {
                const int at = atomicAdd(&s.count, 1);
                if (at < kListCap) s.list[at] = make_word(v, v0 + j);
              }
            }
          }
        }
      }
      __syncthreads();
      const int n = s.count;
      __syncthreads();
      if (bad || n > kListCap) {
        // Rounds: the tile's best words one after the other.
        if (t == 0) s.count = before;
        __syncthreads();
        // First what the tiles before hold of values equal to the threshold.
        if (!was_first && !complete && before < a.top)
          fill_equal<E>(s, logits, v_begin, max(v_begin, p0 * VEC - lead), floor_key,
                        a.top - before);
        select_words(s, s.count, a.top);
        if (t < a.top) s.list[t] = s.kept[t];
        uint64_t last = ~0ull;
        for (int i = 0; i < a.top; ++i) {
          uint64_t best = 0;
#pragma unroll
          for (int u = 0; u < NP; ++u) {
            const int p = p0 + u * kThreads + t;
            const int v0 = p * VEC - lead;
#pragma unroll
            for (int j = 0; j < VEC; ++j) {
              const int v = v0 + j;
              if (p < pack_end && v >= 0 && v < a.vocab) {
                const uint64_t w = make_word(E::load(x[u].v[j]), v);
                if (w < last && w > best) best = w;
              }
            }
          }
#pragma unroll
          for (int o = 1; o < kWave; o <<= 1) {
            const uint64_t other = shfl_xor_word(best, o);
            best = other > best ? other : best;
          }
          __syncthreads();
          if (lane == 0) s.wave_word[wave] = best;
          __syncthreads();
#pragma unroll
          for (int w = 0; w < kWaves; ++w) best = s.wave_word[w] > best ? s.wave_word[w] : best;
          if (t == 0) s.list[a.top + i] = best;
          if (best == 0) {
            for (int k = i + t; k < a.top; k += kThreads) s.list[a.top + k] = 0;
            break;
          }
          last = best;
        }
        select_words(s, 2 * a.top, a.top);
        if (t < a.top) s.list[t] = s.kept[t];
        complete = s.kept[a.top - 1] == 0;  // fewer values than alternatives so far
        __syncthreads();
        if (t == 0) s.count = complete ? 0 : a.top;
        if (complete) {
          // Only the row's last tile can leave it so.
          if (t < a.top && s.kept[t] != 0) atomicAdd(&s.count, 1);
        } else {
          floor_key = static_cast<uint32_t>(s.kept[a.top - 1] >> 32);
          floor_value = key_value(floor_key);
        }
        __syncthreads();
      } else if (n > kListCap / 2) {
        select_words(s, n, a.top);
        if (t < a.top) s.list[t] = s.kept[t];
        if (t == 0) s.count = a.top;
        floor_key = static_cast<uint32_t>(s.kept[a.top - 1] >> 32);
        floor_value = key_value(floor_key);
        __syncthreads();
      }
    }
  }

  // The workgroup's sums, relative to its maximum (of the wave's reference
  // where every value is below it).
  const float wave_max = fmaxf(xor_max<1, kWave>(top_value), kLowest);
  {
    float S = 0.f, N = 0.f;
    add_sums(ref == -INFINITY ? kLowest : ref, group_sum<kWave>(sum), group_sum<kWave>(ent),
             wave_max, c, S, N);
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
    if (!complete && s.count < a.top) {
      const int v_end = min(a.vocab, pack_end * VEC - lead);
      fill_equal<E>(s, logits, v_begin, v_end, floor_key, a.top - s.count);
    }
    select_words(s, s.count, a.top);
  }
  if (a.parts == 1) {
    write_row<E>(a, s, row, logits, r, temperature, S, N);
    return;
  }

  // Publish, count in; the last part of the row joins all of them.
  char* records = a.workspace + static_cast<int64_t>(row) * a.parts * a.part_bytes;
  uint64_t* mine = reinterpret_cast<uint64_t*>(records + part * a.part_bytes);
  if (t == 0) {
    store_agent(mine, __builtin_bit_cast(uint64_t, Float2{r, S}));
    store_agent(mine + 1, __builtin_bit_cast(uint64_t, Float2{N, 0.f}));
  }
  if (TOP && t < a.top) store_agent(mine + 2 + t, s.kept[t]);
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
    for (int i = t; i < a.parts * a.top; i += kThreads) {
      const int q = i / a.top;
      s.list[i] = load_agent(
          reinterpret_cast<const uint64_t*>(records + q * a.part_bytes) + 2 + (i - q * a.top));
    }
    select_words(s, a.parts * a.top, a.top);
  }
  const float all = xor_max<1, kWave>(rs.x);
  S = N = 0.f;
  add_sums(rs.x, rs.y, nn.x, all, c, S, N);
  write_row<E>(a, s, row, logits, all, temperature, group_sum<kWave>(S),
               group_sum<kWave>(N));
}
static_assert(kMaxParts <= kWave, "a lane per part");

// Parts of a row: enough workgroups to fill the chip twice, each of at least
// kMinPartPacks packs. From the sizes alone, so a workspace fits every call.
constexpr int kMinPartPacks = 512;
int32_t row_parts(int32_t rows, int32_t vocab, int32_t dtype) {
  const int vec = dtype == MI_DTYPE_F32 ? 4 : 8;
  const int64_t packs = (static_cast<int64_t>(vocab) + 2 * vec - 2) / vec;
  const int64_t want = (512 + rows - 1) / rows;
  const int64_t most = std::max<int64_t>(1, packs / kMinPartPacks);
  return static_cast<int32_t>(std::min<int64_t>(std::min<int64_t>(want, most), kMaxParts));
}

constexpr int kPartBytes = 16;  // (maximum, S), (E, -); then the words

template <typename E, bool TOP, bool ENT>
int32_t launch_logprobs(const LogprobArgs& a, int32_t rows, hipStream_t stream) {
  const uint32_t blocks = static_cast<uint32_t>(rows) * static_cast<uint32_t>(a.parts);
  logprob_kernel<E, 4, TOP, ENT><<<blocks, kThreads, 0, stream>>>(a);
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
  const int32_t parts = row_parts(num_rows, vocab_size, dtype);
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
  if (static_cast<int64_t>(num_rows) * row_parts(num_rows, vocab_size, dtype) >
      0xffffffffll / kThreads)
    return fail(MI_ERR_UNSUPPORTED, "mi_token_logprobs: too many rows for one launch");
  LogprobArgs a;
  a.logits = logits;
  a.row_stride = num_rows > 1 ? row_stride : 0;
  a.vocab = vocab_size;
  a.parts = row_parts(num_rows, vocab_size, dtype);
  const int vec = dtype == MI_DTYPE_F32 ? 4 : 8;
  // Every alignment of a row fits: the most packs that it can touch.
  const int packs = (vocab_size + 2 * vec - 2) / vec;
  a.part_packs = (packs + a.parts - 1) / a.parts;
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
