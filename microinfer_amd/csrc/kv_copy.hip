// Copies of cache pages within a K/V pool, all layers in one launch: forked
// sequences' partial pages, beams that change parents, compaction.
//
// A parallel assignment K[dst_i] = K'[src_i] (K' the pool before the call).
// The pairs come from the host's block manager, so they are ordered there:
// a pair whose destination nobody else reads is independent of the rest and
// runs anywhere; the others form groups that one thread per 16-byte word
// walks in an order in which every block is read before it is overwritten (a
// chain from its end, a cycle with its first word kept in registers). Only
// words at the same place of a page depend on each other, so no thread waits
// for another. The lists travel in the kernel's arguments: no upload and
// nothing to keep alive.
//
// Bound by memory: every row is read and written once. 1000 pages of 16 tokens
// x 28 layers x 8 heads (3.7 GB) take 706 us, 5.2 TB/s read and written, where a
// large copy reaches 4.7; one partial page 2.5 us, an empty launch's time;
// 64 of them from 8 parents (87 MB) 15.3 us, 5.7 TB/s as the parents' rows are
// read from the caches. Dependent pairs: a swap 4.1 us, 100 swaps 137 and a chain
// of 100 pages 70 (5.3 TB/s), a chain of 1000 886 and a cycle of 255 226 (4.1: a
// thread per word walks them, page after page). Stores go past the caches: 10.7 us
// for one page and loads that wait for each other, 2.5 so.
#include <algorithm>
#include <new>
#include <utility>
#include <vector>

#include "mi_common.h"
#include "mi_fork.h"

namespace mi {
namespace {

// The rows of a page as three nested dimensions, fastest first: tokens, KV
// heads and K/V in the order of their strides, so that neighbouring lanes
// touch neighbouring memory in every layout.
struct PageShape {
  int64_t stride[3];  // bytes
  uint32_t size[3];
  int32_t token_dim;  // which of the three counts tokens
  uint32_t words_per_row;
  uint32_t words_per_token;  // all heads, K and V
  int64_t layer_stride, block_stride;  // bytes
};

struct CopyOp {
  int32_t src, dst, tokens;
};

// 3.6 KB of the 4 KB that a launch's arguments may take.
constexpr int kMaxOps = 256;
struct CopyList {
  CopyOp op[kMaxOps];
};
constexpr int64_t kMaxGroupBlocks = 1 << 23;
// Groups of dependent copies: group g is ops [start[g], start[g + 1]). dst = -1
// keeps the source's word, src = -1 writes the kept word.
struct GroupList {
  CopyOp op[kMaxOps];
  uint16_t start[kMaxOps + 1];
};

typedef uint32_t Words4 __attribute__((ext_vector_type(4)));

constexpr int kCopyThreads = 256;
// Words in flight per thread: 1, 8 and 64 forked pages of 28 layers 2.5, 3.4 and
// 15.3 us with two, 2.7, 3.5 and 16.0 with four, 3.2, 4.2 and 16.3 with eight.
constexpr int kCopyUnroll = 2;
// More bytes than the last-level cache holds: nothing read stays in it, so
// reading past it costs nothing and leaves it to others (1000 pages of 28
// layers 706 us, 721 without). Fewer may lie in it, as forked pages do, which
// were just written (64 of them 16 us, 30 past it).
constexpr int64_t kStreamBytes = int64_t(1) << 28;

// Byte offset of word w among the words of a page's first `tokens` rows, and
// its token row.
__device__ __forceinline__ int64_t word_offset(const PageShape& p, uint32_t tokens, uint32_t w,
                                               int word_bytes, uint32_t* token) {
  const uint32_t size0 = p.token_dim == 0 ? tokens : p.size[0];
  const uint32_t size1 = p.token_dim == 1 ? tokens : p.size[1];
  const uint32_t row = w / p.words_per_row;
  const uint32_t col = w - row * p.words_per_row;
  const uint32_t r1 = row / size0;
  const uint32_t i0 = row - r1 * size0;
  const uint32_t i2 = r1 / size1;
  const uint32_t i1 = r1 - i2 * size1;
  *token = p.token_dim == 0 ? i0 : p.token_dim == 1 ? i1 : i2;
  return i0 * p.stride[0] + i1 * p.stride[1] + i2 * p.stride[2] +
         static_cast<int64_t>(col) * word_bytes;
}

// One slice of one pair's rows in one layer: a workgroup. All of a thread's
// loads are issued before its first store (words past the end load the page's
// first), and the stores are not kept in the caches, where nobody reads them
// before the next step: they would push out what is read.
template <typename W, bool STREAM>
__global__ __launch_bounds__(kCopyThreads) void kv_copy_kernel(char* base, const PageShape p,
                                                              const CopyList list) {
  const CopyOp op = list.op[blockIdx.y];
  const uint32_t words = p.words_per_token * op.tokens;
  const uint32_t first = blockIdx.x * (kCopyThreads * kCopyUnroll);
  if (first >= words) return;
  char* layer = base + blockIdx.z * p.layer_stride;
  const char* from = layer + op.src * p.block_stride;
  char* to = layer + op.dst * p.block_stride;
  W v[kCopyUnroll];
  int64_t off[kCopyUnroll];
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u) {
    const uint32_t w = first + u * kCopyThreads + threadIdx.x;
    uint32_t token;
    off[u] = word_offset(p, op.tokens, w < words ? w : 0, sizeof(W), &token);
    const W* at = reinterpret_cast<const W*>(from + off[u]);
    v[u] = STREAM ? __builtin_nontemporal_load(at) : *at;
  }
#pragma unroll
  for (int u = 0; u < kCopyUnroll; ++u)
    if (first + u * kCopyThreads + threadIdx.x < words)
      __builtin_nontemporal_store(v[u], reinterpret_cast<W*>(to + off[u]));
}

// Dependent copies: a thread per word of the page walks its group's ops.
template <typename W>
__global__ __launch_bounds__(kCopyThreads) void kv_copy_group_kernel(char* base,
                                                                    const PageShape p,
                                                                    const GroupList list,
                                                                    int slices) {
  const int group = blockIdx.x / slices;
  const uint32_t w = (blockIdx.x - group * slices) * kCopyThreads + threadIdx.x;
  if (w >= p.words_per_token * p.size[p.token_dim]) return;
  uint32_t token;
  char* at = base + blockIdx.y * p.layer_stride +
             word_offset(p, p.size[p.token_dim], w, sizeof(W), &token);
  W kept{};
  for (int i = list.start[group]; i < list.start[group + 1]; ++i) {
    const CopyOp op = list.op[i];
    if (token >= static_cast<uint32_t>(op.tokens)) continue;
    W v = kept;
    if (op.src >= 0) v = *reinterpret_cast<const W*>(at + op.src * p.block_stride);
    if (op.dst >= 0)
      *reinterpret_cast<W*>(at + op.dst * p.block_stride) = v;
    else
      kept = v;
  }
}

// The pairs in launch order: independent ones, and groups of dependent ones.
struct Order {
  std::vector<CopyOp> single;
  std::vector<std::vector<CopyOp>> groups;  // in order; a cycle's ops are its last
  std::vector<size_t> whole_from;           // per group: ops from here on share a launch
};

// Which op writes a block: a table of the pool's blocks, or for few pairs the
// sorted destinations. A table takes 24 ns per 1000 blocks to clear, sorting
// and finding 35 ns a pair: calls of 1 and 500 pairs in a pool of 150000 blocks
// 11.0 and 21.6 us with a table, 7.5 and 34.4 without.
class Writers {
 public:
  Writers(const int32_t* dst, int32_t num_pairs, int32_t num_blocks) {
    if (num_pairs < num_blocks / 1024) {
      sorted_.reserve(num_pairs);
      for (int32_t i = 0; i < num_pairs; ++i) sorted_.push_back({dst[i], 0});
      std::sort(sorted_.begin(), sorted_.end());
    } else {
      table_.assign(num_blocks, 0);
    }
  }
  // Of block b: 1 + the index of the op that writes it, -1 if its pair needs no
  // op, 0 if no pair writes it.
  int32_t operator[](int32_t b) {
    const int32_t* at = find(b);
    return at == nullptr ? 0 : *at;
  }
  void set(int32_t b, int32_t value) { *find(b) = value; }

 private:
  int32_t* find(int32_t b) {
    if (!table_.empty()) return &table_[b];
    const auto it = std::lower_bound(sorted_.begin(), sorted_.end(), std::make_pair(b, INT32_MIN));
    return it != sorted_.end() && it->first == b ? &it->second : nullptr;
  }
  std::vector<int32_t> table_;
  std::vector<std::pair<int32_t, int32_t>> sorted_;
};

// Orders `ops` (distinct destinations, src != dst).
void order_pairs(const std::vector<CopyOp>& ops, Writers& into, Order* out) {
  const int n = static_cast<int>(ops.size());
  // readers[i]: how many ops still to run read the block that op i writes.
  std::vector<int32_t> readers(n, 0), group(n);
  for (int i = 0; i < n; ++i) group[i] = i;
  auto root = [&](int i) {
    while (group[i] != i) i = group[i] = group[group[i]];
    return i;
  };
  for (int i = 0; i < n; ++i) {
    const int writer = into[ops[i].src] - 1;
    if (writer < 0) continue;
    ++readers[writer];
    group[root(i)] = root(writer);
  }
  std::vector<int32_t> members(n, 0), place(n, -1);
  for (int i = 0; i < n; ++i) ++members[root(i)];
  auto put = [&](const CopyOp& op, int i) {
    const int r = root(i);
    if (place[r] < 0) {
      place[r] = static_cast<int32_t>(out->groups.size());
      out->groups.emplace_back();
      out->whole_from.push_back(SIZE_MAX);
    }
    out->groups[place[r]].push_back(op);
  };
  std::vector<int32_t> ready;
  std::vector<char> done(n, 0);
  for (int i = 0; i < n; ++i)
    if (readers[i] == 0) ready.push_back(i);
  for (size_t at = 0; at < ready.size(); ++at) {
    const int i = ready[at];
    done[i] = 1;
    if (members[root(i)] == 1)
      out->single.push_back(ops[i]);
    else
      put(ops[i], i);
    const int writer = into[ops[i].src] - 1;
    if (writer >= 0 && --readers[writer] == 0) ready.push_back(writer);
  }
  // What is left are cycles, whose other readers have run: keep the block
  // that op i writes, copy into it from behind until its reader is reached.
  for (int i = 0; i < n; ++i) {
    if (done[i]) continue;
    put(CopyOp{ops[i].dst, -1, INT32_MAX}, i);
    out->whole_from[place[root(i)]] = out->groups[place[root(i)]].size() - 1;
    for (int j = i; !done[j]; j = into[ops[j].src] - 1) {
      done[j] = 1;
      CopyOp op = ops[j];
      if (op.src == ops[i].dst) op.src = -1;
      put(op, j);
    }
  }
}

template <typename W>
int32_t launch_copies(char* base, const PageShape& shape, int32_t row_bytes, int32_t layers,
                      const Order& order, hipStream_t stream) {
  PageShape p = shape;
  p.words_per_row = row_bytes / sizeof(W);
  p.words_per_token = p.words_per_row;
  for (int i = 0; i < 3; ++i)
    if (i != p.token_dim) p.words_per_token *= p.size[i];
  const uint32_t page_words = p.words_per_token * p.size[p.token_dim];
  const uint32_t per = kCopyThreads * kCopyUnroll;
  int64_t tokens = 0;
  for (const CopyOp& op : order.single) tokens += op.tokens;
  const bool stream_reads = tokens * p.words_per_token * layers > kStreamBytes / int64_t(sizeof(W));
  for (size_t i = 0; i < order.single.size(); i += kMaxOps) {
    const int n = static_cast<int>(std::min<size_t>(kMaxOps, order.single.size() - i));
    CopyList list;
    std::copy_n(order.single.begin() + i, n, list.op);
    int32_t most = 0;
    for (int k = 0; k < n; ++k) most = std::max(most, list.op[k].tokens);
    const uint32_t slices = (p.words_per_token * most + per - 1) / per;
    const dim3 grid(slices, n, layers);
    if (stream_reads)
      kv_copy_kernel<W, true><<<grid, kCopyThreads, 0, stream>>>(base, p, list);
    else
      kv_copy_kernel<W, false><<<grid, kCopyThreads, 0, stream>>>(base, p, list);
    const int32_t status = check_launch("mi_kv_copy_blocks");
    if (status != MI_OK) return status;
  }
  const uint32_t thin = (page_words + kCopyThreads - 1) / kCopyThreads;
  GroupList list;
  int ops = 0, groups = 0;
  auto flush = [&]() {
    if (ops == 0) return static_cast<int32_t>(MI_OK);
    if (list.start[groups] != ops) list.start[++groups] = static_cast<uint16_t>(ops);
    kv_copy_group_kernel<W><<<dim3(groups * thin, layers), kCopyThreads, 0, stream>>>(base, p,
                                                                                    list, thin);
    ops = groups = 0;
    return check_launch("mi_kv_copy_blocks");
  };
  list.start[0] = 0;
  for (size_t g = 0; g < order.groups.size(); ++g) {
    const std::vector<CopyOp>& all = order.groups[g];
    for (size_t i = 0; i < all.size();) {
      // A cycle goes whole; other ops one by one, in order over the launches.
      const size_t take = i == order.whole_from[g] ? all.size() - i : 1;
      // A launch's threads are counted in 32 bits.
      if (ops + take > static_cast<size_t>(kMaxOps) ||
          (groups + 1) * static_cast<int64_t>(thin) > kMaxGroupBlocks) {
        const int32_t status = flush();
        if (status != MI_OK) return status;
      }
      for (size_t k = 0; k < take; ++k) list.op[ops++] = all[i++];
    }
    list.start[++groups] = static_cast<uint16_t>(ops);
  }
  return flush();
}

int32_t copy_blocks(char* keys, char* values, int64_t layer_stride, int64_t block_stride,
                    int64_t token_stride, int64_t head_stride, const int32_t* src,
                    const int32_t* dst, const int32_t* tokens, int32_t num_pairs,
                    int32_t num_layers, int32_t num_kv_heads, int32_t row_bytes,
                    int32_t block_size, int32_t num_blocks, hipStream_t stream) {
  std::vector<CopyOp> ops;
  ops.reserve(num_pairs);
  for (int32_t i = 0; i < num_pairs; ++i)
    if (src[i] < 0 || src[i] >= num_blocks || dst[i] < 0 || dst[i] >= num_blocks)
      return fail(MI_ERR_INVALID_ARGUMENT, "mi_kv_copy_blocks: block id outside the pool");
  Writers into(dst, num_pairs, num_blocks);
  for (int32_t i = 0; i < num_pairs; ++i) {
    const int32_t n = tokens == nullptr ? block_size : tokens[i];
    if (n < 0 || n > block_size)
      return fail(MI_ERR_INVALID_ARGUMENT, "mi_kv_copy_blocks: tokens outside the block");
    if (into[dst[i]] != 0)
      return fail(MI_ERR_INVALID_ARGUMENT, "mi_kv_copy_blocks: a block is written twice");
    const bool copies = n > 0 && src[i] != dst[i];
    if (copies) ops.push_back(CopyOp{src[i], dst[i], n});
    into.set(dst[i], copies ? static_cast<int32_t>(ops.size()) : -1);
  }
  if (ops.empty()) return MI_OK;
  Order order;
  bool free_order = true;
  for (const CopyOp& op : ops) free_order = free_order && into[op.src] <= 0;
  if (free_order)
    order.single.swap(ops);
  else
    order_pairs(ops, into, &order);
  for (size_t g = 0; g < order.groups.size(); ++g)
    if (order.whole_from[g] != SIZE_MAX &&
        order.groups[g].size() - order.whole_from[g] > static_cast<size_t>(kMaxOps))
      return fail(MI_ERR_UNSUPPORTED, "mi_kv_copy_blocks: a cycle of more than 255 blocks");

  // Tokens, KV heads and K/V by their stride.
  struct Dim {
    int64_t stride;
    uint32_t size;
    bool token;
  } dims[3] = {{token_stride, static_cast<uint32_t>(block_size), true},
               {head_stride, static_cast<uint32_t>(num_kv_heads), false},
               {values - keys, 2, false}};
  std::stable_sort(dims, dims + 3, [](const Dim& a, const Dim& b) {
    return std::abs(a.stride) < std::abs(b.stride);
  });
  PageShape p;
  p.token_dim = 0;
  for (int i = 0; i < 3; ++i) {
    p.stride[i] = dims[i].stride;
    p.size[i] = dims[i].size;
    if (dims[i].token) p.token_dim = i;
  }
  p.layer_stride = layer_stride;
  p.block_stride = block_stride;
  const uint64_t bits = static_cast<uint64_t>(row_bytes) | layer_stride | block_stride |
                        token_stride | head_stride | reinterpret_cast<uintptr_t>(keys) |
                        reinterpret_cast<uintptr_t>(values);
  if ((bits & 15u) == 0)
    return launch_copies<Words4>(keys, p, row_bytes, num_layers, order, stream);
  if ((bits & 3u) == 0)
    return launch_copies<uint32_t>(keys, p, row_bytes, num_layers, order, stream);
  return launch_copies<uint16_t>(keys, p, row_bytes, num_layers, order, stream);
}

}  // namespace
}  // namespace mi

extern "C" int32_t mi_kv_copy_blocks(void* key_cache, void* value_cache, int64_t layer_stride,
                                     int64_t block_stride, int64_t token_stride,
                                     int64_t head_stride, const int32_t* src,
                                     const int32_t* dst, const int32_t* tokens,
                                     int32_t num_pairs, int32_t num_layers,
                                     int32_t num_kv_heads, int32_t head_dim,
                                     int32_t block_size, int32_t num_blocks, int32_t dtype,
                                     void* stream) {
  using namespace mi;
  clear_error();
  if (!valid_dtype(dtype)) return fail(MI_ERR_INVALID_ARGUMENT, "mi_kv_copy_blocks: bad dtype");
  if (num_pairs < 0 || num_layers <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
      block_size <= 0 || num_blocks <= 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_kv_copy_blocks: invalid sizes");
  if (layer_stride < 0 || block_stride < 0 || token_stride < 0 || head_stride < 0)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_kv_copy_blocks: negative stride");
  const int64_t es = static_cast<int64_t>(dtype_size(dtype));
  // Word indexes and the launch's grid stay within 32 bits.
  if (static_cast<int64_t>(num_kv_heads) * block_size > (int64_t(1) << 24) ||
      head_dim > (1 << 14) ||
      2 * es * head_dim * num_kv_heads * block_size > (int64_t(1) << 28) || num_layers > 65535)
    return fail(MI_ERR_UNSUPPORTED, "mi_kv_copy_blocks: page or layer count too large");
  if (num_pairs == 0) return MI_OK;
  if (!key_cache || !value_cache || !src || !dst)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_kv_copy_blocks: null pointer");
  if (reinterpret_cast<uintptr_t>(key_cache) % es || reinterpret_cast<uintptr_t>(value_cache) % es)
    return fail(MI_ERR_INVALID_ARGUMENT, "mi_kv_copy_blocks: misaligned pointer");
  try {
    return copy_blocks(static_cast<char*>(key_cache), static_cast<char*>(value_cache),
                       layer_stride * es, block_stride * es, token_stride * es, head_stride * es,
                       src, dst, tokens, num_pairs, num_layers, num_kv_heads,
                       static_cast<int32_t>(head_dim * es), block_size, num_blocks,
                       static_cast<hipStream_t>(stream));
  } catch (const std::bad_alloc&) {
    return fail(MI_ERR_HIP, "mi_kv_copy_blocks: out of host memory");
  }
}
