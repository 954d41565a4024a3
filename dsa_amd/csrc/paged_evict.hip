// Eviction from a paged cache: each sequence cut, in place, to its newest keys and
// those of largest accumulated weight.
//
// n keys become m = min(n, keep): the newest r = min(recent, m), and of the n - r
// others the m - r of largest weight, ties to the lowest position.  Kept keys below m
// stay where they are; those from m on fill, in order, the positions below m that are
// freed, of which there are as many.  Attention takes the keys of a sequence in any
// order, so that nothing else has to move, and no move's source is another's
// destination: the moves need no order either.
//
// A list (a sequence's, or one kv head's of it) has a threshold, found by three passes
// over the weights' order-preserving 32-bit keys, 11, 11 and 10 bits, and from it its
// holes and its sources, the i-th of either being one move; the last launch moves keys,
// values, scales and weights.  Up to 16K positions a list is one workgroup's, beyond
// that the passes are launches.  Where the page table has room for more, the device
// knows which lists are longer: they are listed, and the launches deal out their chunks.
#include <algorithm>
#include <type_traits>

#include "paged.hpp"
#include "waveops.hpp"

namespace dsa {
namespace {

constexpr uint32_t kThreads = 1024;

struct Threshold;

// Lists that are longer than a workgroup's LDS has room for.
struct Listed {
  uint32_t count, chunks;
  uint32_t unused[2];
  uint2 of[1];  // {list, chunks of those before it}
};

struct EvictArgs {
  PagedView cache;
  const int32_t* page_table;
  int64_t table_stride;
  uint32_t columns;
  const int32_t* lengths;
  float* weights;         // [kv_heads][cache rows]
  uint64_t row_count;
  uint32_t keep, recent;
  uint32_t lists;         // of a sequence: kv_heads or 1
  int32_t* out_lengths;
  int64_t* kept;          // [sequences][lists][keep]
  // Workspace, for each list: its moves {to, from} (most_moves apart) and how many there
  // are; for each long one, in their order: the three passes' bins and thresholds; and of
  // their chunks, one behind the other, counts and the order of every weight.
  uint32_t* bins;
  uint2* moves;
  uint32_t* counts;
  uint4* chunks;
  Threshold* thresholds;  // after each pass
  uint32_t* order;
  Listed* listed;         // null where no list can be long
  uint32_t most_chunks, most_long;  // that there is room for
  uint32_t most_moves;    // of a list: no more than it keeps, nor than lie past those
};

__device__ __forceinline__ uint32_t cache_row(const EvictArgs& a, const int32_t* table, uint32_t key) {
  const uint32_t page = min((uint32_t)table[key >> a.cache.shift], a.cache.pages - 1u);
  return (page << a.cache.shift) | (key & ((1u << a.cache.shift) - 1u));
}

__device__ __forceinline__ uint32_t keys_of(const EvictArgs& a, uint32_t sequence) {
  const int64_t capacity = (int64_t)a.columns << a.cache.shift;
  return (uint32_t)max((int64_t)0, min((int64_t)a.lengths[sequence], capacity));
}

// Larger for larger weights; 0 for NaN.
__device__ __forceinline__ uint32_t order_of(float w) { return w == w ? float_to_ordered(w) : 0u; }

// A list: its sequence's keys before and after, and what is chosen among.
struct List {
  const int32_t* pages;
  uint32_t sequence, g, n, m;
  uint32_t old;   // positions that are chosen from: the first
  uint32_t want;  // of them, fewer than there are
};

__device__ __forceinline__ List list_of(const EvictArgs& a, uint32_t list) {
  List l;
  l.sequence = list / a.lists;
  l.g = list % a.lists;
  l.pages = a.page_table + (int64_t)l.sequence * a.table_stride;
  l.n = keys_of(a, l.sequence);
  l.m = min(l.n, a.keep);
  l.old = l.n - min(a.recent, l.m);
  l.want = l.m - (l.n - l.old);
  return l;
}

// The orders of positions first + kThreads * e + (this thread) of those that are chosen
// from; 0 past them.  Four positions under way at a time, of eight heads where a key's
// weight is their sum: a head after the other waits for memory as often as there are
// heads.
template <int kEach>
__device__ __forceinline__ void orders_of(const EvictArgs& a, const List& l, uint32_t first, uint32_t (&key)[kEach]) {
  constexpr int kTogether = kEach < 4 ? kEach : 4;
#pragma unroll
  for (uint32_t e = 0; e < kEach; e += kTogether) {
#pragma unroll
    for (int i = 0; i < kTogether; ++i) key[e + i] = 0;
    if (first + kThreads * e >= l.old) continue;  // for all threads
    uint32_t row[kTogether];
    float w[8][kTogether];
#pragma unroll
    for (int i = 0; i < kTogether; ++i)
      row[i] = cache_row(a, l.pages, min(first + threadIdx.x + kThreads * (e + i), l.n - 1u));
    if (a.lists > 1u || a.cache.kv_heads == 1u) {
#pragma unroll
      for (int i = 0; i < kTogether; ++i) w[0][i] = a.weights[l.g * a.row_count + row[i]];
    } else {
      double sum[kTogether] = {};
      for (uint32_t h0 = 0; h0 < a.cache.kv_heads; h0 += 8u) {
#pragma unroll
        for (uint32_t h = 0; h < 8; ++h)
#pragma unroll
          for (int i = 0; i < kTogether; ++i) w[h][i] = a.weights[min(h0 + h, a.cache.kv_heads - 1u) * a.row_count + row[i]];
#pragma unroll
        for (uint32_t h = 0; h < 8; ++h)
#pragma unroll
          for (int i = 0; i < kTogether; ++i) sum[i] += h0 + h < a.cache.kv_heads ? (double)w[h][i] : 0.0;
      }
#pragma unroll
      for (int i = 0; i < kTogether; ++i) w[0][i] = (float)sum[i];
    }
#pragma unroll
    for (int i = 0; i < kTogether; ++i)
      if (first + threadIdx.x + kThreads * (e + i) < l.old) key[e + i] = order_of(w[0][i]);
  }
}

// Where the want-th largest of a list's orders lies: its digits so far, how many with
// those digits are still wanted, and whether there are more of them.
struct Threshold {
  uint32_t prefix, rest, ties;
};
constexpr uint32_t kShift[3] = {21u, 10u, 0u};  // of each pass's digit
constexpr uint32_t kBins = 2048;

// The digit of `pass` added to the threshold.
__device__ __forceinline__ void locate_digit(const uint32_t* bins, uint32_t pass, Locate& shared, Threshold& t) {
  if (threadIdx.x < kWave) {
    const Locate l = wave_locate<32>(bins, t.rest, false);
    if (threadIdx.x == 0) shared = l;
  }
  __syncthreads();
  t.prefix |= shared.digit << kShift[pass];
  t.rest = shared.rem;
  t.ties = shared.count > shared.rem;
  __syncthreads();
}

// A bit for each of a thread's positions that lies below `end`.  (No difference is taken
// under a condition here, as in `end > at ? end - at : 0`: the compiler takes it for one
// that never wraps, and concludes at <= end for comparisons further on.)
template <int kEach>
__device__ __forceinline__ uint32_t bits_below(uint32_t at, uint32_t end) {
  return (1u << min(end - min(end, at), (uint32_t)kEach)) - 1u;
}

// Which of a thread's kEach positions from `at` on are kept; `rank` is that of its first
// key at the threshold among all of those.
template <int kEach>
__device__ __forceinline__ uint32_t kept_of(const List& l, const Threshold& t, const uint32_t (&key)[kEach], uint32_t at,
                                            uint32_t rank) {
  const uint32_t old = l.want > 0 ? bits_below<kEach>(at, l.old) : 0u;
  uint32_t keeps = bits_below<kEach>(at, l.n) & ~bits_below<kEach>(at, l.old);  // the newest
#pragma unroll
  for (uint32_t e = 0; e < kEach; ++e) {
    const uint32_t level = (key[e] == t.prefix) & (old >> e & 1u);
    const uint32_t chosen = (key[e] > t.prefix) | (level & (uint32_t)(!t.ties || rank < t.rest));
    rank += level;
    keeps |= (chosen & (old >> e & 1u)) << e;
  }
  return keeps;
}

// Records what the workgroup's positions from `first` on do, kEach neighbouring ones a
// thread, its kept ones the bits of `keeps`: kept ones below m stay, the others there
// are holes; kept ones from m on are sources; evicted ones there lose their weight.
// `before`: the workgroup's holes and, in the upper half, sources before the thread's,
// `all` of them; `hole`, `source`: the list's before the workgroup's.  Through LDS, so
// that neighbouring lanes store to neighbouring places.
template <int kEach>
__device__ __forceinline__ void settle(const EvictArgs& a, const List& l, uint32_t list, uint32_t first, uint32_t keeps,
                                       uint32_t before, uint32_t all, uint32_t hole, uint32_t source,
                                       uint32_t* moving, uint32_t* masks) {
  const uint32_t tid = threadIdx.x;
  const uint32_t at = first + tid * kEach;
  const uint32_t below = bits_below<kEach>(at, l.m);
  const uint32_t holes = all & 0xffffu, sources = all >> 16;
  uint32_t my_hole = before & 0xffffu, my_source = holes + (before >> 16);
  masks[tid] = keeps;
#pragma unroll
  for (uint32_t e = 0; e < kEach; ++e) {
    if ((~keeps & below) >> e & 1u) moving[my_hole++] = at + e;
    if ((keeps & ~below) >> e & 1u) moving[my_source++] = at + e;
  }
  __syncthreads();
  int64_t* kept = a.kept + (uint64_t)list * a.keep;
  uint2* moves = a.moves + (uint64_t)list * a.most_moves;
  for (uint32_t i = tid; i < holes; i += kThreads) moves[hole + i].x = moving[i];
  for (uint32_t i = tid; i < sources; i += kThreads) moves[source + i].y = moving[holes + i];
  uint32_t row[kEach];
  uint32_t evicted = 0;
#pragma unroll
  for (uint32_t e = 0; e < kEach; ++e) {
    const uint32_t within = tid + kThreads * e, i = first + within;
    const uint32_t keep = masks[within / kEach] >> within % kEach & 1u;
    if (keep & (uint32_t)(i < l.m)) kept[i] = i;
    evicted |= ((keep ^ 1u) & (uint32_t)(i >= l.m) & (uint32_t)(i < l.n)) << e;
    row[e] = cache_row(a, l.pages, min(i, l.n - 1u));
  }
  const uint32_t heads = a.lists > 1u ? 1u : a.cache.kv_heads;
  for (uint32_t h = 0; h < heads; ++h)
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e)
      if (evicted >> e & 1u) a.weights[(l.g + h) * a.row_count + row[e]] = 0.f;
}

// Holes and, in the upper half, sources among a thread's positions.
template <int kEach>
__device__ __forceinline__ uint32_t count_moves(const List& l, uint32_t at, uint32_t keeps) {
  const uint32_t below = bits_below<kEach>(at, l.m);
  return (uint32_t)__popc(~keeps & below) | (uint32_t)__popc(keeps & ~below) << 16;
}

// Positions that keep theirs where nothing is evicted, and those that a list has no key
// for.
__device__ __forceinline__ void fill_kept(const EvictArgs& a, const List& l, uint32_t list, uint32_t first, uint32_t step) {
  int64_t* kept = a.kept + (uint64_t)list * a.keep;
  for (uint32_t i = (l.n > l.m ? l.m : 0u) + first; i < a.keep; i += step) kept[i] = i < l.m ? (int64_t)i : -1;
}

// A list in one workgroup's LDS up to this many positions: 64 KiB of orders.
constexpr uint32_t kMostInLds = 16 * kThreads;
// Longer lists: a chunk of one a workgroup, one launch a pass.  The passes' counts meet
// in global memory.
constexpr uint32_t kChunkEach = 8;
constexpr uint32_t kChunk = kThreads * kChunkEach;

// Whether a list of n keys is too long for one workgroup, and loses some.
__device__ __forceinline__ bool is_long(uint32_t n, uint32_t keep) { return n > kMostInLds && n > keep; }

// Lists what is too long for one workgroup and loses keys.  One workgroup's work.  (Keys
// of one place in the cache each have room; past that nothing is listed.)
__device__ __forceinline__ void list_long(const EvictArgs& a, uint32_t lists, uint32_t* scan, uint32_t* listed) {
  uint32_t count = 0, chunks = 0;  // `chunks` stops past the room, before it could wrap
  if (threadIdx.x == 0) *listed = 0;
  for (uint32_t base = 0; base < lists; base += kThreads) {
    const uint32_t list = base + threadIdx.x;
    const uint32_t n = list < lists ? keys_of(a, list / a.lists) : 0u;
    const uint32_t own = is_long(n, a.keep) ? (n + kChunk - 1u) / kChunk : 0u;
    uint32_t all_chunks, all;
    const uint32_t before = chunks + block_excl_scan<16>(own, scan, all_chunks);
    const bool fits = own > 0 && before + own <= a.most_chunks;  // those that do are the first
    const uint32_t rank = block_excl_scan<16>(fits ? 1u : 0u, scan + 16, all);
    if (fits) a.listed->of[count + rank] = make_uint2(list, before);
    if (fits && rank + 1u == all) *listed = before + own;
    count += all, chunks = min(chunks + all_chunks, a.most_chunks + 1u);
    __syncthreads();
  }
  if (threadIdx.x > 0) return;
  a.listed->count = count;
  a.listed->chunks = *listed;
}

// How many of the lists before a sequence's are long.  For a whole workgroup.
__device__ __forceinline__ uint32_t long_before(const EvictArgs& a, uint32_t sequence, uint32_t* scan) {
  uint32_t own = 0, all;
  for (uint32_t s = threadIdx.x; s < sequence; s += kThreads) own += is_long(keys_of(a, s), a.keep);
  block_excl_scan<16>(own, scan, all);
  return all * a.lists;
}

// One workgroup a list, whose orders lie in LDS: kEach neighbouring positions a thread,
// so that every rank is one scan.  Latency bound: 11 us for one list of 4160 positions,
// 19 us for 128 of 16K.
template <int kEach>
__global__ __launch_bounds__(kThreads) void paged_evict_select_kernel(EvictArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t order[kThreads * (kEach + 1)];  // a thread's, then one word of room
  __shared__ __attribute__((aligned(16))) uint32_t bins[kBins];
  __shared__ __attribute__((aligned(16))) uint32_t scan[2][16];
  __shared__ Locate found;
  const uint32_t tid = threadIdx.x;
  if (a.listed && blockIdx.x == 0) {
    list_long(a, gridDim.x - 1u, scan[0], bins);
    return;
  }
  const uint32_t list = blockIdx.x - (a.listed ? 1u : 0u);
  const List l = list_of(a, list);
  const bool whole = l.n == l.m || l.n > kThreads * kEach;  // nothing to evict, or other launches do
  if (tid == 0) {
    if (l.g == 0) a.out_lengths[l.sequence] = (int32_t)l.m;
    if (whole) a.counts[list] = 0;
  }
  fill_kept(a, l, list, tid, kThreads);
  if (l.n == l.m) return;
  if (whole) {
    if (!a.listed) return;  // more keys than the cache has rows
    const uint32_t rank = long_before(a, l.sequence, scan[0]) + l.g;
    if (rank >= a.most_long) return;  // (the same, of several sequences)
    for (uint32_t i = tid; i < 3u * kBins; i += kThreads) a.bins[(uint64_t)rank * 3u * kBins + i] = 0;
    return;
  }
  for (uint32_t i = tid; i < kBins; i += kThreads) bins[i] = 0;
  uint32_t key[kEach];
  // (eight at a time, which leaves the registers of 1024 threads room)
  constexpr uint32_t kPart = kEach < 8 ? kEach : 8;
#pragma unroll 1
  for (uint32_t e0 = 0; e0 < kEach; e0 += kPart) {
    uint32_t part[kPart];
    orders_of<kPart>(a, l, kThreads * e0, part);
#pragma unroll
    for (uint32_t e = 0; e < kPart; ++e) {
      const uint32_t i = tid + kThreads * (e0 + e);
      order[i / kEach * (kEach + 1) + i % kEach] = part[e];
    }
  }
  __syncthreads();
  const uint32_t at = tid * kEach;
#pragma unroll
  for (uint32_t e = 0; e < kEach; ++e) key[e] = order[tid * (kEach + 1) + e];
  Threshold t = {0u, l.want, 0u};
  if (l.want > 0) {
    for (uint32_t pass = 0; pass < 3; ++pass) {
      if (pass > 0) {
        for (uint32_t i = tid; i < kBins; i += kThreads) bins[i] = 0;
        __syncthreads();
      }
#pragma unroll
      for (uint32_t e = 0; e < kEach; ++e) {
        const bool counts = at + e < l.old && (pass == 0 || key[e] >> kShift[pass - 1] == t.prefix >> kShift[pass - 1]);
        if (counts) atomicAdd(&bins[key[e] >> kShift[pass] & (pass == 2 ? 1023u : 2047u)], 1u);
      }
      __syncthreads();
      locate_digit(bins, pass, found, t);
      if (!t.ties) break;  // every key with these digits is kept: the least that they can stand for is the threshold
    }
  }
  uint32_t rank = 0, all;
  if (t.ties) {  // keys of equal weight, of which some are kept
    uint32_t level = 0;
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) level += at + e < l.old && key[e] == t.prefix;
    rank = block_excl_scan<16>(level, scan[0], all);
  }
  const uint32_t keeps = kept_of<kEach>(l, t, key, at, rank);
  const uint32_t before = block_excl_scan<16>(count_moves<kEach>(l, at, keeps), scan[1], all);
  const uint32_t holes = all & 0xffffu;
  settle<kEach>(a, l, list, 0, keeps, before, all, 0, 0, order, bins);
  int64_t* kept = a.kept + (uint64_t)list * a.keep;
  for (uint32_t i = tid; i < holes; i += kThreads) kept[order[i]] = order[holes + i];
  if (tid == 0) a.counts[list] = holes;
}

// A chunk of a listed list.
struct ChunkAt {
  uint32_t rank, list, before, chunk;  // the list's place among the listed, chunks of others before its, which of its own
};
__device__ __forceinline__ ChunkAt chunk_at(const Listed* listed, uint32_t item) {
  const uint32_t rank = last_at_most(listed->of, listed->count, item);
  const uint2 of = listed->of[rank];
  return {rank, of.x, of.y, item - of.y};
}
// The threshold after kPass passes: what the launch before this one's left of it, and
// the digit that its bins say.
template <int kPass>
__device__ __forceinline__ Threshold threshold_of(const EvictArgs& a, const List& l, const ChunkAt& c, Locate& found) {
  Threshold t = {0u, l.want, 0u};
  if (kPass == 0 || l.want == 0) return t;
  Threshold* kept = a.thresholds + (uint64_t)c.rank * 3u;
  if (kPass > 1) t = kept[kPass > 1 ? kPass - 2 : 0];
  locate_digit(a.bins + ((uint64_t)c.rank * 3u + kPass - 1) * kBins, kPass - 1, found, t);
  if (c.chunk == 0 && threadIdx.x == 0) kept[kPass - 1] = t;
  return t;
}

template <int kPass>
__global__ __launch_bounds__(kThreads) void paged_evict_count_kernel(EvictArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t bins[kBins];
  __shared__ Locate found;
  const uint32_t tid = threadIdx.x;
  for (uint32_t item = blockIdx.x; item < a.listed->chunks; item += gridDim.x) {
    const ChunkAt c = chunk_at(a.listed, item);
    const List l = list_of(a, c.list);
    const uint32_t first = c.chunk * kChunk;
    if (first >= l.old || l.want == 0) continue;
    const Threshold t = threshold_of<kPass>(a, l, c, found);
    for (uint32_t i = tid; i < kBins; i += kThreads) bins[i] = 0;
    __syncthreads();
    uint32_t* order = a.order + (uint64_t)item * kChunk;
    uint32_t own[kChunkEach];
    if (kPass == 0) orders_of<kChunkEach>(a, l, first, own);
#pragma unroll
    for (uint32_t e = 0; e < kChunkEach; ++e) {
      const uint32_t i = tid + kThreads * e;  // (inside the chunk's room, past the list's end too)
      if (kPass == 0)
        order[i] = own[e];
      else
        own[e] = order[i];
    }
#pragma unroll
    for (uint32_t e = 0; e < kChunkEach; ++e) {
      const uint32_t i = first + tid + kThreads * e;
      const uint32_t key = own[e];
      const bool counts = i < l.old && (kPass == 0 || key >> kShift[kPass ? kPass - 1 : 0] == t.prefix >> kShift[kPass ? kPass - 1 : 0]);
      if (counts) atomicAdd(&bins[key >> kShift[kPass] & (kPass == 2 ? 1023u : 2047u)], 1u);
    }
    __syncthreads();
    uint32_t* to = a.bins + ((uint64_t)c.rank * 3u + kPass) * kBins;
    for (uint32_t i = tid; i < kBins; i += kThreads)
      if (bins[i]) atomicAdd(&to[i], bins[i]);
    __syncthreads();
  }
}

// A thread's orders in a chunk: kChunkEach neighbouring positions.
__device__ __forceinline__ void load_orders(const EvictArgs& a, const List& l, uint32_t item, uint32_t at,
                                            uint32_t (&key)[kChunkEach]) {
  const uint32_t* order = a.order + (uint64_t)item * kChunk + threadIdx.x * kChunkEach;
  if (at < l.old && l.want > 0) {  // the chunk's room holds 0 past the list
    const uint4 lo = *reinterpret_cast<const uint4*>(order), hi = *reinterpret_cast<const uint4*>(order + 4);
    key[0] = lo.x, key[1] = lo.y, key[2] = lo.z, key[3] = lo.w;
    key[4] = hi.x, key[5] = hi.y, key[6] = hi.z, key[7] = hi.w;
  } else {
#pragma unroll
    for (uint32_t e = 0; e < kChunkEach; ++e) key[e] = 0;
  }
}

// Of each chunk: keys at the threshold, and above it or newest, below position m and
// from there on.
__global__ __launch_bounds__(kThreads) void paged_evict_chunk_kernel(EvictArgs a) {
  __shared__ Locate found;
  __shared__ uint32_t sums[4];
  for (uint32_t item = blockIdx.x; item < a.listed->chunks; item += gridDim.x) {
    const ChunkAt c = chunk_at(a.listed, item);
    const List l = list_of(a, c.list);
    const uint32_t first = c.chunk * kChunk;
    const Threshold t = threshold_of<3>(a, l, c, found);
    if (threadIdx.x < 4u) sums[threadIdx.x] = 0;
    __syncthreads();
    const uint32_t at = first + threadIdx.x * kChunkEach;
    uint32_t key[kChunkEach];
    load_orders(a, l, item, at, key);
    uint32_t count[4] = {0u, 0u, 0u, 0u};
#pragma unroll
    for (uint32_t e = 0; e < kChunkEach; ++e) {
      const uint32_t past = at + e >= l.m ? 2u : 0u;
      const bool level = l.want > 0 && at + e < l.old && key[e] == t.prefix;
      const bool sure = at + e < l.n && (at + e >= l.old || (l.want > 0 && key[e] > t.prefix));
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) count[i] += (i == past && level) || (i == past + 1u && sure);
    }
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      const uint32_t all = (uint32_t)__builtin_amdgcn_readlane(wave_incl_scan(count[i]), kWave - 1);
      if (lane_id() == 0 && all) atomicAdd(&sums[i], all);
    }
    __syncthreads();
    if (threadIdx.x == 0)
      a.chunks[item] = make_uint4(sums[0], sums[1], sums[2], sums[3]);
    __syncthreads();
  }
}

// What is kept, a chunk a workgroup, from the counts of the chunks before it.
__global__ __launch_bounds__(kThreads) void paged_evict_settle_kernel(EvictArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t scan[2][16];
  __shared__ uint32_t moving[kChunk], masks[kThreads];
  __shared__ uint32_t start[3];  // ranks of the chunk's first: key at the threshold, hole, source
  for (uint32_t item = blockIdx.x; item < a.listed->chunks; item += gridDim.x) {
    const ChunkAt c = chunk_at(a.listed, item);
    const List l = list_of(a, c.list);
    const uint32_t first = c.chunk * kChunk;
    const Threshold t = l.want > 0 ? a.thresholds[(uint64_t)c.rank * 3u + 2u] : Threshold{0u, 0u, 0u};
    if (threadIdx.x < kWave) {
      // Keys at the threshold are kept while their rank is below t.rest; that rank follows
      // the chunks, so a chunk keeps as many as are left of them.
      uint32_t level = 0, kept_below = 0, kept_past = 0;
      for (uint32_t base = 0; base < c.chunk; base += kWave) {
        const uint32_t i = base + lane_id();
        const uint4 v = i < c.chunk ? a.chunks[c.before + i] : make_uint4(0u, 0u, 0u, 0u);
        const uint32_t upto = level + wave_incl_scan(v.x + v.z);
        const uint32_t from = upto - v.x - v.z;
        const uint32_t limit = t.ties ? t.rest : 0xffffffffu;
        const uint32_t below = min(v.x, limit - min(limit, from));
        const uint32_t past = min(v.z, limit - min(limit, from + v.x));
        kept_below += (uint32_t)__builtin_amdgcn_readlane(wave_incl_scan(v.y + below), kWave - 1);
        kept_past += (uint32_t)__builtin_amdgcn_readlane(wave_incl_scan(v.w + past), kWave - 1);
        level = (uint32_t)__builtin_amdgcn_readlane(upto, kWave - 1);
      }
      if (threadIdx.x == 0) {
        start[0] = level;
        start[1] = min(first, l.m) - kept_below;
        start[2] = kept_past;
      }
    }
    __syncthreads();
    const uint32_t at = first + threadIdx.x * kChunkEach;
    uint32_t key[kChunkEach];
    load_orders(a, l, item, at, key);
    uint32_t rank = start[0], all;
    if (t.ties) {
      uint32_t level = 0;
#pragma unroll
      for (uint32_t e = 0; e < kChunkEach; ++e) level += at + e < l.old && key[e] == t.prefix;
      rank += block_excl_scan<16>(level, scan[0], all);
    }
    const uint32_t keeps = kept_of<kChunkEach>(l, t, key, at, rank);
    const uint32_t before = block_excl_scan<16>(count_moves<kChunkEach>(l, at, keeps), scan[1], all);
    settle<kChunkEach>(a, l, c.list, first, keeps, before, all, start[1], start[2], moving, masks);
    if (threadIdx.x == 0 && first < l.m && l.m <= first + kChunk) a.counts[c.list] = start[1] + (all & 0xffffu);
    __syncthreads();
  }
}

// Moves: 16 bytes of a head's key and of its value a thread, two at a time; a move's
// heads are neighbouring threads, so that what heads share, a row's scales in one cache
// line, is written by one workgroup.  The first thread of a head has its scales and weight
// too.  What is on its way is held in the compiler's own vectors: arrays of uint4 went to
// LDS or scratch (16 sequences of 16K bf16 keys cut to 4K, 128 lists, 316 MB read and
// written: 60 us, 5.3 TB/s, and 88 us with them).
template <Store kStore, int kPieces>
__global__ __launch_bounds__(256) void paged_evict_move_kernel(EvictArgs a) {
  constexpr uint32_t kPairs = 256 / kPieces;  // of a move and a head, of the workgroup at a time
  constexpr uint32_t kBlocks = kStore == kE2M1 ? kPieces * 32 / kPowerDims : 1;  // powers of a head
  typedef typename std::conditional<kBlocks == 8, uint64_t, typename std::conditional<kBlocks == 4, uint32_t, uint16_t>::type>::type Powers;
  const uint32_t list = blockIdx.y;
  const uint32_t sequence = list / a.lists;
  const int32_t* pages = a.page_table + (int64_t)sequence * a.table_stride;
  const uint2* moves = a.moves + (uint64_t)list * a.most_moves;
  const uint32_t count = a.counts[list];
  if (a.listed) {  // (a long list's; the others' again)
    for (uint32_t i = blockIdx.x * 256u + threadIdx.x; i < count; i += gridDim.x * 256u)
      a.kept[(uint64_t)list * a.keep + moves[i].x] = moves[i].y;
  }
  const uint32_t piece = threadIdx.x % kPieces;
  const uint32_t heads = a.lists > 1u ? 1u : a.cache.kv_heads;
  const uint32_t step = gridDim.x * kPairs;
  const uint32_t pair = blockIdx.x * kPairs + threadIdx.x / kPieces;  // (the grid is small: both fit)
  uint32_t i = pair / heads, h = pair % heads;
  auto next = [&]() {
    i += step / heads;
    h += step % heads;
    if (h >= heads) {
      h -= heads;
      ++i;
    }
  };
  while (i < count) {
    u32x2 move[2];
    uint32_t g[2];
    move[0] = *reinterpret_cast<const u32x2*>(moves + i);
    g[0] = a.lists > 1u ? list % a.lists : h;
    next();
    const bool both = i < count;
    move[1] = *reinterpret_cast<const u32x2*>(moves + (both ? i : count - 1u));
    g[1] = a.lists > 1u ? list % a.lists : h;
    next();
    uint32_t to[2], from[2];
    char *keys[2], *values[2];
    float* weights[2];
    u32x4 k[2], v[2];
    float weight[2], key_scale[2], value_scale[2];
    Powers key_powers[2], value_powers[2];
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      to[m] = cache_row(a, pages, move[m].x);
      from[m] = cache_row(a, pages, move[m].y);
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      keys[m] = a.cache.keys + g[m] * a.cache.key_head + 16u * piece;
      values[m] = a.cache.values + g[m] * a.cache.value_head + 16u * piece;
      weights[m] = a.weights + g[m] * a.row_count;
      k[m] = *reinterpret_cast<const u32x4*>(keys[m] + a.cache.key_offset(from[m]));
      v[m] = *reinterpret_cast<const u32x4*>(values[m] + a.cache.value_offset(from[m]));
      if (piece > 0) continue;
      weight[m] = weights[m][from[m]];
      if constexpr (kStore == kE4M3) {
        const uint64_t f = (uint64_t)from[m] * a.cache.kv_heads + g[m];
        key_scale[m] = a.cache.key_scales[f];
        value_scale[m] = a.cache.value_scales[f];
      }
      if constexpr (kStore == kE2M1) {
        const uint64_t f = a.cache.power_offset<kBlocks * kPowerDims>(from[m], g[m]);
        key_powers[m] = *reinterpret_cast<const Powers*>(a.cache.key_powers + f);
        value_powers[m] = *reinterpret_cast<const Powers*>(a.cache.value_powers + f);
      }
    }
#pragma unroll
    for (int m = 0; m < 2; ++m) {
      if (m == 1 && !both) break;
      *reinterpret_cast<u32x4*>(keys[m] + a.cache.key_offset(to[m])) = k[m];
      *reinterpret_cast<u32x4*>(values[m] + a.cache.value_offset(to[m])) = v[m];
      if (piece > 0) continue;
      weights[m][to[m]] = weight[m];
      weights[m][from[m]] = 0.f;
      if constexpr (kStore == kE4M3) {
        const uint64_t t = (uint64_t)to[m] * a.cache.kv_heads + g[m];
        a.cache.key_scales[t] = key_scale[m];
        a.cache.value_scales[t] = value_scale[m];
      }
      if constexpr (kStore == kE2M1) {
        const uint64_t t = a.cache.power_offset<kBlocks * kPowerDims>(to[m], g[m]);
        *reinterpret_cast<Powers*>(a.cache.key_powers + t) = key_powers[m];
        *reinterpret_cast<Powers*>(a.cache.value_powers + t) = value_powers[m];
      }
    }
  }
}

template <Store kStore>
void launch_move(const EvictArgs& a, int32_t pieces, dim3 grid, hipStream_t s) {
  if constexpr (kStore == kE2M1) {
    if (pieces == 2) hipLaunchKernelGGL((paged_evict_move_kernel<kStore, 2>), grid, dim3(256), 0, s, a);
  }
  if constexpr (kStore != k16Bit) {
    if (pieces == 4) hipLaunchKernelGGL((paged_evict_move_kernel<kStore, 4>), grid, dim3(256), 0, s, a);
  }
  if (pieces == 8) hipLaunchKernelGGL((paged_evict_move_kernel<kStore, 8>), grid, dim3(256), 0, s, a);
  if constexpr (kStore != kE2M1) {
    if (pieces == 16) hipLaunchKernelGGL((paged_evict_move_kernel<kStore, 16>), grid, dim3(256), 0, s, a);
  }
  if constexpr (kStore == k16Bit) {
    if (pieces == 32) hipLaunchKernelGGL((paged_evict_move_kernel<kStore, 32>), grid, dim3(256), 0, s, a);
  }
}

constexpr int64_t kChunkWorkgroups = 512;  // that long lists' chunks are dealt to: what runs at a time

struct EvictPlan {
  int64_t lists, most_chunks;  // no chunks: every list is one workgroup's
  int64_t most_long, most_moves;  // long lists, moves of a list
  int64_t moves, counts, thresholds, listed, chunk_counts, order, bytes;  // offsets, after the bins
};

EvictPlan evict_plan(const dsa_paged_cache* cache, int64_t sequences, int64_t columns, int64_t keep, bool per_head) {
  EvictPlan p = {};
  const int64_t capacity = columns * cache->page_size, heads = per_head ? cache->kv_heads : 1;
  p.lists = sequences * heads;
  const int64_t rows = cache->pages * cache->page_size;
  if (std::min(capacity, rows) > kMostInLds) {
    // A cache row is one sequence's, and a list of more than two chunks has at most half
    // as many again as its keys fill.  (Each list by its own length: 256 sequences of 4160
    // keys, a list a head of 8, in tables with room for 128K: 140 us, and 1490 with every
    // list in chunks; with room for 8K 101.)
    static_assert(kMostInLds == 2 * kChunk, "");
    p.most_chunks = std::min(heads * std::min(sequences * ((capacity + kChunk - 1) / kChunk), rows * 3 / kMostInLds), (int64_t)1 << 30);
  }
  p.most_long = std::min(p.lists, p.most_chunks / 3);  // what is listed has three chunks at least, within their room
  p.moves = p.most_long * 3 * kBins * 4;
  p.most_moves = std::max(std::min(keep, capacity - keep), (int64_t)0);
  p.counts = p.moves + p.lists * p.most_moves * 8;
  p.thresholds = p.counts + p.lists * 4;
  p.listed = (p.thresholds + p.most_long * 36 + 15) / 16 * 16;
  p.chunk_counts = p.listed + (p.most_chunks ? (16 + p.lists * 8 + 15) / 16 * 16 : 0);
  p.order = p.chunk_counts + p.most_chunks * 16;
  p.bytes = p.order + p.most_chunks * kChunk * 4;
  return p;
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int64_t dsa_paged_evict_workspace_bytes(const dsa_paged_cache* cache, int64_t sequences, int64_t columns,
                                                   int64_t keep, int32_t per_head) {
  if (!cache || cache->kv_heads <= 0 || cache->page_size <= 0 || sequences <= 0 || columns <= 0 || keep <= 0) return 0;
  return evict_plan(cache, sequences, columns, keep, per_head != 0).bytes;
}

extern "C" int dsa_paged_evict(const dsa_paged_cache* cache, const int32_t* page_table, int64_t table_stride,
                               int64_t columns, const int32_t* lengths, int64_t sequences, float* weights, int64_t keep,
                               int64_t recent, int32_t per_head, int32_t* out_lengths, int64_t* kept, void* workspace,
                               int64_t workspace_bytes, void* stream) {
  EvictArgs a = {};
  if (int st = make_paged_view(cache, a.cache)) return st;
  DSA_REQUIRE(page_table && lengths && weights && out_lengths && kept, "null pointer argument");
  DSA_REQUIRE(sequences > 0 && sequences <= (1 << 20), "sequences out of range");
  DSA_REQUIRE(columns > 0 && columns < (1LL << 31) && columns * cache->page_size <= (1LL << 30) && table_stride >= columns,
              "page table of %lld columns out of range", (long long)columns);
  DSA_REQUIRE(keep > 0 && keep <= (1LL << 30), "keep %lld must be in 1..2^30", (long long)keep);
  DSA_REQUIRE(recent >= 0 && recent <= keep, "recent %lld must be in 0..keep", (long long)recent);
  const EvictPlan p = evict_plan(cache, sequences, columns, keep, per_head != 0);
  if (!workspace || workspace_bytes < p.bytes || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(DSA_STATUS_WORKSPACE_TOO_SMALL, "paged eviction needs %lld bytes of 16-byte aligned workspace",
                (long long)p.bytes);
  DSA_REQUIRE(p.lists < 65536, "too many sequences for one call");
  // The first launch writes the new lengths, and every one reads the old ones.
  DSA_REQUIRE(out_lengths + sequences <= lengths || lengths + sequences <= out_lengths,
              "out_lengths must not overlap lengths");
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.columns = (uint32_t)columns;
  a.lengths = lengths;
  a.weights = weights;
  a.row_count = (uint64_t)cache->pages * cache->page_size;
  a.keep = (uint32_t)keep;
  a.recent = (uint32_t)recent;
  a.lists = per_head ? (uint32_t)cache->kv_heads : 1u;
  a.out_lengths = out_lengths;
  a.kept = kept;
  char* base = static_cast<char*>(workspace);
  a.bins = reinterpret_cast<uint32_t*>(base);
  a.moves = reinterpret_cast<uint2*>(base + p.moves);
  a.counts = reinterpret_cast<uint32_t*>(base + p.counts);
  a.thresholds = reinterpret_cast<Threshold*>(base + p.thresholds);
  a.chunks = reinterpret_cast<uint4*>(base + p.chunk_counts);
  a.order = reinterpret_cast<uint32_t*>(base + p.order);
  a.listed = p.most_chunks ? reinterpret_cast<Listed*>(base + p.listed) : nullptr;
  a.most_chunks = (uint32_t)p.most_chunks;
  a.most_long = (uint32_t)p.most_long;
  a.most_moves = (uint32_t)p.most_moves;
  hipStream_t s = static_cast<hipStream_t>(stream);
  const int64_t capacity = columns * cache->page_size;
  const dim3 lists((unsigned)p.lists + (p.most_chunks ? 1u : 0u));
  if (capacity > 8 * kThreads)
    hipLaunchKernelGGL(paged_evict_select_kernel<16>, lists, dim3(kThreads), 0, s, a);
  else if (capacity > 2 * kThreads)
    hipLaunchKernelGGL(paged_evict_select_kernel<8>, lists, dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL(paged_evict_select_kernel<2>, lists, dim3(kThreads), 0, s, a);
  if (p.most_chunks) {
    const dim3 chunks((unsigned)std::min(p.most_chunks, kChunkWorkgroups));
    hipLaunchKernelGGL(paged_evict_count_kernel<0>, chunks, dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(paged_evict_count_kernel<1>, chunks, dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(paged_evict_count_kernel<2>, chunks, dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(paged_evict_chunk_kernel, chunks, dim3(kThreads), 0, s, a);
    hipLaunchKernelGGL(paged_evict_settle_kernel, chunks, dim3(kThreads), 0, s, a);
  }
  if (int st = check_launch("paged_evict_select_kernel")) return st;
  if (p.most_moves == 0) return 0;
  const int32_t bytes = cache->dtype == kFP4E2M1   ? cache->head_dim / 2
                        : cache->dtype == kFP8E4M3 ? cache->head_dim
                                                   : 2 * cache->head_dim;
  const int32_t pieces = bytes / 16;
  const int64_t heads = per_head ? 1 : cache->kv_heads;
  const int64_t fill = (4096 + p.lists - 1) / p.lists;
  const int64_t blocks = std::min((p.most_moves * heads * pieces + 511) / 512, fill);
  const dim3 grid((unsigned)blocks, (unsigned)p.lists);
  if (cache->dtype == kFP4E2M1)
    launch_move<kE2M1>(a, pieces, grid, s);
  else if (cache->dtype == kFP8E4M3)
    launch_move<kE4M3>(a, pieces, grid, s);
  else
    launch_move<k16Bit>(a, pieces, grid, s);
  return check_launch("paged_evict_move_kernel");
}
