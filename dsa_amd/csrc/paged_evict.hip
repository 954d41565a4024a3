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
// Two launches.  The first finds each list's threshold (a list is a sequence's, or one
// kv head's of it) by three passes over the weights' order-preserving 32-bit keys,
// 11, 11 and 10 bits, and from it the list of moves; the second moves keys, values,
// scales and weights.
#include "paged.hpp"
#include "waveops.hpp"

namespace dsa {
namespace {

constexpr uint32_t kThreads = 1024;
constexpr uint32_t kEach = 4;                  // positions of a thread and pass
constexpr uint32_t kSpan = kThreads * kEach;   // of the workgroup

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
  // Workspace, for each list: {holes that were filled}, the keys' order, the moves
  // {to, from}; key_stride and keep entries apart.
  uint32_t* counts;
  uint32_t* order;
  uint64_t order_stride;
  uint2* moves;
  uint32_t pieces;        // bytes / 16 of a head's keys
  uint32_t head_powers;   // of an e2m1 head
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

__global__ __launch_bounds__(kThreads) void paged_evict_select_kernel(EvictArgs a) {
  __shared__ __attribute__((aligned(16))) uint32_t bins[2048];
  __shared__ __attribute__((aligned(16))) uint32_t scan[2][16];
  __shared__ Locate found;
  const uint32_t tid = threadIdx.x;
  const uint32_t list = blockIdx.x;
  const uint32_t sequence = list / a.lists, g = list % a.lists;
  const uint32_t n = keys_of(a, sequence);
  const uint32_t m = min(n, a.keep);
  const int32_t* pages = a.page_table + (int64_t)sequence * a.table_stride;
  int64_t* kept = a.kept + (uint64_t)list * a.keep;
  if (tid == 0) {
    if (g == 0) a.out_lengths[sequence] = (int32_t)m;
    a.counts[list] = 0;
  }
  for (uint32_t i = (n > m ? m : 0u) + tid; i < a.keep; i += kThreads) kept[i] = i < m ? (int64_t)i : -1;
  if (n == m) return;
  const uint32_t old = n - min(a.recent, m);   // positions that are chosen from
  const uint32_t want = m - (n - old);         // of them, fewer than there are
  uint32_t* order = a.order + (uint64_t)list * a.order_stride;
  uint2* moves = a.moves + (uint64_t)list * a.keep;

  // The weights' order, and the want-th largest of it digit by digit.
  uint32_t prefix = 0, rest = want;
  bool ties = false;  // more keys are at the threshold than are kept
  auto clear = [&]() {
    for (uint32_t i = tid; i < 2048u; i += kThreads) bins[i] = 0;
    __syncthreads();
  };
  clear();
  for (uint32_t i = tid; i < old; i += kThreads) {
    const uint32_t row = cache_row(a, pages, i);
    uint32_t key;
    if (a.lists > 1u || a.cache.kv_heads == 1u) {
      key = order_of(a.weights[g * a.row_count + row]);
    } else {
      double sum = 0.0;
      for (uint32_t h = 0; h < a.cache.kv_heads; ++h) sum += (double)a.weights[h * a.row_count + row];
      key = order_of((float)sum);
    }
    order[i] = key;
    atomicAdd(&bins[key >> 21], 1u);
  }
  if (want > 0) {
    for (int pass = 0; pass < 3; ++pass) {
      const uint32_t shift = pass == 0 ? 21u : pass == 1 ? 10u : 0u;
      const uint32_t mask = pass == 2 ? 1023u : 2047u;
      if (pass > 0) {
        clear();
        const uint32_t above = pass == 1 ? 21u : 10u;
        for (uint32_t i = tid; i < old; i += kThreads) {
          const uint32_t key = order[i];
          if (key >> above == prefix >> above) atomicAdd(&bins[(key >> shift) & mask], 1u);
        }
      }
      __syncthreads();
      if (tid < kWave) {
        const Locate l = wave_locate<32>(bins, rest, false);
        if (tid == 0) found = l;
      }
      __syncthreads();
      prefix |= found.digit << shift;
      rest = found.rem;
      ties = found.count > found.rem;
    }
  }
  __syncthreads();  // the order, as every thread has written it

  // What is kept, position by position.  Every hole lies below every source, so the
  // i-th source finds the i-th hole written.
  uint32_t tied = 0, holes = 0, sources = 0;
  for (uint32_t base = 0; base < n; base += kSpan) {
    const uint32_t at = base + kEach * tid;
    uint32_t key[kEach];
    uint32_t level = 0;
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
      key[e] = at + e < old ? order[at + e] : 0u;
      level += want > 0 && at + e < old && key[e] == prefix;
    }
    uint32_t rank = tied;
    if (ties) {
      uint32_t all;
      rank += block_excl_scan<16>(level, scan[0], all);
      tied += all;
    }
    bool keeps[kEach];
    uint32_t moved = 0;  // holes and, in the upper half, sources
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
      const bool chosen = want > 0 && (key[e] > prefix || (key[e] == prefix && (!ties || rank < rest)));
      rank += want > 0 && at + e < old && key[e] == prefix;
      keeps[e] = at + e < n && (at + e >= old || chosen);
      if (at + e < m && !keeps[e]) moved += 1u;
      if (at + e >= m && keeps[e]) moved += 1u << 16;
    }
    uint32_t all;
    const uint32_t rank_moved = block_excl_scan<16>(moved, scan[1], all);
    uint32_t hole = holes + (rank_moved & 0xffffu), source = sources + (rank_moved >> 16);
    holes += all & 0xffffu;
    sources += all >> 16;
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
      if (at + e >= m) break;
      if (keeps[e])
        kept[at + e] = at + e;
      else
        moves[hole++].x = at + e;
    }
    __syncthreads();
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
      if (at + e < m || at + e >= n) continue;
      if (keeps[e]) {
        kept[moves[source].x] = at + e;
        moves[source++].y = at + e;
      } else {
        const uint32_t row = cache_row(a, pages, at + e);
        if (a.lists > 1u || a.cache.kv_heads == 1u)
          a.weights[g * a.row_count + row] = 0.f;
        else
          for (uint32_t h = 0; h < a.cache.kv_heads; ++h) a.weights[h * a.row_count + row] = 0.f;
      }
    }
    __syncthreads();
  }
  if (tid == 0) a.counts[list] = holes;
}

// 16 bytes of a move a thread: first the keys, then the values of a head.  The thread
// of a head's first 16 has its scales and weight too.
template <Store kStore>
__global__ __launch_bounds__(256) void paged_evict_move_kernel(EvictArgs a) {
  const uint32_t list = blockIdx.y;
  const uint32_t sequence = list / a.lists;
  const uint32_t heads = a.lists > 1u ? 1u : a.cache.kv_heads;
  const int32_t* pages = a.page_table + (int64_t)sequence * a.table_stride;
  const uint2* moves = a.moves + (uint64_t)list * a.keep;
  const uint32_t units = 2u * a.pieces * heads;
  const uint64_t all = (uint64_t)a.counts[list] * units;
  for (uint64_t i = (uint64_t)blockIdx.x * 256u + threadIdx.x; i < all; i += (uint64_t)gridDim.x * 256u) {
    const uint2 move = moves[i / units];
    uint32_t unit = (uint32_t)(i % units);
    const uint32_t g = a.lists > 1u ? list % a.lists : unit / (2u * a.pieces);
    unit %= 2u * a.pieces;
    const bool value = unit >= a.pieces;
    unit -= value ? a.pieces : 0u;
    const uint32_t to = cache_row(a, pages, move.x), from = cache_row(a, pages, move.y);
    char* base = value ? a.cache.values + g * a.cache.value_head : a.cache.keys + g * a.cache.key_head;
    const uint64_t source = value ? a.cache.value_offset(from) : a.cache.key_offset(from);
    const uint64_t target = value ? a.cache.value_offset(to) : a.cache.key_offset(to);
    *reinterpret_cast<uint4*>(base + target + 16u * unit) = *reinterpret_cast<const uint4*>(base + source + 16u * unit);
    if (unit > 0) continue;
    if constexpr (kStore == kE4M3) {
      float* scales = value ? a.cache.value_scales : a.cache.key_scales;
      scales[(uint64_t)to * a.cache.kv_heads + g] = scales[(uint64_t)from * a.cache.kv_heads + g];
    }
    if constexpr (kStore == kE2M1) {
      uint8_t* powers = value ? a.cache.value_powers : a.cache.key_powers;
      const uint64_t t = a.cache.power_offset<kPowerDims>(to, g), f = a.cache.power_offset<kPowerDims>(from, g);
      for (uint32_t p = 0; p < a.head_powers; ++p) powers[t * a.head_powers + p] = powers[f * a.head_powers + p];
    }
    if (!value) {
      float* weights = a.weights + g * a.row_count;
      weights[to] = weights[from];
      weights[from] = 0.f;
    }
  }
}

struct EvictPlan {
  int64_t lists, order_stride, bytes;
};

EvictPlan evict_plan(const dsa_paged_cache* cache, int64_t sequences, int64_t columns, int64_t keep, bool per_head) {
  EvictPlan p;
  p.lists = sequences * (per_head ? cache->kv_heads : 1);
  p.order_stride = columns * cache->page_size;
  p.bytes = p.lists * 8 * keep + p.lists * 4 * p.order_stride + p.lists * 4;
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
  a.moves = static_cast<uint2*>(workspace);
  a.order = reinterpret_cast<uint32_t*>(a.moves + p.lists * keep);
  a.order_stride = (uint64_t)p.order_stride;
  a.counts = a.order + p.lists * p.order_stride;
  const int32_t bytes = cache->dtype == kFP4E2M1   ? cache->head_dim / 2
                        : cache->dtype == kFP8E4M3 ? cache->head_dim
                                                   : 2 * cache->head_dim;
  a.pieces = (uint32_t)bytes / 16;
  a.head_powers = (uint32_t)cache->head_dim / kPowerDims;
  hipStream_t s = static_cast<hipStream_t>(stream);
  hipLaunchKernelGGL(paged_evict_select_kernel, dim3((unsigned)p.lists), dim3(kThreads), 0, s, a);
  if (int st = check_launch("paged_evict_select_kernel")) return st;
  // A list moves at most keep keys, and no more than lie past it.
  const int64_t most = keep < p.order_stride - keep ? keep : p.order_stride - keep;
  if (most <= 0) return 0;
  const int64_t units = most * 2 * a.pieces * (per_head ? 1 : cache->kv_heads);
  const int64_t fill = (4096 + p.lists - 1) / p.lists;
  const int64_t blocks = (units + 255) / 256 < fill ? (units + 255) / 256 : fill;
  const dim3 grid((unsigned)blocks, (unsigned)p.lists);
  if (cache->dtype == kFP4E2M1)
    hipLaunchKernelGGL((paged_evict_move_kernel<kE2M1>), grid, dim3(256), 0, s, a);
  else if (cache->dtype == kFP8E4M3)
    hipLaunchKernelGGL((paged_evict_move_kernel<kE4M3>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((paged_evict_move_kernel<k16Bit>), grid, dim3(256), 0, s, a);
  return check_launch("paged_evict_move_kernel");
}
