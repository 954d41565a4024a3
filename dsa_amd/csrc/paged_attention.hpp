// What the paged attention kernels share: arguments, the split of the work and
// the layout of the partial results that the combine kernel joins.
#pragma once

#include "paged.hpp"
#include "waveops.hpp"

namespace dsa {

constexpr float kLog2E = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// Running maximum of a softmax that is only raised when a score passes it by
// more than kSlack (in powers of two), so that most key tiles rescale nothing
// and share no maximum between lanes.  The stored reference is the maximum at
// the last raise less kLift: weights are 2^(score - reference), about 2^kLift
// at that maximum and at most 2^(kLift + kSlack) = 2^14, inside fp16; the lift
// keeps fp16's small weights above its subnormal range.
constexpr float kLift = 6.f;
constexpr float kSlack = 8.f;
constexpr float kNoKeys = -FLT_MAX;  // reference of a row that has seen no key

struct PagedAttentionArgs {
  PagedView cache;
  const char* queries;  // [tokens][heads][dim], rows query_stride bytes apart
  int64_t query_stride;
  const int32_t* page_table;  // [sequences][columns], rows table_stride apart
  int64_t table_stride;
  uint32_t columns;
  const int32_t* lengths;   // [sequences] keys, the new tokens' included
  const int32_t* starts;    // nullable (tokens / sequences each): [sequences + 1] first token of each
  const int64_t* indices;   // selected attention: [tokens][k], rows index_stride apart
  int64_t index_stride;
  uint32_t k;
  uint32_t sequences, tokens, heads;
  uint32_t group;           // query heads per kv head
  uint32_t splits;          // pieces that a row's keys are cut into
  uint32_t causal;
  uint32_t most_rows;       // sequences of more (token, head) rows per kv head are another kernel's
  uint32_t least_rows;
  float scale;              // times log2 e
  char* out;                // [tokens][heads][dim]
  float* lse;               // nullable: [tokens][heads]
  float* part_out;          // [tokens][heads][splits][dim], splits > 1
  float2* part_sum;         // [tokens][heads][splits] {reference, sum}
  uint32_t* arrived;        // pieces of each row tile that are done (stream kernel); zero between calls
};

struct Span {
  uint32_t first, count;  // a sequence's new tokens
};

__device__ __forceinline__ Span tokens_of(const PagedAttentionArgs& a, uint32_t sequence) {
  if (!a.starts) {
    const uint32_t each = a.tokens / a.sequences;
    return {sequence * each, each};
  }
  const int32_t t = (int32_t)a.tokens;
  const int32_t first = min(max(a.starts[sequence], 0), t);
  const int32_t last = min(max(a.starts[sequence + 1], first), t);
  return {(uint32_t)first, (uint32_t)(last - first)};
}

__device__ __forceinline__ uint32_t keys_of(const PagedAttentionArgs& a, uint32_t sequence) {
  const int64_t capacity = (int64_t)a.columns << a.cache.shift;
  return (uint32_t)max((int64_t)0, min((int64_t)a.lengths[sequence], capacity));
}

// The cache row of a key of a sequence.  A page id outside the cache is read as
// its last page: the result is unspecified, the access in bounds.
__device__ __forceinline__ uint32_t cache_row(const PagedAttentionArgs& a, const int32_t* table, uint32_t key) {
  const uint32_t page = min((uint32_t)table[key >> a.cache.shift], a.cache.pages - 1u);
  return (page << a.cache.shift) | (key & ((1u << a.cache.shift) - 1u));
}

// A tile of `size` consecutive (token, head) rows of one kv head of a sequence.
struct RowTile {
  uint32_t sequence;
  uint32_t index;  // of the tile among its sequence's
  Span span;
};

// Tile `item` of the sequences of least_rows .. most_rows rows, counted over them
// in order; every wave searches for itself.  False past the last.
__device__ __forceinline__ bool find_row_tile(const PagedAttentionArgs& a, uint32_t item, uint32_t size, RowTile& tile) {
  const uint32_t lane = lane_id();
  for (uint32_t b = 0; b < a.sequences; b += kWave) {
    Span s = {0, 0};
    if (b + lane < a.sequences) s = tokens_of(a, b + lane);
    const uint32_t n = s.count * a.group;
    const uint32_t tiles = n < a.least_rows || n > a.most_rows ? 0u : (n + size - 1u) / size;
    const uint32_t upto = wave_incl_scan(tiles);
    const uint64_t owner = __ballot(item < upto);
    if (owner) {
      const int at = __builtin_ctzll(owner);
      tile.sequence = b + (uint32_t)at;
      tile.index = item - (uint32_t)__builtin_amdgcn_readlane(upto - tiles, at);
      tile.span.first = (uint32_t)__builtin_amdgcn_readlane(s.first, at);
      tile.span.count = (uint32_t)__builtin_amdgcn_readlane(s.count, at);
      return true;
    }
    item -= (uint32_t)__builtin_amdgcn_readlane(upto, kWave - 1);
  }
  return false;
}

// The sequence of a token.
__device__ __forceinline__ uint32_t sequence_of(const PagedAttentionArgs& a, uint32_t token) {
  if (!a.starts) return token / (a.tokens / a.sequences);
  const uint32_t lane = lane_id();
  uint32_t before = 0;
  for (uint32_t b = 0; b < a.sequences; b += kWave)
    before += (uint32_t)__popcll(__ballot(b + lane < a.sequences && a.starts[b + lane + 1] <= (int32_t)token));
  return min(before, a.sequences - 1u);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));

// ds_read_b64_tr_b16: lane i of a group of 16 reads 8 bytes at its own address;
// with rows r = i / 4 and 4-element runs i % 4 of a 4 x 16 block, lane i gets
// column i: one element of each of the four rows.
__device__ __forceinline__ uint2 read_transposed(const char* lds) {
  typedef __attribute__((address_space(3))) s16x4* Ptr;
  return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Ptr)(lds)));
}

// 8 bytes past the caches that XCDs do not share (agent-scope accesses), for
// pieces that another workgroup of the same launch joins.
__device__ __forceinline__ void store_shared(float2* p, float x, float y) {
  __hip_atomic_store(reinterpret_cast<uint64_t*>(p), __builtin_bit_cast(uint64_t, make_float2(x, y)), __ATOMIC_RELAXED,
                     __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ float2 load_shared(const float2* p) {
  return __builtin_bit_cast(float2, __hip_atomic_load(reinterpret_cast<const uint64_t*>(p), __ATOMIC_RELAXED,
                                                      __HIP_MEMORY_SCOPE_AGENT));
}

// Four dims of a row's result: `o` their weighted sum under `reference`, `total`
// the weights' sum.  Of one piece, for the join (kShared: in this launch):
template <int D, bool kShared>
__device__ __forceinline__ void store_part(const PagedAttentionArgs& a, uint32_t token, uint32_t head, uint32_t piece,
                                           uint32_t dim, floatx4 o, float reference, float total) {
  const uint64_t at = ((uint64_t)token * a.heads + head) * a.splits + piece;
  float* to = a.part_out + at * D + dim;
  if constexpr (kShared) {
    store_shared(reinterpret_cast<float2*>(to), o[0], o[1]);
    store_shared(reinterpret_cast<float2*>(to) + 1, o[2], o[3]);
    if (dim == 0) store_shared(a.part_sum + at, reference, total);
  } else {
    *reinterpret_cast<floatx4*>(to) = o;
    if (dim == 0) a.part_sum[at] = make_float2(reference, total);
  }
}
// Of all keys:
template <class Tag, int D>
__device__ __forceinline__ void store_out(const PagedAttentionArgs& a, uint32_t token, uint32_t head, uint32_t dim,
                                          floatx4 o, float reference, float total) {
  const uint64_t row = (uint64_t)token * a.heads + head;
  const float inv = total > 0.f ? 1.f / total : total;  // NaN stays
  *reinterpret_cast<uint2*>(a.out + (row * D + dim) * 2) =
      make_uint2(pack2(Tag{}, o[0] * inv, o[1] * inv), pack2(Tag{}, o[2] * inv, o[3] * inv));
  if (a.lse && dim == 0) a.lse[row] = total == 0.f ? -INFINITY : (reference + log2f(total)) * kLn2;
}

constexpr int kChunkRows = 128;  // rows of a workgroup of the chunk kernel

// paged_chunk.hip: the chunk kernel over `grid` workgroups.
int launch_paged_chunk(const PagedAttentionArgs& a, int32_t dim, int32_t cache_dtype, uint32_t grid, hipStream_t s);

}  // namespace dsa
