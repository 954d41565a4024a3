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

// One split's result of one row, or the final one where nothing is split:
// `o` is four dims' weighted sum under `reference`, `total` the weights' sum.
template <class Tag, int D>
__device__ __forceinline__ void store_row(const PagedAttentionArgs& a, uint32_t token, uint32_t head, uint32_t piece,
                                          uint32_t dim, floatx4 o, float reference, float total) {
  const uint64_t row = (uint64_t)token * a.heads + head;
  if (a.splits > 1) {
    const uint64_t at = row * a.splits + piece;
    *reinterpret_cast<floatx4*>(a.part_out + at * D + dim) = o;
    if (dim == 0) a.part_sum[at] = make_float2(reference, total);
    return;
  }
  const float inv = total > 0.f ? 1.f / total : 0.f;
  *reinterpret_cast<uint2*>(a.out + (row * D + dim) * 2) =
      make_uint2(pack2(Tag{}, o[0] * inv, o[1] * inv), pack2(Tag{}, o[2] * inv, o[3] * inv));
  if (a.lse && dim == 0) a.lse[row] = total > 0.f ? (reference + log2f(total)) * kLn2 : -INFINITY;
}

}  // namespace dsa
