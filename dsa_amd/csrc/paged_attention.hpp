// What the paged attention kernels share: arguments, the split of the work and
// the layout of the partial results that the combine kernel joins.
#pragma once

#include <type_traits>

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
// keeps fp16's small weights above its subnormal range.  They are divided out at the
// end, so a row's sum overflows where its values reach 2^114 over the number of keys
// that weigh alike, which only bf16 values can.
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
  uint32_t splits;          // selected attention: pieces that a list is cut into
  uint32_t cuts;            // else: pieces that the batch is cut for (0: no row tile is cut)
  uint32_t causal;
  uint32_t most_rows;       // sequences of more (token, head) rows per kv head are another kernel's
  uint32_t least_rows;
  uint32_t whole;           // row tiles of a single sequence that are not cut (see find_piece)
  uint32_t clears;          // this launch answers the tokens that no sequence has (see clear_unowned)
  float scale;              // times log2 e
  char* out;                // [tokens][heads][dim]
  float* lse;               // nullable: [tokens][heads]
  // Results of the pieces of row tiles that have several, [slot][kv_heads]
  // [part_rows]: outputs [dim], and {reference, sum}.
  float* part_out;
  float2* part_sum;
  uint32_t parts;           // rows that part_out and part_sum have room for
  uint32_t part_rows;
  uint2* part_of;           // chunk kernel: [tokens][heads] {part of the row's first piece, pieces}
  uint32_t* arrived;        // stream kernel: pieces of each row tile that are done; zero between calls
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

// One piece of the work: a tile of a sequence's (token, head) rows of one kv head
// against some of its keys.
constexpr uint32_t kMostSplits = 256;  // pieces of a tile

struct Piece {
  uint32_t sequence;
  Span span;
  uint32_t keys;   // of the sequence
  uint32_t tile;   // of the sequence's rows
  uint32_t units;  // of every piece of the tile but the last
  uint32_t index, count;
  uint32_t slot;   // of the tile's first piece, where there are several
};

// Piece `id` of the sequences of least_rows .. most_rows rows, in tiles of
// kTileRows rows and units of kUnit keys, at least kLeast units a piece.  No piece
// is longer than one length for the whole batch, whatever the sequences' lengths,
// so every wave sums the batch's work first: one load and a scan for up to 64
// sequences.  `cuts` pieces fill the GPU once, and a few more would run alone
// after them; so for up to 64 sequences that length grows, by up to 28 %, while the
// pieces do not fit (many sequences of unlike lengths still may not).  A tile is cut
// evenly (ragged fp16 chunks, us: 111, and 129 with the remainder in a
// tile's last piece).  At most cuts + tiles pieces, and at most 2 cuts of tiles
// that have several.  With `whole`, a multiple of cuts, there is one sequence: its
// first `whole` tiles fill the GPU some times over, and only the others are cut, into
// at most cuts pieces together.  `starts` that fall would name tokens twice and make
// more pieces than the launch has: there are none then, so that no tile is left with
// some of its pieces done and its counter raised.
template <uint32_t kTileRows, uint32_t kUnit, uint32_t kLeast>
__device__ __forceinline__ bool find_piece(const PagedAttentionArgs& a, uint32_t id, Piece& p) {
  const uint32_t lane = lane_id();
  if (a.whole) {
    p.sequence = 0;
    p.span = tokens_of(a, 0);
    p.keys = keys_of(a, 0);
    const uint32_t rows = p.span.count * a.group;
    const uint32_t tiles = rows >= a.least_rows && rows <= a.most_rows ? (rows + kTileRows - 1u) / kTileRows : 0u;
    const uint32_t units = (p.keys + kUnit - 1u) / kUnit;
    p.tile = id;
    p.units = max(1u, units);
    p.index = 0;
    p.count = 1;
    p.slot = 0;
    if (id < a.whole || tiles <= a.whole) return id < tiles;
    const uint32_t rest = tiles - a.whole;
    p.count = min(max(1u, min(a.cuts / rest, units / kLeast)), kMostSplits);
    p.tile = a.whole + (id - a.whole) / p.count;
    p.index = (id - a.whole) % p.count;
    p.units = max(1u, (units + p.count - 1u) / p.count);
    p.slot = (p.tile - a.whole) * p.count;
    return p.tile < tiles;
  }
  Span span = {0, 0};
  uint32_t keys = 0, units = 0, tiles = 0;
  auto look = [&](uint32_t b) {
    span = {0, 0};
    keys = 0;
    if (b + lane < a.sequences) {
      span = tokens_of(a, b + lane);
      keys = keys_of(a, b + lane);
    }
    const uint32_t rows = span.count * a.group;
    tiles = rows >= a.least_rows && rows <= a.most_rows ? (rows + kTileRows - 1u) / kTileRows : 0u;
    units = tiles ? (keys + kUnit - 1u) / kUnit : 0u;
  };
  auto pieces_of = [&](uint32_t each) { return max(1u, (units + each - 1u) / each); };
  p.units = 0x7fffffffu;
  if (a.cuts) {
    uint64_t all = 0;
    uint32_t most = 0;
    bool falls = false;
    for (uint32_t b = 0; b < a.sequences; b += kWave) {
      look(b);
      falls |= a.starts && b + lane < a.sequences && a.starts[b + lane + 1u] < a.starts[b + lane];
      // (two scans: a sequence's tiles x units may pass 32 bits)
      const uint64_t work = (uint64_t)tiles * units;
      all += (uint32_t)__builtin_amdgcn_readlane(wave_incl_scan((uint32_t)(work & 0xffffffu)), kWave - 1);
      all += (uint64_t)(uint32_t)__builtin_amdgcn_readlane(wave_incl_scan((uint32_t)(work >> 24)), kWave - 1) << 24;
      most = max(most, wave_max_u32(units));
    }
    if (__any(falls)) return false;
    p.units = max(max(kLeast, (most + kMostSplits - 1u) / kMostSplits), (uint32_t)((all + a.cuts - 1u) / a.cuts));
    if (a.sequences <= kWave) {
      for (uint32_t i = 0; i < 8; ++i) {
        if ((uint32_t)__builtin_amdgcn_readlane(wave_incl_scan(tiles * pieces_of(p.units)), kWave - 1) <= a.cuts) break;
        p.units += (p.units + 31u) / 32u;
      }
    }
  }
  p.slot = 0;
  for (uint32_t b = 0; b < a.sequences; b += kWave) {
    if (!a.cuts || a.sequences > kWave) look(b);
    const uint32_t each = pieces_of(p.units);
    const uint32_t pieces = tiles * each;
    const uint32_t upto = wave_incl_scan(pieces);
    const uint32_t several = each > 1u ? pieces : 0u;
    const uint32_t slots = wave_incl_scan(several);
    const uint64_t owner = __ballot(id < upto);
    if (owner) {
      const int at = __builtin_ctzll(owner);
      const uint32_t within = id - (uint32_t)__builtin_amdgcn_readlane(upto - pieces, at);
      p.sequence = b + (uint32_t)at;
      p.count = (uint32_t)__builtin_amdgcn_readlane(each, at);
      p.tile = within / p.count;
      p.index = within % p.count;
      p.slot += (uint32_t)__builtin_amdgcn_readlane(slots - several, at) + p.tile * p.count;
      p.units = max(1u, ((uint32_t)__builtin_amdgcn_readlane(units, at) + p.count - 1u) / p.count);
      p.keys = (uint32_t)__builtin_amdgcn_readlane(keys, at);
      p.span.first = (uint32_t)__builtin_amdgcn_readlane(span.first, at);
      p.span.count = (uint32_t)__builtin_amdgcn_readlane(span.count, at);
      return true;
    }
    id -= (uint32_t)__builtin_amdgcn_readlane(upto, kWave - 1);
    p.slot += (uint32_t)__builtin_amdgcn_readlane(slots, kWave - 1);
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

// Values that some rows of a causal tile do not see.  Their weight there is 0, which
// an infinity or NaN would survive; so a tile's values from the first one on that not
// every row sees are staged with what is not finite as 0 (`drop_nonfinite`), and at
// the end, if there was any, rows that do see it get it back (`add_nonfinite`).
// Costs under 1 % of the larger calls, and 0.2 us of one sequence's decode step of 11;
// 3 % of ragged chunks, whose tiles are many of them a sequence's last (109, 112 us).

// Whether any of a 16-byte run of a value row is not finite; those become 0.
template <class Tag, bool kFp8>
__device__ __forceinline__ bool drop_nonfinite(u32x4& v) {
  constexpr uint32_t kExponent = kFp8 ? 0x7f7f7f7fu : std::is_same<Tag, Bf16Tag>::value ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t kUnit = kFp8 ? 0x01010101u : std::is_same<Tag, Bf16Tag>::value ? 0x00800080u : 0x04000400u;
  constexpr uint32_t kSigns = kFp8 ? 0x80808080u : 0x80008000u;
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const uint32_t found = ((v[i] & kExponent) + kUnit) & kSigns;  // an exponent of ones (e4m3: NaN) carries
    v[i] &= ~(kFp8 ? (found >> 7) * 0xffu : (found >> 15) * 0xffffu);
    any |= found;
  }
  return any != 0;
}

__device__ __forceinline__ bool is_finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// Adds what is not finite of dims dim .. dim + 3 of a value row.
template <class Tag, bool kFp8>
__device__ __forceinline__ void add_nonfinite(const PagedAttentionArgs& a, uint32_t row, uint32_t g, uint32_t dim,
                                              float* o) {
  const char* at = a.cache.values + g * a.cache.value_head + a.cache.value_offset(row);
  float v[4];
  if constexpr (kFp8) {
    const int w = *reinterpret_cast<const int*>(at + dim);
    const float scale = a.cache.value_scales[(uint64_t)row * a.cache.kv_heads + g];
    v[0] = __builtin_amdgcn_cvt_f32_fp8(w, 0) * scale;
    v[1] = __builtin_amdgcn_cvt_f32_fp8(w, 1) * scale;
    v[2] = __builtin_amdgcn_cvt_f32_fp8(w, 2) * scale;
    v[3] = __builtin_amdgcn_cvt_f32_fp8(w, 3) * scale;
  } else {
    const uint2 w = *reinterpret_cast<const uint2*>(at + 2u * dim);
    const float2 lo = unpack2(Tag{}, w.x), hi = unpack2(Tag{}, w.y);
    v[0] = lo.x, v[1] = lo.y, v[2] = hi.x, v[3] = hi.y;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) o[i] += is_finite(v[i]) ? 0.f : v[i];
}

// Four dims of a row's result: `o` their weighted sum under `reference`, `total`
// the weights' sum.
template <class Tag, int D>
__device__ __forceinline__ void store_out(const PagedAttentionArgs& a, uint64_t row, uint32_t dim, floatx4 o,
                                          float reference, float total) {
  const float inv = total > 0.f ? 1.f / total : total;  // NaN stays
  *reinterpret_cast<uint2*>(a.out + (row * D + dim) * 2) =
      make_uint2(pack2(Tag{}, o[0] * inv, o[1] * inv), pack2(Tag{}, o[2] * inv, o[3] * inv));
  if (a.lse && dim == 0) a.lse[row] = total == 0.f ? -INFINITY : (reference + log2f(total)) * kLn2;
}

// Results of the tokens before the first sequence's and past the last one's, which a
// batch padded to a fixed number of tokens has: as rows without keys, 0 and -inf.
// Dealt to the launch's threads, 16 bytes at a time.
template <int D, uint32_t kThreads>
__device__ __forceinline__ void clear_unowned(const PagedAttentionArgs& a) {
  if (!a.clears) return;
  const uint32_t first = tokens_of(a, 0).first;
  const Span last = tokens_of(a, a.sequences - 1u);
  const uint32_t end = max(first, last.first + last.count);
  if (first == 0 && end == a.tokens) return;
  const uint64_t count = ((uint64_t)first + a.tokens - end) * a.heads;  // rows
  const uint64_t from = (uint64_t)first * a.heads;                      // those past it lie behind the sequences'
  const uint64_t skip = (uint64_t)(end - first) * a.heads;
  for (uint64_t i = (uint64_t)blockIdx.x * kThreads + threadIdx.x; i < count * (D / 8); i += (uint64_t)gridDim.x * kThreads) {
    uint64_t row = i / (D / 8);
    row += row < from ? 0u : skip;
    *reinterpret_cast<uint4*>(a.out + (row * D + i % (D / 8) * 8u) * 2u) = make_uint4(0u, 0u, 0u, 0u);
    if (a.lse && i % (D / 8) == 0) a.lse[row] = -INFINITY;
  }
}

// The chunk kernels' products and tiles.
typedef float floatx16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ floatx16 mfma_32x32x16(Bf16Tag, uint4 a, uint4 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma_32x32x16(F16Tag, uint4 a, uint4 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

constexpr uint32_t kTileKeys = 64;

// Bytes between the rows of a tile in LDS.  Padded, not exchanged, so that every
// address of a tile is one register and an offset: keys are read 16 rows at one
// 16-byte chunk, values 4 rows at 64 bytes, and each falls on all banks once.
template <int D>
constexpr int kKeyRow = 2 * D + 16;
template <int D>
constexpr int kValueRow = 2 * D + 64;

constexpr int kChunkRows = 128;        // rows of a workgroup of the chunk kernel
constexpr int kLeastChunkKeys = 256;   // keys of a piece of it

// paged_prefill.hip: the kernel of many rows, over `grid` workgroups, and its rows a
// workgroup.
constexpr int32_t prefill_rows(int64_t dim) { return dim == 256 ? 128 : 256; }
int launch_paged_prefill(const PagedAttentionArgs& a, int32_t dim, int32_t cache_dtype, uint32_t grid, hipStream_t s);

// paged_chunk.hip: the chunk kernel (head_dim 64 or 128).
int launch_paged_chunk(const PagedAttentionArgs& a, int32_t dim, int32_t cache_dtype, uint32_t grid, hipStream_t s);

}  // namespace dsa
