// Attention over a paged key/value cache: a few query rows against many keys.
//
//   s_j = scale q . k_j,  o = sum_j exp(s_j) v_j / sum_j exp(s_j)
//
// over the keys a row sees: its sequence's first ones up to its own position,
// or the positions its index list names.  One pass over the keys with the
// running maximum and sum of the softmax; scores, weights' sum and output stay
// in fp32, and the weights (times an fp8 value's scale) are rounded to the queries'
// type for the second product, whose error then is of the output's own rounding.
//
// A workgroup takes 16 rows, which are (token, head) pairs of one kv head,
// against one piece of the keys; its four waves take steps of 32 keys each.  Bound
// by HBM: 16 sequences of 32K bf16 keys (2.15 GB) take 368 us, 5.8 TB/s, where a
// plain read of 2 GiB makes 5.9; 4 of up to 128K fp8 keys 160 us, 5.0 TB/s.
// Keys are the A operand of v_mfma_f32_16x16x32 and queries the B operand, so a
// lane ends with eight scores of ONE row (lane & 15) and those are, as they
// stand, the B operand of the second product: its k index is any order of the
// 32 keys that both operands share, and here is the order the scores have.  The
// values' transposed operand is read from LDS by ds_read_b64_tr_b16.  Every row
// of the cache is read once, as 16-byte loads of up to 128 contiguous bytes a row.
#include "paged_attention.hpp"

namespace dsa {
namespace {

constexpr uint32_t kStep = 32;   // keys per wave and step
// Steps of a piece, at least: two for each wave.  (One sequence of 4096 bf16 keys,
// us: 10.9, with one step 13.0, whose twice as many pieces take longer to join.)
constexpr uint32_t kLeastSteps = 8;
constexpr uint32_t kGroup = 8;   // steps whose cache rows a wave looks up at a time
// Workgroups that run at a time: what the registers of each head_dim allow on 256
// CUs.  Work is cut to fill them once.
template <int D>
constexpr int kPerCu = D == 64 ? 3 : D == 128 ? 2 : 1;
constexpr int64_t resident_workgroups(int64_t dim) { return 256 * (dim == 64 ? kPerCu<64> : dim == 128 ? kPerCu<128> : kPerCu<256>); }
constexpr int kCounters = 4096;  // of row tiles that are cut, by kv head

// LDS that the lanes of one wave share: a wave's LDS accesses are served in
// order, so only the compiler has to keep them so.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Place of 16-byte chunk `chunk` of row `row` in a wave's key or value tile of
// kBytes a row.  The chunks of a row are exchanged by an exclusive or with bits of
// the row, so that the accesses served together fall on different banks: rows
// stored 64 or 128 bytes at a time, 16 rows read at one chunk (keys), 8 rows at
// two (half a transposed read of values).
template <int kBytes>
__device__ __forceinline__ uint32_t tile_place(uint32_t row, uint32_t chunk) {
  uint32_t x;
  if constexpr (kBytes == 64)
    x = (row >> 2) & 3u;
  else if constexpr (kBytes == 128)
    x = (((row >> 1) & 1u) << 2) | (((row >> 2) & 1u) << 1) | ((row >> 3) & 1u);
  else
    x = ((row & 1u) << 3) | (((row >> 1) & 1u) << 2) | (((row >> 2) & 1u) << 1) | ((row >> 3) & 1u);
  return row * kBytes + ((chunk ^ x) << 4);
}

// A step's rows on their way from the cache.  Neighbouring lanes load neighbouring
// 16-byte runs of a row (kLanes of them, 128 bytes where the row has as many): one
// load that touches a different row in every lane moves a quarter of the bytes a
// cycle, and held a decode step of cached keys that are all in L2 to 8 TB/s.
template <bool kFp8, int D>
struct Tile {
  static constexpr int kBytes = kFp8 ? D : 2 * D;               // of a cache row
  static constexpr int kLanes = kBytes < 128 ? kBytes / 16 : 8;  // that share a row
  static constexpr int kRows = 64 / kLanes;                      // of one load
  static constexpr int kPasses = kStep / kRows;
  static constexpr int kLoads = kBytes / (16 * kLanes);          // of one row
  u32x4 k[kPasses][kLoads];
  u32x4 v[kPasses][kLoads];
  float scale;  // fp8: lane l < 32 the key scale of key l, else the value scale of key l - 32
};

// What a workgroup of the stream kernel takes.
enum Work {
  kDense,     // a piece of a sequence's keys
  kBeside,    // the same for two heads that lie side by side, eight waves
  kSelected,  // a piece of a token's list
  kSolo,      // four tokens' lists, each wave one by itself
};

// Heads of a workgroup, four waves each, and waves that a SIMD holds.
template <Work kWork>
constexpr int kHeadsOf = kWork == kBeside ? 2 : 1;
template <int D, Work kWork>
constexpr int kPerSimd = kWork == kBeside ? 2 : kPerCu<D>;

template <class Tag, bool kFp8, int D, Work kWork>
__global__ __launch_bounds__(256 * kHeadsOf<kWork>, (kPerSimd<D, kWork>)) void paged_stream_kernel(PagedAttentionArgs a) {
  using T = Tile<kFp8, D>;
  constexpr bool kListed = kWork == kSelected || kWork == kSolo;
  constexpr int kHeads = kHeadsOf<kWork>;
  constexpr uint32_t kWaves = 4;  // of a head
  constexpr uint32_t kThreads = 64 * kWaves * kHeads;
  constexpr uint32_t kAhead = kFp8 ? 2 : 1;  // steps on their way in registers
  constexpr int kQ = D / 32;  // k-steps of the first product
  constexpr int kO = D / 16;  // dim tiles of the second
  // A wave's value tile (at the end its output) and key tile, one offset apart.
  constexpr uint32_t kValues = kStep * D * 2;
  __shared__ __attribute__((aligned(16))) char tiles[kWaves * kHeads][kValues + kStep * T::kBytes];
  // A wave's cache rows of this group of steps and the next; negative: padding.
  __shared__ __attribute__((aligned(16))) int32_t table[kWaves * kHeads][2][kGroup * kStep];
  __shared__ __attribute__((aligned(16))) float scales[kWaves * kHeads][64];
  __shared__ float2 sums[kWaves * kHeads][16];
  __shared__ uint32_t last_piece;
  const uint32_t lane = lane_id();
  const uint32_t wave = threadIdx.x / kWave;
  const uint32_t col = lane & 15u;
  const uint32_t quad = lane >> 4;

  // Workgroups go round-robin over the XCDs.  Heads vary fastest, so a kv head's
  // rows meet in few L2s; but the heads of an fp8 piece, whose scales share cache
  // lines, follow each other on one XCD (16 bit / fp8 decode steps, us: heads
  // fastest 385 / 209, heads on one XCD 397 / 191).
  constexpr bool kTogether = kFp8 && !kListed;
  const uint32_t turn = kTogether ? blockIdx.x / kXcds : blockIdx.x;
  const uint32_t kinds = a.cache.kv_heads / kHeads;
  const uint32_t g0 = turn % kinds * kHeads;
  const uint32_t g = kHeads == 1 ? g0 : g0 + wave / kWaves;  // this wave's head
  const uint32_t id = kTogether ? turn / kinds * kXcds + blockIdx.x % kXcds : turn / kinds;

  uint32_t sequence, token0, row0, rows, length, begin, end, pieces, index, slot, tile_slot, seen0 = 0;
  if constexpr (kListed) {
    // a piece of the list of a tile of a token's heads
    const uint32_t tiles = (a.group + 15u) / 16u;
    const uint32_t item = kWork == kSolo ? 4u * id + wave : id / a.splits;
    const uint32_t piece = kWork == kSolo ? 0u : id % a.splits;
    token0 = item / tiles;
    if (kWork == kSolo && token0 >= a.tokens) return;
    row0 = item % tiles * 16u;
    rows = a.group;
    sequence = sequence_of(a, token0);
    length = keys_of(a, sequence);
    if (a.starts) {
      const Span span = tokens_of(a, sequence);
      if (token0 - span.first >= span.count) length = 0;  // no sequence's
    }
    const uint32_t visible = length ? a.k : 0u;
    const uint32_t chunk = max(kLeastSteps * kStep, ((a.k + a.splits - 1u) / a.splits + 31u) & ~31u);
    begin = min(piece * chunk, visible);
    end = min(begin + chunk, visible);
    pieces = a.splits;
    index = piece;
    tile_slot = item;
    slot = item * a.splits;
  } else {
    Piece piece;
    const bool found = find_piece<16, kStep, kLeastSteps>(a, id, piece);
    clear_unowned<D, kThreads>(a);
    if (!found) return;
    sequence = piece.sequence;
    token0 = piece.span.first;
    row0 = piece.tile * 16u;
    rows = piece.span.count * a.group;
    length = piece.keys;
    // row r sees keys below seen0 + r / group + 1 of a causal chunk; its tile's last sees most
    seen0 = length - piece.span.count;  // may wrap below zero: see `sees`
    const uint32_t last = min(row0 + 16u, rows) - 1u;
    const uint32_t visible = a.causal ? (uint32_t)max(0, (int32_t)(seen0 + last / a.group + 1u)) : length;
    begin = (uint32_t)min((uint64_t)piece.index * piece.units * kStep, (uint64_t)visible);
    end = (uint32_t)min((uint64_t)begin + (uint64_t)piece.units * kStep, (uint64_t)visible);
    pieces = piece.count;
    index = piece.index;
    tile_slot = slot = piece.slot;
  }

  // This lane's row, and the keys it sees.
  const uint32_t my_row = min(row0 + col, rows - 1u);
  const uint32_t my_token = kListed ? token0 : token0 + my_row / a.group;
  const uint32_t my_head = g * a.group + (kListed ? my_row : my_row % a.group);
  const bool partly = !kListed && a.causal;
  const uint32_t sees = partly ? (uint32_t)max(0, (int32_t)(seen0 + my_row / a.group + 1u)) : end;
  const uint32_t all_see = partly ? (uint32_t)max(0, (int32_t)(seen0 + row0 / a.group + 1u)) : end;

  auto out_row = [&](uint32_t h, uint32_t r) {
    const uint64_t token = kListed ? token0 : token0 + (row0 + r) / a.group;
    return token * a.heads + (g0 + h) * a.group + (kListed ? row0 + r : (row0 + r) % a.group);
  };
  auto part_at = [&](uint32_t piece, uint32_t h, uint32_t r) {
    return ((uint64_t)piece * a.cache.kv_heads + g0 + h) * a.part_rows + r;
  };

  uint4 q[kQ];
  {
    const char* p = a.queries + (int64_t)my_token * a.query_stride + (uint64_t)my_head * D * 2;
#pragma unroll
    for (int j = 0; j < kQ; ++j) {
      const uint32_t d = kFp8 ? 64u * (j / 2) + 16u * quad + 8u * (j % 2) : 32u * j + 8u * quad;
      q[j] = *reinterpret_cast<const uint4*>(p + d * 2);
    }
  }
  const uint32_t load_row = lane / T::kLanes;
  const uint32_t load_chunk = lane % T::kLanes;
  const char* key_base = a.cache.keys + g * a.cache.key_head + 16u * load_chunk;
  const char* value_base = a.cache.values + g * a.cache.value_head + 16u * load_chunk;
  const int32_t* pages = a.page_table + (int64_t)sequence * a.table_stride;
  const int64_t* list = kListed ? a.indices + (int64_t)token0 * a.index_stride : nullptr;

  floatx4 o[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float reference = kNoKeys;
  float total = 0.f;  // of this lane's keys
  char* mine = tiles[wave];
  char* my_keys = mine + kValues;
  uint32_t tr_place[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i)
    tr_place[i] = tile_place<2 * D>(4u * quad + (col >> 2), 2u * i + ((col & 3u) >> 1)) + 8u * (col & 1u);

  // The steps of a piece are dealt to its head's waves (a list of its own is all
  // the wave's), step s at keys first_key(s).
  constexpr uint32_t kApart = kWork == kSolo ? 1 : kWaves;
  const uint32_t from = kWork == kSolo ? 0u : wave % kWaves;
  const uint32_t steps = (end - begin + kStep - 1u) / kStep;
  const uint32_t own = steps > from ? (steps - from + kApart - 1u) / kApart : 0u;
  auto first_key = [&](uint32_t step) { return begin + (kApart * step + from) * kStep; };
  auto rows_at = [&](uint32_t step) { return table[wave][step / kGroup % 2u] + step % kGroup * kStep; };

  // The cache rows of a group of steps, in three parts so that a group's look-ups
  // run under the steps before it: list entries, page ids, the table.  Lane l has
  // keys l % 32 of steps 2 j + l / 32.
  constexpr uint32_t kRounds = kGroup / 2;
  uint32_t key[kRounds], page[kRounds];
  auto look_keys = [&](uint32_t group) {
#pragma unroll
    for (uint32_t j = 0; j < kRounds; ++j) {
      const uint32_t at = first_key(group * kGroup + 2u * j + lane / 32u) + lane % 32u;
      key[j] = min(at, end - 1u);
      if constexpr (kListed) {
        const int64_t named = list[key[j]];
        key[j] = at < end && named >= 0 && named < (int64_t)length ? (uint32_t)named : 0x80000000u;
      }
    }
  };
  auto look_pages = [&]() {
#pragma unroll
    for (uint32_t j = 0; j < kRounds; ++j) page[j] = (uint32_t)pages[(key[j] & 0x7fffffffu) >> a.cache.shift];
  };
  auto look_rows = [&](uint32_t group) {
#pragma unroll
    for (uint32_t j = 0; j < kRounds; ++j)
      table[wave][group % 2u][64u * j + lane] =
          (int32_t)((min(page[j], a.cache.pages - 1u) << a.cache.shift) | (key[j] & ((1u << a.cache.shift) - 1u)) |
                    (key[j] & 0x80000000u));
    wave_order();
  };

  auto load = [&](T& t, uint32_t step) {
    const int32_t* at = rows_at(step);
#pragma unroll
    for (int i = 0; i < T::kPasses; ++i) {
      const uint32_t row = (uint32_t)at[T::kRows * i + load_row] & 0x7fffffffu;
      const char* kp = key_base + a.cache.key_offset(row);
      const char* vp = value_base + a.cache.value_offset(row);
#pragma unroll
      for (int j = 0; j < T::kLoads; ++j) t.k[i][j] = *reinterpret_cast<const u32x4*>(kp + 16 * T::kLanes * j);
#pragma unroll
      for (int j = 0; j < T::kLoads; ++j) t.v[i][j] = *reinterpret_cast<const u32x4*>(vp + 16 * T::kLanes * j);
    }
    if constexpr (kFp8) {
      const uint32_t row = (uint32_t)at[lane & 31u] & 0x7fffffffu;
      t.scale = (lane < 32u ? a.cache.key_scales : a.cache.value_scales)[(uint64_t)row * a.cache.kv_heads + g];
    }
  };

  // Both tiles to LDS, rows as they are; fp8 values widened.
  bool dropped = false;
  auto stage = [&](const T& t, uint32_t step) {
    const int32_t* at = rows_at(step);
    const uint32_t key0 = first_key(step);
    const bool hides = !kListed && key0 + kStep > all_see;  // from some row
#pragma unroll
    for (int i = 0; i < T::kPasses; ++i) {
      const uint32_t r = T::kRows * i + load_row;
      bool drop = false;
      if constexpr (kListed) drop = at[r] < 0;  // padding's weight is 0, which NaN would survive
#pragma unroll
      for (int j = 0; j < T::kLoads; ++j) {
        const uint32_t c = T::kLanes * j + load_chunk;
        *reinterpret_cast<u32x4*>(my_keys + tile_place<T::kBytes>(r, c)) = t.k[i][j];
        u32x4 v = t.v[i][j];
        if (kListed && drop) v = u32x4{0u, 0u, 0u, 0u};
        if (hides && key0 + r >= all_see) dropped |= drop_nonfinite<Tag, kFp8>(v);
        if constexpr (kFp8) {
          *reinterpret_cast<uint4*>(mine + tile_place<2 * D>(r, 2u * c)) = fp8x8_to_bf16x8_paired(make_uint2(v.x, v.y));
          *reinterpret_cast<uint4*>(mine + tile_place<2 * D>(r, 2u * c + 1u)) = fp8x8_to_bf16x8_paired(make_uint2(v.z, v.w));
        } else {
          *reinterpret_cast<u32x4*>(mine + tile_place<2 * D>(r, c)) = v;
        }
      }
    }
    if constexpr (kFp8) {
      float scale = t.scale;
      if (kListed && at[lane & 31u] < 0) scale = 0.f;
      if (hides && lane >= 32u && key0 + lane - 32u >= all_see && !is_finite(scale)) {
        scale = 0.f;
        dropped = true;
      }
      scales[wave][lane] = scale;
    }
    wave_order();
  };

  auto compute = [&](uint32_t step) {
    const int32_t* at = rows_at(step);
    // Scores of keys 16 h + 4 quad + i, in powers of two.
    float x[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < T::kBytes / 64; ++j) {
        const uint4 k = *reinterpret_cast<const uint4*>(my_keys + tile_place<T::kBytes>(16u * h + col, 4u * j + quad));
        if constexpr (kFp8) {
          s = mfma_16x16x32(Tag{}, fp8x8_to_bf16x8_paired(make_uint2(k.x, k.y)), q[2 * j], s);
          s = mfma_16x16x32(Tag{}, fp8x8_to_bf16x8_paired(make_uint2(k.z, k.w)), q[2 * j + 1], s);
        } else {
          s = mfma_16x16x32(Tag{}, k, q[j], s);
        }
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) x[4 * h + i] = s[i] * a.scale;
      if constexpr (kFp8) {
        const floatx4 ks = *reinterpret_cast<const floatx4*>(&scales[wave][16 * h + 4 * quad]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * h + i] *= ks[i];
      }
      if constexpr (kListed) {
        const int4 r = *reinterpret_cast<const int4*>(&at[16 * h + 4 * quad]);
        x[4 * h] = r.x < 0 ? -INFINITY : x[4 * h];
        x[4 * h + 1] = r.y < 0 ? -INFINITY : x[4 * h + 1];
        x[4 * h + 2] = r.z < 0 ? -INFINITY : x[4 * h + 2];
        x[4 * h + 3] = r.w < 0 ? -INFINITY : x[4 * h + 3];
      }
    }
    const uint32_t key0 = first_key(step);
    if (!kListed && key0 + kStep > min(all_see, end)) {
      const uint32_t limit = min(sees, end);
#pragma unroll
      for (int i = 0; i < 8; ++i) x[i] = key0 + 16u * (i / 4) + 4u * quad + (i % 4) < limit ? x[i] : -INFINITY;
    }
    float most = x[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) most = fmaxf(most, x[i]);
    if (__any(most > reference + (kLift + kSlack))) {
      most = fmaxf(most, __shfl_xor(most, 16, kWave));
      most = fmaxf(most, __shfl_xor(most, 32, kWave));
      const float raised = fmaxf(reference, most - kLift);
      const float shrink = exp2_fast(reference - raised);
      reference = raised;
      total *= shrink;
#pragma unroll
      for (int i = 0; i < kO; ++i) o[i] *= shrink;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = exp2_fast(x[i] - reference);
      total += x[i];
    }
    if constexpr (kFp8) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const floatx4 vs = *reinterpret_cast<const floatx4*>(&scales[wave][32 + 16 * h + 4 * quad]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[4 * h + i] *= vs[i];
      }
    }
    const uint4 p = make_uint4(pack2(Tag{}, x[0], x[1]), pack2(Tag{}, x[2], x[3]), pack2(Tag{}, x[4], x[5]),
                               pack2(Tag{}, x[6], x[7]));
#pragma unroll
    for (int i = 0; i < kO; ++i) {
      const uint2 lo = read_transposed(mine + tr_place[i]);
      const uint2 hi = read_transposed(mine + tr_place[i] + 16 * D * 2);
      o[i] = mfma_16x16x32(Tag{}, make_uint4(lo.x, lo.y, hi.x, hi.y), p, o[i]);
    }
    wave_order();
  };

  if (own > 0) {
    look_keys(0);
    look_pages();
    look_rows(0);
  }
  if (own == 1) {  // nothing to load ahead
    T tile;
    load(tile, 0);
    stage(tile, 0);
    compute(0);
  } else if (own > 1) {
    // The tiles in registers are kAhead steps on their way while LDS holds the one
    // at work; past the end they repeat the last.  Look-ups are issued ahead of a
    // step's loads, whose wait they then do not lengthen.  (No way out of the loop
    // but its end: with one after each step the compiler waits for every load in
    // flight at its head.)
    T tile[kAhead];
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) load(tile[i], min(i, own - 1u));
    for (uint32_t first = 0; first < own; first += kAhead) {
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) {
        const uint32_t step = first + i;
        const uint32_t group = step / kGroup + 1u;
        if (group * kGroup < own) {
          if (step % kGroup == 0) look_keys(group);
          if (step % kGroup == 2) look_pages();
          if (step % kGroup == 5) look_rows(group);
        }
        stage(tile[i], min(step, own - 1u));
        load(tile[i], min(step + kAhead, own - 1u));
        __builtin_amdgcn_sched_barrier(0);
        if (step < own) compute(step);
      }
    }
  }

  if (!kListed && __any(dropped)) {
    for (uint32_t k = max(begin, all_see); k < end; ++k)
      if ((k - begin) / kStep % kWaves == from && k < sees) {
        const uint32_t row = cache_row(a, pages, k);
#pragma unroll
        for (int i = 0; i < kO; ++i) {
          float back[4] = {0.f, 0.f, 0.f, 0.f};
          add_nonfinite<Tag, kFp8>(a, row, g, 16u * i + 4u * quad, back);
          o[i] += floatx4{back[0], back[1], back[2], back[3]};
        }
      }
  }

  // Join a head's waves: every wave scales its sums to the largest reference.
  total += __shfl_xor(total, 16, kWave);
  total += __shfl_xor(total, 32, kWave);
  if constexpr (kWork == kSolo) {
    if (row0 + col < rows) {
#pragma unroll
      for (int i = 0; i < kO; ++i) store_out<Tag, D>(a, out_row(0, col), 16u * i + 4u * quad, o[i], reference, total);
    }
    return;
  }
  if (quad == 0) sums[wave][col] = make_float2(reference, total);
  __syncthreads();
  const uint32_t first_wave = wave / kWaves * kWaves;
  float most = sums[first_wave][col].x;
#pragma unroll
  for (uint32_t w = 1; w < kWaves; ++w) most = fmaxf(most, sums[first_wave + w][col].x);
  const float shrink = exp2_fast(reference - most);
#pragma unroll
  for (int i = 0; i < kO; ++i)
    *reinterpret_cast<floatx4*>(mine + col * (D * 4) + (((4u * i + quad) ^ col) << 4)) = o[i] * shrink;
  __syncthreads();
  const uint32_t live = min(16u, rows - row0);
  for (uint32_t i = threadIdx.x; i < kHeads * live * (D / 4); i += kThreads) {
    const uint32_t c = i % (D / 4);
    const uint32_t h = kHeads == 1 ? 0u : i / (D / 4) / live;
    const uint32_t r = i / (D / 4) - h * live;
    const uint32_t w0 = h * kWaves;
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
    float top = sums[w0][r].x;
#pragma unroll
    for (uint32_t w = 1; w < kWaves; ++w) top = fmaxf(top, sums[w0 + w][r].x);
    float weight = 0.f;
#pragma unroll
    for (uint32_t w = 0; w < kWaves; ++w) {
      sum += *reinterpret_cast<const floatx4*>(tiles[w0 + w] + r * (D * 4) + ((c ^ r) << 4));
      weight += sums[w0 + w][r].y * exp2_fast(sums[w0 + w][r].x - top);
    }
    if (pieces == 1u) {
      store_out<Tag, D>(a, out_row(h, r), 4u * c, sum, top, weight);
    } else {
      const uint64_t at = part_at(slot + index, h, r);
      float2* to = reinterpret_cast<float2*>(a.part_out + at * D + 4u * c);
      store_shared(to, sum[0], sum[1]);
      store_shared(to + 1, sum[2], sum[3]);
      if (c == 0) store_shared(a.part_sum + at, top, weight);
    }
  }
  if (pieces == 1u) return;

  // The tile's last piece to finish joins them all, in the order of the pieces:
  // the same bits whichever it is.  The pieces are stored and loaded past the
  // XCDs' own L2s, so no cache is written back or dropped (a release and an
  // acquire of agent scope here took 140 us of a 385 us step): each wave waits for
  // its stores, the counter is raised after all four waves have, and what the
  // last workgroup loads depends on the counter it read.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t* arrived = a.arrived + (tile_slot * kinds + g0 / kHeads);
    const uint32_t before = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last_piece = before + 1u == pieces;
    if (before + 1u == pieces) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last_piece) return;

  // Four dims of a row per thread, the pieces dealt to as many groups of threads as
  // the rows leave, kPieces pieces' loads under way at a time.  (Kept short: it runs
  // once, from a cold instruction cache.)
  constexpr uint32_t kPieces = 8;
  const uint32_t cells = kHeads * live * (D / 4);
  const uint32_t groups = max(1u, kThreads / cells);
  floatx4* joined = reinterpret_cast<floatx4*>(tiles[0]);  // [kThreads]
  floatx2* joined_sum = reinterpret_cast<floatx2*>(table);  // [kThreads]
  static_assert(sizeof(tiles) >= kThreads * sizeof(floatx4) && sizeof(table) >= kThreads * sizeof(floatx2), "join");
  const uint32_t group = threadIdx.x / cells;
  for (uint32_t cell = threadIdx.x % cells; cell < cells; cell += kThreads) {
    const uint32_t h = kHeads == 1 ? 0u : cell / (D / 4) / live;
    const uint32_t r = cell / (D / 4) - h * live;
    const uint32_t dim = 4u * (cell % (D / 4));
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
    float top = kNoKeys;
    float weight = 0.f;
    auto add = [&](float reference, float w, floatx4 v) {
      const float raised = fmaxf(top, reference);
      const float keep = exp2_fast(top - raised);
      const float take = exp2_fast(reference - raised);
      sum = sum * keep + v * take;
      weight = weight * keep + w * take;
      top = raised;
    };
    for (uint32_t p = group; p < pieces && group < groups; p += groups * kPieces) {
      float2 s[kPieces], lo[kPieces], hi[kPieces];
#pragma unroll
      for (uint32_t j = 0; j < kPieces; ++j) {
        const uint64_t at = part_at(slot + min(p + groups * j, pieces - 1u), h, r);
        const float2* from = reinterpret_cast<const float2*>(a.part_out + at * D + dim);
        s[j] = load_shared(a.part_sum + at);
        lo[j] = load_shared(from);
        hi[j] = load_shared(from + 1);
      }
#pragma unroll
      for (uint32_t j = 0; j < kPieces; ++j)
        if (p + groups * j < pieces) add(s[j].x, s[j].y, floatx4{lo[j].x, lo[j].y, hi[j].x, hi[j].y});
    }
    if (groups > 1u) {  // then one round of cells takes every thread
      joined[threadIdx.x] = sum;
      joined_sum[threadIdx.x] = floatx2{top, weight};
      __syncthreads();
      if (group > 0) return;
      for (uint32_t i = 1; i < groups; ++i) {
        const floatx2 s = joined_sum[i * cells + cell];
        add(s[0], s[1], joined[i * cells + cell]);
      }
    }
    if (group == 0) store_out<Tag, D>(a, out_row(h, r), dim, sum, top, weight);
  }
}

// The chunk kernel's pieces of each (token, head) row, four dims a thread:
// references to their maximum, sums and outputs scaled to it and added in the
// order of the pieces.  (A workgroup per row took 38 us for 30000 rows of two
// pieces of 64 dims, which this reads in 5.)
template <class Tag, int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedAttentionArgs a) {
  constexpr uint32_t kLanes = D / 4;
  const uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  const uint64_t row = at / kLanes;
  const uint32_t dim = 4u * (uint32_t)(at % kLanes);
  if (row >= (uint64_t)a.tokens * a.heads) return;
  if (a.starts) {  // a mixed batch: the stream kernel's rows are not in these pieces
    const uint32_t token = (uint32_t)(row / a.heads);
    uint32_t low = 0, high = a.sequences;  // the last sequence that starts at or before the token
    while (high - low > 1u) {
      const uint32_t mid = (low + high) / 2u;
      if (a.starts[mid] <= (int32_t)token) low = mid; else high = mid;
    }
    const Span span = tokens_of(a, low);
    if (token - span.first >= span.count || span.count * a.group < a.least_rows) return;
  }
  // A token outside every sequence has no entry here (a batch padded to a fixed number
  // of tokens), nor has one of `starts` that fall: what stands there is not an index.
  const uint2 of = a.part_of[row];
  const uint32_t apart = a.cache.kv_heads * a.part_rows;
  if (of.y < 2u || of.y > kMostSplits || of.x + (uint64_t)(of.y - 1u) * apart >= a.parts) return;
  const float2* sums = a.part_sum + of.x;
  const float* parts = a.part_out + (uint64_t)of.x * D + dim;
  floatx4 sum = {0.f, 0.f, 0.f, 0.f};
  float top = kNoKeys;
  float total = 0.f;
#pragma unroll 4
  for (uint32_t p = 0; p < of.y; ++p) {
    const float2 s = sums[p * apart];
    const floatx4 v = *reinterpret_cast<const floatx4*>(parts + (uint64_t)p * apart * D);
    const float raised = fmaxf(top, s.x);
    const float keep = exp2_fast(top - raised);
    const float take = exp2_fast(s.x - raised);
    sum = sum * keep + v * take;
    total = total * keep + s.y * take;
    top = raised;
  }
  store_out<Tag, D>(a, row, dim, sum, top, total);
}

template <class Tag, bool kFp8, int D, Work kWork>
void launch_stream_of(const PagedAttentionArgs& a, uint32_t grid, hipStream_t s) {
  if constexpr (kWork != kBeside || Tile<kFp8, D>::kBytes == 128)
    hipLaunchKernelGGL((paged_stream_kernel<Tag, kFp8, D, kWork>), dim3(grid), dim3(256 * kHeadsOf<kWork>), 0, s, a);
}

template <class Tag, bool kFp8, Work kWork>
void launch_stream(const PagedAttentionArgs& a, int32_t dim, uint32_t grid, hipStream_t s) {
  if (dim == 64)
    launch_stream_of<Tag, kFp8, 64, kWork>(a, grid, s);
  else if (dim == 128)
    launch_stream_of<Tag, kFp8, 128, kWork>(a, grid, s);
  else
    launch_stream_of<Tag, kFp8, 256, kWork>(a, grid, s);
}

template <class Tag>
void launch_combine(const PagedAttentionArgs& a, int32_t dim, hipStream_t s) {
  const dim3 grid((unsigned)(((uint64_t)a.tokens * a.heads * (dim / 4) + 255) / 256));
  if (dim == 64)
    hipLaunchKernelGGL((paged_combine_kernel<Tag, 64>), grid, dim3(256), 0, s, a);
  else if (dim == 128)
    hipLaunchKernelGGL((paged_combine_kernel<Tag, 128>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((paged_combine_kernel<Tag, 256>), grid, dim3(256), 0, s, a);
}

int combine(const PagedAttentionArgs& a, int32_t dim, int32_t dtype, hipStream_t s) {
  if (dtype == kBF16)
    launch_combine<Bf16Tag>(a, dim, s);
  else
    launch_combine<F16Tag>(a, dim, s);
  return check_launch("paged_combine_kernel");
}

template <Work kWork>
int launch(const PagedAttentionArgs& a, const dsa_paged_cache* cache, int32_t dtype, int64_t pieces, hipStream_t s) {
  const int64_t grid = pieces * (a.cache.kv_heads / kHeadsOf<kWork>);
  DSA_REQUIRE(grid < (1LL << 31), "too many tokens for one call");
  const int32_t dim = cache->head_dim;
  if (cache->dtype == kFP8E4M3)
    launch_stream<Bf16Tag, true, kWork>(a, dim, (uint32_t)grid, s);
  else if (dtype == kBF16)
    launch_stream<Bf16Tag, false, kWork>(a, dim, (uint32_t)grid, s);
  else
    launch_stream<F16Tag, false, kWork>(a, dim, (uint32_t)grid, s);
  return check_launch("paged_stream_kernel");
}

// Pieces of each row's keys: enough for `want` workgroups, none of fewer than
// `least` keys.
uint32_t splits_for(int64_t workgroups, int64_t want, int64_t most_keys, int64_t least) {
  const int64_t enough = (want + workgroups - 1) / workgroups;
  const int64_t most = (most_keys + least - 1) / least;
  const int64_t splits = enough < most ? enough : most;
  return (uint32_t)(splits < 1 ? 1 : splits > kMostSplits ? kMostSplits : splits);
}

// Tiles of `size` rows over all sequences: each sequence's last one may be partial.
int64_t row_tiles(int64_t sequences, int64_t tokens, int64_t group, bool uniform, int64_t size) {
  if (uniform) return sequences * ((tokens / sequences * group + size - 1) / size);
  const int64_t most = tokens < sequences ? tokens : sequences;  // sequences that have tokens
  return (tokens * group + (size - 1) * most) / size;
}

int check_common(const dsa_paged_cache* cache, const void* queries, int64_t query_stride, const int32_t* page_table,
                 int64_t table_stride, int64_t columns, const int32_t* lengths, const int32_t* starts,
                 int64_t sequences, int64_t tokens, int32_t heads, int32_t dtype, float scale, const void* out,
                 PagedAttentionArgs& a) {
  if (int st = make_paged_view(cache, a.cache)) return st;
  DSA_REQUIRE(sequences > 0 && sequences <= (1 << 20) && tokens >= 0 && tokens < (1LL << 28), "sequences/tokens out of range");
  DSA_REQUIRE(queries && page_table && lengths && out, "null pointer argument");
  DSA_REQUIRE(heads > 0 && heads <= 65536 && heads % cache->kv_heads == 0, "%d heads do not share %d kv heads evenly",
              heads, cache->kv_heads);
  DSA_REQUIRE(dtype == kBF16 || dtype == kF16, "queries are bf16 or fp16 (got %d)", dtype);
  DSA_REQUIRE(dtype == (cache->dtype == kFP8E4M3 ? kBF16 : cache->dtype),
              "queries must have the cache's type (bf16 for an fp8 cache)");
  DSA_REQUIRE(starts || tokens % sequences == 0, "without starts every sequence has as many tokens");
  DSA_REQUIRE(columns > 0 && columns < (1LL << 31) && columns * cache->page_size <= (1LL << 30) && table_stride >= columns,
              "page table of %lld columns out of range", (long long)columns);
  DSA_REQUIRE(query_stride >= (int64_t)heads * cache->head_dim && query_stride % 8 == 0,
              "query_stride must cover the heads and be a multiple of 8");
  DSA_REQUIRE(reinterpret_cast<uintptr_t>(queries) % 16 == 0 && reinterpret_cast<uintptr_t>(out) % 16 == 0,
              "queries and outputs must be 16-byte aligned");
  a.queries = static_cast<const char*>(queries);
  a.query_stride = query_stride * 2;
  a.page_table = page_table;
  a.table_stride = table_stride;
  a.columns = (uint32_t)columns;
  a.lengths = lengths;
  a.starts = starts;
  a.sequences = (uint32_t)sequences;
  a.tokens = (uint32_t)tokens;
  a.heads = (uint32_t)heads;
  a.group = (uint32_t)(heads / cache->kv_heads);
  a.scale = scale * kLog2E;
  return 0;
}

constexpr int64_t kStreamRows = 16;  // most rows of a sequence that the stream kernel takes

// Workspace: the counters, at one place for every shape, then `parts` outputs,
// their sums and where `rows` rows have theirs.
int64_t part_bytes(int64_t parts, int64_t rows, int64_t dim) {
  return parts ? kCounters * 4 + parts * (dim + 2) * 4 + rows * 8 : 0;
}

int take_workspace(PagedAttentionArgs& a, int64_t parts, int64_t rows, int64_t dim, void* workspace, int64_t bytes) {
  if (parts == 0) return 0;
  if (!workspace || bytes < part_bytes(parts, rows, dim) || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(DSA_STATUS_WORKSPACE_TOO_SMALL, "paged attention needs %lld bytes of 16-byte aligned workspace",
                (long long)part_bytes(parts, rows, dim));
  a.arrived = static_cast<uint32_t*>(workspace);
  a.part_out = reinterpret_cast<float*>(a.arrived + kCounters);
  a.part_sum = reinterpret_cast<float2*>(a.part_out + parts * dim);
  a.part_of = reinterpret_cast<uint2*>(a.part_sum + parts);
  a.parts = (uint32_t)parts;
  return 0;
}

// Which kernels a call runs, and what it cuts.
struct Plan {
  uint32_t stream_cuts, stream_rows;  // rows of a part
  uint32_t stream_most;               // rows of a sequence of the stream kernel's
  bool stream_beside;                 // it takes heads side by side
  int64_t stream_pieces;              // at most; 0: no sequence of few rows
  bool prefill;                       // the prefill kernel takes the other sequences, else the chunk kernel
  int32_t chunk_rows;                 // of a tile of theirs
  uint32_t chunk_cuts;                // 0: more row tiles than could be cut to use
  uint32_t chunk_whole;               // row tiles that are not cut all the same
  int64_t chunk_pieces;
  int64_t parts, rows;
};

// Whether the stream kernel takes two heads a workgroup: heads of 128 bytes that lie
// side by side, from 128 MiB of cache on.  The lengths are the GPU's, so the page
// table's room stands for them: short sequences in wide tables take this form too, at
// the cost that the figures of one sequence show.  HBM serves 256 contiguous bytes that one
// workgroup asks for together faster than two requests of 128 at different times
// (fp8 of 128 dims read at 4.6 TB/s, with a head's rows contiguous at 5.6); a cache
// that the last-level cache holds is not bound by that, and eight waves a workgroup
// start and join later.  (us, four waves / eight, 8 kv heads: fp8 of 128 dims, 4
// sequences of up to 128K keys 178 / 160, 16 of 32K 239 / 212, 64 of 4K 119 / 107,
// one of 32K, 67 MB, 27 / 32; 16-bit of 64 dims, 16 of 32K 212 / 191, 64 of 4K 122 /
// 98, one of 32K 23 / 20; 2 kv heads of fp8, 64 of 4K, 128 MiB, 32 / 32, one of 32K
// 25 / 35.  Heads of 64 bytes, fp8 of 64 dims, lose more by two waves a SIMD instead of
// three: 16 of 32K 136 / 178.)
bool heads_lie_beside(const dsa_paged_cache* cache, int64_t sequences, int64_t capacity) {
  return cache->head_dim * (cache->dtype == kFP8E4M3 ? 1 : 2) == 128 && cache->kv_heads % 2 == 0 &&
         cache->key_head_stride == cache->head_dim && cache->value_head_stride == cache->head_dim &&
         sequences * capacity * cache->kv_heads >= 1LL << 19;
}

Plan dense_plan(const dsa_paged_cache* cache, int64_t sequences, int64_t tokens, int64_t heads, int64_t capacity,
                bool uniform) {
  const int64_t kv_heads = cache->kv_heads;
  const int64_t group = heads / kv_heads;
  Plan p = {};
  uniform |= sequences == 1;  // whose starts are 0 and tokens
  const int64_t each = tokens / sequences * group;
  auto at_most = [&](int64_t tiles, int64_t cuts, int64_t least) {
    const int64_t pieces = tiles * ((capacity + least - 1) / least);
    return pieces < tiles + cuts ? pieces : tiles + cuts;
  };
  // Where only `starts` says how the tokens are dealt and there are no more of them
  // than sequences, this is a decode step, and the stream kernel takes it all, some
  // sequence of several tokens in several row tiles: two launches less.  (us, with /
  // without the others' launches, 32 heads on 8 of 128 dims: 64 sequences of 4K keys,
  // bf16 192 / 186, fp8 126 / 119; 16 of 2K 34 / 27, 26 / 21; but 16 tokens of one
  // sequence of 32K and none of 15 others 43 / 68, 43 / 38: that sequence's keys are
  // read once for each 16 rows, and more tokens of it cost more.)
  const bool few = !uniform && tokens <= sequences;
  if (!uniform || each <= kStreamRows) {
    p.stream_beside = heads_lie_beside(cache, sequences, capacity);
    const int64_t kinds = p.stream_beside ? kv_heads / 2 : kv_heads;
    const int64_t fill = p.stream_beside ? 256 : resident_workgroups(cache->head_dim);
    const int64_t cuts = (fill + kinds - 1) / kinds;
    const int64_t tiles = (tokens < sequences ? tokens : sequences) + (few ? tokens * group / kStreamRows : 0);
    p.stream_most = few ? 0xffffffffu : kStreamRows;
    p.stream_cuts = (uint32_t)cuts;
    p.stream_rows = (uint32_t)(uniform ? each : kStreamRows);
    p.stream_pieces = at_most(tiles, cuts, kLeastSteps * kStep);
    p.parts = 2 * cuts * kv_heads * p.stream_rows;
  }
  if (uniform ? each > kStreamRows : !few) {
    // The prefill kernel from more than 128 rows a sequence on, the chunk kernel, of
    // half its rows a workgroup and two or three workgroups a CU, below; head_dim 256
    // has the prefill kernel alone.  (us, chunk / prefill kernel, 32 heads on 8 of
    // 128 dims, 64K keys: 64 rows 71 / 73, 128 rows 78 / 76, 256 rows 114 / 99, 2048
    // rows 646 / 553; 8K keys: 128 rows 25.5 / 28.0, 256 rows 34.9 / 36.3; fp8, 64K:
    // 128 rows 73 / 90, 256 rows 110 / 106; head_dim 256, 64K: 20 rows 118 / 74.)
    p.prefill = cache->head_dim == 256 || tokens * group > 128 * sequences;
    p.chunk_rows = p.prefill ? prefill_rows(cache->head_dim) : kChunkRows;
    const int64_t fill = p.prefill ? 256 : resident_workgroups(cache->head_dim);
    const int64_t cuts = (fill + kv_heads - 1) / kv_heads;
    const int64_t tiles = row_tiles(sequences, tokens, group, uniform, p.chunk_rows);
    // One sequence: row tiles that fill the GPU some times over are not cut, those
    // left over are, but for most of a prompt from its start, whose last tiles to run
    // are its shortest.  (us, all whole / the rest cut, 32 heads on 8 of 128 dims, 32K
    // keys, 32 tiles at a time: 33 tiles 1590 / 977, 48 1593 / 1411, 65 2459 / 1818, 136
    // 3957 / 3538, 258 6087 / 6064; of 8K keys 65 472 / 395, 80, 5120 tokens, 471 / 483,
    // 104 505 / 542.)
    const int64_t rest = tiles % cuts;
    const bool cut = sequences == 1 && tiles >= cuts
                         ? rest > 0 && tiles < 8 * cuts && (tiles < 2 * cuts || 8 * tokens <= 5 * capacity)
                         : tiles < 2 * cuts;
    if (!cut) {
      p.chunk_pieces = tiles;
    } else {
      p.chunk_cuts = (uint32_t)cuts;
      if (sequences == 1 && tiles >= cuts) {
        p.chunk_whole = (uint32_t)(tiles - rest);
        p.chunk_pieces = tiles - rest + (cuts > rest ? cuts : rest);
      } else {
        p.chunk_pieces = at_most(tiles, cuts, kLeastChunkKeys);
      }
      p.rows = tokens * heads;
      if (p.parts < 2 * cuts * kv_heads * p.chunk_rows) p.parts = 2 * cuts * kv_heads * p.chunk_rows;
    }
  }
  return p;
}

struct SelectedPlan {
  int64_t items;
  uint32_t splits, part_rows;
  bool solo;
  int64_t parts;
};

SelectedPlan selected_plan(const dsa_paged_cache* cache, int64_t tokens, int64_t heads, int64_t k) {
  const int64_t kv_heads = cache->kv_heads;
  const int64_t group = heads / kv_heads;
  const int64_t items = tokens * ((group + 15) / 16);
  SelectedPlan p = {items, splits_for(items * kv_heads, resident_workgroups(cache->head_dim), k,
                                     kLeastSteps * kStep), (uint32_t)(group < 16 ? group : 16), false, 0};
  // A list to a wave, once they give every wave that runs at a time one: no joining
  // of waves, and four times the steps for a start.  (Lists of 512 of bf16, 8 kv
  // heads, us, by waves / by workgroups: 128 tokens 24.0 / 23.6, 256 33.5 / 42.9,
  // 1024 118 / 151; of 2048: 82 / 61, 114 / 116, 426 / 449.)
  p.solo = items * kv_heads >= 4 * resident_workgroups(cache->head_dim);
  if (p.splits > 1) p.parts = items * p.splits * kv_heads * p.part_rows;
  return p;
}

bool sizes_valid(const dsa_paged_cache* c, int64_t sequences, int64_t tokens, int32_t heads) {
  return c && c->kv_heads > 0 && c->head_dim > 0 && heads > 0 && heads % c->kv_heads == 0 && sequences > 0 && tokens > 0;
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int64_t dsa_paged_attention_workspace_bytes(const dsa_paged_cache* cache, int64_t sequences, int64_t tokens,
                                                       int32_t heads, int64_t columns, int32_t uniform) {
  if (!sizes_valid(cache, sequences, tokens, heads)) return 0;
  const Plan p = dense_plan(cache, sequences, tokens, heads, columns * cache->page_size, uniform != 0);
  return part_bytes(p.parts, p.rows, cache->head_dim);
}

extern "C" int dsa_paged_attention(const dsa_paged_cache* cache, const void* queries, int64_t query_stride,
                                   const int32_t* page_table, int64_t table_stride, int64_t columns,
                                   const int32_t* lengths, const int32_t* starts, int64_t sequences, int64_t tokens,
                                   int32_t heads, int32_t dtype, float scale, int32_t causal, void* out, float* lse,
                                   void* workspace, int64_t workspace_bytes, void* stream) {
  PagedAttentionArgs a = {};
  if (int st = check_common(cache, queries, query_stride, page_table, table_stride, columns, lengths, starts, sequences,
                            tokens, heads, dtype, scale, out, a))
    return st;
  if (tokens == 0) return 0;
  const Plan p = dense_plan(cache, sequences, tokens, heads, columns * cache->page_size, !starts);
  a.causal = causal != 0;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  // A sequence of few rows (one decoded token, a few drafted ones) is bound by
  // reading its cache, one of many by the products: a mixed batch has both.
  if (int st = take_workspace(a, p.parts, p.rows, cache->head_dim, workspace, workspace_bytes)) return st;
  if (p.stream_pieces) {
    a.cuts = p.stream_cuts;
    a.part_rows = p.stream_rows;
    a.least_rows = 1;
    a.most_rows = p.stream_most;
    a.clears = starts != nullptr;
    const auto launch_stream = p.stream_beside ? launch<kBeside> : launch<kDense>;
    if (int st = launch_stream(a, cache, dtype, (p.stream_pieces + kXcds - 1) / kXcds * kXcds, s)) return st;
  }
  if (p.chunk_pieces) {
    a.cuts = p.chunk_cuts;
    a.whole = p.chunk_whole;
    a.part_rows = (uint32_t)p.chunk_rows;
    a.least_rows = p.stream_pieces ? kStreamRows + 1 : 1;  // fewer: the stream kernel's, if it ran
    a.most_rows = 0xffffffffu;
    a.clears = starts && !p.stream_pieces;
    const int64_t grid = p.chunk_pieces * a.cache.kv_heads;
    DSA_REQUIRE(grid < (1LL << 31), "too many tokens for one call");
    const auto launch_rows = p.prefill ? launch_paged_prefill : launch_paged_chunk;
    if (int st = launch_rows(a, cache->head_dim, cache->dtype, (uint32_t)grid, s)) return st;
    if (p.chunk_cuts) return combine(a, cache->head_dim, dtype, s);
  }
  return 0;
}

extern "C" int64_t dsa_paged_selected_workspace_bytes(const dsa_paged_cache* cache, int64_t tokens, int32_t heads,
                                                      int64_t k) {
  if (!sizes_valid(cache, 1, tokens, heads)) return 0;
  const SelectedPlan p = selected_plan(cache, tokens, heads, k);
  return part_bytes(p.parts, 0, cache->head_dim);
}

extern "C" int dsa_paged_selected_attention(const dsa_paged_cache* cache, const void* queries, int64_t query_stride,
                                            const int32_t* page_table, int64_t table_stride, int64_t columns,
                                            const int32_t* lengths, const int32_t* starts, int64_t sequences,
                                            int64_t tokens, int32_t heads, int32_t dtype, const int64_t* indices,
                                            int64_t index_stride, int64_t k, float scale, void* out, float* lse,
                                            void* workspace, int64_t workspace_bytes, void* stream) {
  PagedAttentionArgs a = {};
  if (int st = check_common(cache, queries, query_stride, page_table, table_stride, columns, lengths, starts, sequences,
                            tokens, heads, dtype, scale, out, a))
    return st;
  DSA_REQUIRE(k >= 0 && k < (1LL << 31) - 64 && (indices || k == 0) && index_stride >= k, "index lists of %lld out of range",
              (long long)k);
  if (tokens == 0) return 0;
  const SelectedPlan p = selected_plan(cache, tokens, heads, k);
  a.splits = p.splits;
  a.part_rows = p.part_rows;
  a.indices = indices;
  a.index_stride = index_stride;
  a.k = (uint32_t)k;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  if (int st = take_workspace(a, p.parts, 0, cache->head_dim, workspace, workspace_bytes)) return st;
  if (p.solo) return launch<kSolo>(a, cache, dtype, (p.items + 3) / 4, static_cast<hipStream_t>(stream));
  return launch<kSelected>(a, cache, dtype, p.items * p.splits, static_cast<hipStream_t>(stream));
}
