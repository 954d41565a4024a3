// The softmax weights that each cached key has of a batch's newest tokens.
//
//   w_j += sum over the rows (tokens and heads of the key's kv head) that see key j of
//          exp(scale q . k_j - lse)
//
// The rows' log sums are known, so a score needs no other one: one product, one fused
// multiply-add, one exponential and one sum, and no maximum.  A wave keeps 16 kSets
// keys in registers, the A operand of v_mfma_f32_16x16x32, and its keys' sums beside
// them; the rows pass by as the B operand, from LDS, where a workgroup's four waves
// share them.  A lane's scores are all of one row, whose log sum is one register, and
// the 16 lanes of a key add theirs once, at the end.
//
// That is the kernel of many rows, bound by the exponentials and the products (prompt of
// 4096 tokens over as many 4-bit keys, 32 heads on 8, 78 us, 84 where its inputs are in
// no cache).  Where the keys are too few workgroups for them, the rows are cut into
// pieces, whose sums a second kernel adds in order (5 us).  Few rows (a decoded token) are bound by reading the
// keys: there the rows stay, in LDS, and the keys pass by, loaded a step ahead.
//
// Which of the two takes a sequence is known to the device alone where `starts` says how
// many tokens each has.  There the kernel of few rows also lists the sequences that it
// leaves to the other, which deals its workgroups to what is listed.
#include <algorithm>

#include "paged_attention.hpp"
#include "waveops.hpp"

namespace dsa {
namespace {

constexpr uint32_t kStage = 64;  // rows in LDS at a time
constexpr int64_t kManyWorkgroups = 2048;  // that the work is dealt to, where there is as much
// The same for few rows, two a CU, each then of up to 32 steps in turn: a start and an end
// cost as much as some steps.  (us, dealt to 256 / 512 / 1024 / 2048: one sequence of 32K
// bf16 keys, 8 heads of 128 dims, 16.6 / 16.8 / 19.9 / 25.0, 16 of 4096 4-bit ones 18.6 /
// 15.4 / 16.4 / 18.8; 16 of 32K bf16 keys, which have more steps than that, 218 to 220.)
constexpr int64_t kFewWorkgroups = 512;
constexpr uint32_t kMostSteps = 32;

// Sequences of many rows among some of few.
struct Chunks {
  uint32_t count, tiles, pieces;  // sequences, their tiles of keys, pieces of each tile's rows
  uint32_t unused;
  uint2 of[1];  // {sequence, tiles before it}
};

struct WeightArgs {
  PagedAttentionArgs batch;
  Quotient by_group;  // of a row: its token
  float* weights;     // [kv_heads][cache rows]
  float* parts;       // of several pieces: [sequences][kv_heads][share][keys of a tile]
  // Workgroups of each sequence and kv head: what there is work for (its tiles of keys are
  // cut into that many pieces of rows, or spread over as many workgroups), and how many
  // there are, which a sequence of more takes in turn.
  uint32_t share, slots;
  uint32_t few_share, few_slots;
  Chunks* chunks;     // of a mixed batch; else all sequences are one kernel's
  uint64_t row_count;
};

__device__ __forceinline__ float* weights_of(const WeightArgs& a, uint32_t g) { return a.weights + g * a.row_count; }

// The sum over the 16 lanes of a row, in each of them.
__device__ __forceinline__ float row16_sum(float v) {
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x128, 0xf, 0xf, false));  // row_ror:8
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x124, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x122, 0xf, 0xf, false));
  v += __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(v), 0x121, 0xf, 0xf, false));
  return v;
}

// Adds to a weight.  (An atomic, since sequences may share a page; else each weight is
// added to once.)
__device__ __forceinline__ void add_weight(const WeightArgs& a, const int32_t* pages, uint32_t g, uint32_t key, float v) {
  __hip_atomic_fetch_add(weights_of(a, g) + cache_row(a.batch, pages, key), v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

constexpr int kSets = 4;  // of 16 keys, of a wave
constexpr uint32_t kTile = 4 * 16 * kSets;  // keys of a workgroup

// What a workgroup does to one tile of a sequence's keys: piece `piece` of `pieces` of its
// rows, whose sums go to `parts` if there are several.
template <class Tag, Store kStore, int D>
__device__ __forceinline__ void weigh_tile(const WeightArgs& w, uint32_t g, uint32_t sequence, uint32_t tile, uint32_t piece,
                                           uint32_t pieces, float* parts) {
  const PagedAttentionArgs& a = w.batch;
  constexpr bool kFp8 = kStore == kE4M3;
  constexpr bool kFp4 = kStore == kE2M1;
  constexpr int kQ = D / 32;               // products of a tile of scores
  constexpr uint32_t kKeys = 16 * kSets;   // of a wave
  constexpr uint32_t kRow = 2 * D + 16;    // bytes of a row in LDS
  constexpr uint32_t kRuns = D / 8;        // 16-byte runs of a row
  constexpr uint32_t kLoads = kStage * kRuns / 256;
  __shared__ __attribute__((aligned(16))) char rows_tile[2][kStage * kRow];
  // {log2 sum, keys that the row sees (as bits)}.  A row whose log sum is -inf has no weight
  // to give, also to keys that it sees (their scores are all -inf then): it sees none here.
  __shared__ float2 row_of[2][kStage];
  const uint32_t tid = threadIdx.x, lane = lane_id(), wave = tid / kWave, col = lane & 15u, quad = lane >> 4;

  const uint32_t length = keys_of(a, sequence);
  const uint32_t tile0 = tile * 4u * kKeys;
  if (tile0 >= length) return;
  const Span span = tokens_of(a, sequence);
  // This piece's rows, from those on that see the tile's first key.
  const int64_t before = (int64_t)length - span.count;  // keys that token 0 sees, less its own
  const uint32_t first = a.causal ? (uint32_t)min((int64_t)span.count, max((int64_t)0, (int64_t)tile0 - before)) : 0u;
  const uint32_t rows_all = (span.count - first) * a.group;
  const uint32_t each = ((rows_all + pieces - 1u) / pieces + kStage - 1u) / kStage * kStage;
  const uint32_t begin = min(piece * each, rows_all), end = min(begin + each, rows_all);
  const uint32_t key0 = tile0 + wave * kKeys;
  const int32_t* pages = a.page_table + (int64_t)sequence * a.table_stride;

  float sum[kSets][4];
#pragma unroll
  for (int s = 0; s < kSets; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[s][i] = 0.f;

  if (begin < end) {
    // A stage's rows.  Where whole tokens fill it and it ends within the sequence, a
    // thread's places are the same in every stage, past a base that all threads share;
    // else each row's token and head are worked out (for every stage that was 15 % more
    // vector instructions, 28.0 and 24.4 million a prompt of 4096).
    const char* base = a.queries + (int64_t)(span.first + first) * a.query_stride + (uint64_t)g * a.group * D * 2u;
    const float* base_lse = a.lse + (uint64_t)(span.first + first) * a.heads + g * a.group;
    const bool whole = kStage % a.group == 0;
    uint64_t place[kLoads];
#pragma unroll
    for (uint32_t i = 0; i < kLoads; ++i) {
      const uint32_t at = tid + 256u * i, t = w.by_group(at / kRuns);
      place[i] = (uint64_t)t * a.query_stride + ((at / kRuns - t * a.group) * D + at % kRuns * 8u) * 2u;
    }
    u32x4 staged[kLoads];
    float2 staged_of;
    auto load = [&](uint32_t r0) {
      const uint32_t t0 = w.by_group(r0);
      if (whole && r0 + kStage <= rows_all) {
        const char* from = base + (int64_t)t0 * a.query_stride;
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) staged[i] = *reinterpret_cast<const u32x4*>(from + place[i]);
      } else {
#pragma unroll
        for (uint32_t i = 0; i < kLoads; ++i) {
          const uint32_t at = tid + 256u * i, r = min(r0 + at / kRuns, rows_all - 1u), t = w.by_group(r);
          staged[i] = *reinterpret_cast<const u32x4*>(base + (int64_t)t * a.query_stride + ((r - t * a.group) * D + at % kRuns * 8u) * 2u);
        }
      }
      if (tid < kStage) {
        const uint32_t r = min(r0 + tid, rows_all - 1u), t = w.by_group(r);
        const int64_t sees = a.causal ? before + first + t + 1 : (int64_t)length;
        const float lse = base_lse[(uint64_t)t * a.heads + (r - t * a.group)];
        staged_of = make_float2(lse * kLog2E, __uint_as_float(r0 + tid < end && lse != -INFINITY ? (uint32_t)max((int64_t)0, sees) : 0u));
      }
    };
    auto stage = [&](uint32_t slot) {
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) {
        const uint32_t at = tid + 256u * i;
        *reinterpret_cast<u32x4*>(rows_tile[slot] + at / kRuns * kRow + at % kRuns * 16u) = staged[i];
      }
      if (tid < kStage) row_of[slot][tid] = staged_of;
    };
    load(begin);
    __builtin_amdgcn_sched_barrier(0);  // under way before the keys are waited for
    // This wave's keys.  A lane has of key 16 s + col the dims that its quarter of each
    // product takes; the order of the dims is the store's.
    uint4 k[kSets][kQ];
    float by[kFp8 ? kSets : 1][4];
#pragma unroll
    for (int s = 0; s < kSets; ++s) {
      const uint32_t row = cache_row(a, pages, min(key0 + 16u * s + col, length - 1u));
      const char* from = a.cache.keys + g * a.cache.key_head + a.cache.key_offset(row);
      if constexpr (kFp4) {
        const uint8_t* powers = a.cache.key_powers + a.cache.power_offset<D>(row, g);
        uint32_t codes[kQ];
        if constexpr (D == 64) {
          const uint2 v = *reinterpret_cast<const uint2*>(from + 8u * quad);
          codes[0] = v.x, codes[1] = v.y;
        } else {
#pragma unroll
          for (int i = 0; i < D / 128; ++i) {
            const uint4 v = *reinterpret_cast<const uint4*>(from + D / 8u * quad + 16u * i);
            codes[4 * i] = v.x, codes[4 * i + 1] = v.y, codes[4 * i + 2] = v.z, codes[4 * i + 3] = v.w;
          }
        }
#pragma unroll
        for (int j = 0; j < kQ; ++j) k[s][j] = fp4x8_to_bf16x8(codes[j], power_of(powers[(D / 4u * quad + 8u * j) / kPowerDims]));
      } else if constexpr (kFp8) {
#pragma unroll
        for (int j = 0; j < kQ / 2; ++j) {
          const uint4 v = *reinterpret_cast<const uint4*>(from + 64u * j + 16u * quad);
          k[s][2 * j] = fp8x8_to_bf16x8_paired(make_uint2(v.x, v.y));
          k[s][2 * j + 1] = fp8x8_to_bf16x8_paired(make_uint2(v.z, v.w));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const uint32_t of = cache_row(a, pages, min(key0 + 16u * s + 4u * quad + i, length - 1u));
          by[s][i] = a.scale * a.cache.key_scales[(uint64_t)of * a.cache.kv_heads + g];
        }
      } else {
#pragma unroll
        for (int j = 0; j < kQ; ++j) k[s][j] = *reinterpret_cast<const uint4*>(from + 64u * j + 16u * quad);
      }
    }

    // Row sub + col of a stage, in the order of dims that the keys have.
    auto read_row = [&](uint32_t slot, uint32_t sub, uint4 (&q)[kQ]) {
      const char* row = rows_tile[slot] + (sub + col) * kRow;
#pragma unroll
      for (int j = 0; j < kQ; ++j) {
        const uint32_t d = kFp4   ? D / 4u * quad + 8u * j
                           : kFp8 ? 64u * (j / 2) + 16u * quad + 8u * (j % 2)
                                  : 32u * j + 8u * quad;
        q[j] = *reinterpret_cast<const uint4*>(row + 2u * d);
      }
    };
    auto multiply = [&](const uint4 (&q)[kQ], floatx4 (&x)[kSets]) {
#pragma unroll
      for (int j = 0; j < kQ; ++j)
#pragma unroll
        for (int s = 0; s < kSets; ++s)
          x[s] = mfma_16x16x32(Tag{}, k[s][j], q[j], j == 0 ? floatx4{0.f, 0.f, 0.f, 0.f} : x[s]);
    };
    stage(0);
    __syncthreads();
    uint32_t slot = 0;
    for (uint32_t r0 = begin; r0 < end; r0 += kStage, slot ^= 1u) {
      const bool more = r0 + kStage < end;
      if (more) load(r0 + kStage);
      static_assert(kStage == kWave, "a lane a row");
      if (__all(__float_as_uint(row_of[slot][lane].y) >= key0 + kKeys)) {
        // Every row sees every key: the products of 16 rows under the exponentials of
        // the 16 before, operands read from LDS a turn ahead.
        constexpr uint32_t kTurns = kStage / 16u;
        constexpr int kProducts = kSets * kQ;
        uint4 q[2][kQ];
        floatx4 x[2][kSets];
        float lse[2];
        read_row(slot, 0, q[0]);
        float last = 0.f;  // a weight that is added a product later: an exponential's result has to wait
#pragma unroll
        for (uint32_t n = 0; n <= kTurns; ++n) {
          if (n + 1u < kTurns) read_row(slot, 16u * (n + 1u), q[(n + 1) % 2]);
          if (n < kTurns) lse[n % 2] = row_of[slot][16u * n + col].x;  // for the next turn
          __builtin_amdgcn_sched_barrier(0);
#pragma unroll
          for (int m = 0; m < kProducts; ++m) {
            const int j = m / kSets, s = m % kSets;
            if (n < kTurns)
              x[n % 2][s] = mfma_16x16x32(Tag{}, k[s][j], q[n % 2][j], j == 0 ? floatx4{0.f, 0.f, 0.f, 0.f} : x[n % 2][s]);
            if (n > 0) {
#pragma unroll
              for (int e = 4 * kSets * m / kProducts; e < 4 * kSets * (m + 1) / kProducts; ++e) {
                const float p = exp2_fast(fmaf(x[(n + 1) % 2][e / 4][e % 4], kFp8 ? by[kFp8 ? e / 4 : 0][e % 4] : a.scale, -lse[(n + 1) % 2]));
                const int before_e = e == 0 ? 4 * kSets - 1 : e - 1;
                sum[before_e / 4][before_e % 4] += last;
                last = p;
              }
            }
            __builtin_amdgcn_sched_barrier(0);
          }
        }
        sum[kSets - 1][3] += last;
      } else {
        for (uint32_t sub = 0; sub < kStage && r0 + sub < end; sub += 16u) {
          const float2 of = row_of[slot][sub + col];
          const uint32_t sees = __float_as_uint(of.y);
          if (!__any(sees > key0)) continue;  // these rows see none of the wave's keys
          uint4 q[kQ];
          floatx4 x[kSets];
          read_row(slot, sub, q);
          multiply(q, x);
#pragma unroll
          for (int s = 0; s < kSets; ++s)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              const float p = exp2_fast(fmaf(x[s][i], kFp8 ? by[kFp8 ? s : 0][i] : a.scale, -of.x));
              sum[s][i] += key0 + 16u * s + 4u * quad + i < sees ? p : 0.f;
            }
        }
      }
      if (more) stage(slot ^ 1u);
      __syncthreads();
    }
  }

  // The 16 lanes of a key, each in turn over its four neighbours, then one lane a key.
#pragma unroll
  for (int s = 0; s < kSets; ++s) {
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[s][i] = row16_sum(sum[s][i]);
    if (col < 4u) {
      const float v = col == 0 ? sum[s][0] : col == 1 ? sum[s][1] : col == 2 ? sum[s][2] : sum[s][3];
      const uint32_t key = key0 + 16u * s + 4u * quad + col;
      if (pieces > 1u) {
        parts[key - tile0] = v;
      } else if (key < length && begin < end) {
        add_weight(w, pages, g, key, v);
      }
    }
  }
}

// How a sequence's work is cut where it has w.share workgroups: by its own keys, whatever
// the page table has room for.
struct Cut {
  uint32_t tiles, pieces;  // of each tile's rows
};
__device__ __forceinline__ Cut cut_of(const WeightArgs& w, uint32_t sequence) {
  const uint32_t tiles = (keys_of(w.batch, sequence) + kTile - 1u) / kTile;
  const uint32_t rows = tokens_of(w.batch, sequence).count * w.batch.group;
  return {tiles, max(1u, min(w.share / max(tiles, 1u), (rows + 4u * kStage - 1u) / (4u * kStage)))};
}

// Heads vary fastest, then pieces, then tiles: a causal chunk's first keys, which most
// rows see, come first.
template <class Tag, Store kStore, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_weights_kernel(WeightArgs w) {
  const uint32_t heads = w.batch.cache.kv_heads;
  uint32_t id = blockIdx.x;
  const uint32_t g = id % heads;
  id /= heads;
  const uint32_t sequence = id % w.batch.sequences;
  const Cut cut = cut_of(w, sequence);
  for (uint32_t item = id / w.batch.sequences; item < cut.tiles * cut.pieces; item += w.slots)
    weigh_tile<Tag, kStore, D>(w, g, sequence, item / cut.pieces, item % cut.pieces, cut.pieces,
                               w.parts + (((uint64_t)sequence * heads + g) * w.share + item) * kTile);
}

// A listed sequence's tile.
struct ChunkTile {
  uint32_t sequence, tile;
};
__device__ __forceinline__ ChunkTile chunk_tile(const Chunks* chunks, uint32_t at) {
  const uint2 of = chunks->of[last_at_most(chunks->of, chunks->count, at)];
  return {of.x, at - of.y};
}

// The same for the listed sequences of a mixed batch, dealt to the workgroups in turn.
template <class Tag, Store kStore, int D>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_weights_chunks_kernel(WeightArgs w) {
  const uint32_t heads = w.batch.cache.kv_heads;
  const uint32_t pieces = w.chunks->pieces, all = w.chunks->tiles * heads * pieces;
  for (uint32_t item = blockIdx.x; item < all; item += gridDim.x) {
    uint32_t id = item;
    const uint32_t g = id % heads;
    id /= heads;
    const uint32_t piece = id % pieces;
    id /= pieces;
    const ChunkTile t = chunk_tile(w.chunks, id);
    weigh_tile<Tag, kStore, D>(w, g, t.sequence, t.tile, piece, pieces, w.parts + (((uint64_t)id * heads + g) * pieces + piece) * kTile);
  }
}

// Lists the sequences of more than kStage rows, and cuts their tiles' rows into as many
// pieces as leave every workgroup some.  One workgroup's work.
__device__ __forceinline__ void list_chunks(const WeightArgs& w, uint32_t* scan) {
  const PagedAttentionArgs& a = w.batch;
  uint32_t count = 0, tiles = 0, most = 0;
  for (uint32_t base = 0; base < a.sequences; base += 256u) {
    const uint32_t sequence = base + threadIdx.x;
    uint32_t own = 0, rows = 0;
    if (sequence < a.sequences) {
      rows = tokens_of(a, sequence).count * a.group;
      if (rows > kStage) own = (keys_of(a, sequence) + kTile - 1u) / kTile;
    }
    uint32_t all, all_tiles;
    const uint32_t rank = block_excl_scan<4>(own > 0u ? 1u : 0u, scan, all);
    const uint32_t before = block_excl_scan<4>(own, scan + 4, all_tiles);
    if (own > 0) w.chunks->of[count + rank] = make_uint2(sequence, tiles + before);
    most = max(most, own > 0 ? rows : 0u);
    count += all, tiles += all_tiles;
    __syncthreads();
  }
  if (threadIdx.x == 0) scan[0] = 0;
  __syncthreads();
  if (most) atomicMax(scan, most);
  __syncthreads();
  if (threadIdx.x > 0) return;
  const uint32_t wide = tiles * a.cache.kv_heads;
  uint32_t pieces = 1;
  if (wide > 0) pieces = min(((uint32_t)kManyWorkgroups + wide - 1u) / wide, (scan[0] + 4u * kStage - 1u) / (4u * kStage));
  w.chunks->count = count;
  w.chunks->tiles = tiles;
  w.chunks->pieces = pieces;
}

// Few rows: those of a sequence, up to kStage, lie in LDS while its keys pass by, 32 a wave and step,
// loaded as 128 neighbouring bytes by eight lanes, through LDS of the wave's own.  A
// workgroup takes up to kMostSteps steps of each of its four waves, and more in turn.  A wave has 16 KiB of keys on
// their way, whatever their type (16 sequences of 32K bf16 keys: 217 us; 227 with 8 KiB, 220 with 16 in one run), and
// nothing that the steps wait for is loaded after them: cache rows are looked up a group
// of steps ahead, a row's powers of two come with it.
template <class Tag, Store kStore, int D>
__global__ __launch_bounds__(256, D == 256 && kStore == k16Bit ? 1 : 2) void paged_weights_few_kernel(WeightArgs w) {
  const PagedAttentionArgs& a = w.batch;
  constexpr bool kFp8 = kStore == kE4M3;
  constexpr bool kFp4 = kStore == kE2M1;
  constexpr int kQ = D / 32;
  constexpr uint32_t kStep = 32;
  constexpr uint32_t kGroup = 8;                              // steps that are looked up at a time
  constexpr uint32_t kRow = 2 * D + 16;                       // bytes of a row in LDS
  constexpr uint32_t kRuns = D / 8;
  constexpr int kBytes = kRowBytes<kStore, D>;                // of a key
  constexpr uint32_t kAhead = kBytes >= 512 ? 1 : kBytes >= 256 ? 2 : 4;  // steps on their way
  constexpr uint32_t kLanes = kBytes < 128 ? kBytes / 16 : 8;  // that share a key
  constexpr uint32_t kRows = 64 / kLanes;                     // of one load
  constexpr int kPasses = kStep / kRows;
  constexpr int kLoads = kBytes / (16 * kLanes);              // of one key
  constexpr uint32_t kKeyRow = kBytes + 16;
  constexpr int kPowerWords = D == 256 ? 2 : 1;
  __shared__ __attribute__((aligned(16))) char rows_tile[kStage * kRow];
  __shared__ float2 row_of[kStage];
  __shared__ __attribute__((aligned(16))) char key_tile[4][kStep * kKeyRow];
  __shared__ uint32_t table[4][2][kGroup * kStep];            // a wave's cache rows of this group of steps and the next
  const uint32_t tid = threadIdx.x, lane = lane_id(), wave = tid / kWave, col = lane & 15u, quad = lane >> 4;

  uint32_t id = blockIdx.x;
  if (w.chunks) {
    if (id == 0) {
      list_chunks(w, reinterpret_cast<uint32_t*>(rows_tile));
      return;
    }
    --id;
  }
  const uint32_t g = id % a.cache.kv_heads;
  id /= a.cache.kv_heads;
  const uint32_t sequence = id % a.sequences;
  const uint32_t length = keys_of(a, sequence);
  // Neighbouring steps a workgroup, as many as its share of the sequence.
  const uint32_t most = min(max((length + 4u * kStep * w.few_share - 1u) / (4u * kStep * w.few_share), 1u), kMostSteps);
  uint32_t tile0 = id / a.sequences * (4u * kStep * most);
  if (tile0 >= length) return;
  const Span span = tokens_of(a, sequence);
  const int64_t before = (int64_t)length - span.count;
  const uint32_t rows = span.count * a.group;
  if (rows == 0 || rows > kStage) return;  // (more: listed)
  const int32_t* pages = a.page_table + (int64_t)sequence * a.table_stride;
  uint32_t steps;
  const uint32_t load_row = lane / kLanes, load_chunk = lane % kLanes;
  const char* key_base = a.cache.keys + g * a.cache.key_head + 16u * load_chunk;
  auto first_key = [&](uint32_t step) { return tile0 + (4u * step + wave) * kStep; };

  struct Tile {
    u32x4 k[kPasses][kLoads];
    float scale;                  // e4m3: of key `lane`
    uint32_t power[kPowerWords];  // e2m1: of key `lane`
  };
  // Lane l looks up keys l % 32 of steps 2 j + l / 32 of a group; past the end, the last.
  uint32_t page[kGroup / 2];
  auto key_at = [&](uint32_t group, uint32_t j) {
    return min(first_key(group * kGroup + 2u * j + lane / 32u) + lane % 32u, length - 1u);
  };
  auto look = [&](uint32_t group) {
#pragma unroll
    for (uint32_t j = 0; j < kGroup / 2; ++j) page[j] = (uint32_t)pages[key_at(group, j) >> a.cache.shift];
  };
  auto place = [&](uint32_t group) {
#pragma unroll
    for (uint32_t j = 0; j < kGroup / 2; ++j)
      table[wave][group % 2u][64u * j + lane] =
          (min(page[j], a.cache.pages - 1u) << a.cache.shift) | (key_at(group, j) & ((1u << a.cache.shift) - 1u));
    wave_order();
  };
  auto rows_at = [&](uint32_t step) { return table[wave][step / kGroup % 2u] + step % kGroup * kStep; };
  auto load = [&](Tile& t, uint32_t step) {
    const uint32_t* at = rows_at(step);
#pragma unroll
    for (int i = 0; i < kPasses; ++i) {
      const char* from = key_base + a.cache.key_offset(at[kRows * i + load_row]);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) t.k[i][j] = *reinterpret_cast<const u32x4*>(from + 16 * kLanes * j);
    }
    if constexpr (kFp8) t.scale = a.cache.key_scales[(uint64_t)at[lane & 31u] * a.cache.kv_heads + g];
    if constexpr (kFp4) {
      const uint8_t* powers = a.cache.key_powers + a.cache.power_offset<D>(at[lane & 31u], g);
      if constexpr (D == 64) {
        t.power[0] = *reinterpret_cast<const uint16_t*>(powers);
      } else {
#pragma unroll
        for (int i = 0; i < kPowerWords; ++i) t.power[i] = reinterpret_cast<const uint32_t*>(powers)[i];
      }
    }
  };

  auto compute = [&](uint32_t step, float scale, const uint32_t (&power)[kPowerWords]) {
    const char* mine = key_tile[wave];
    const uint32_t key0 = first_key(step);
    uint4 k[2][kQ];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const char* key = mine + (16u * h + col) * kKeyRow;
      if constexpr (kFp4) {
        uint32_t of[kPowerWords];
#pragma unroll
        for (int i = 0; i < kPowerWords; ++i) of[i] = (uint32_t)__shfl((int)power[i], 16 * h + col, kWave);
        // this lane's quarter of the key's blocks: half a block, one, or two
        const uint32_t mine_of = D == 256 ? (quad < 2u ? of[0] : of[kPowerWords - 1]) : of[0];
        const uint32_t at = D == 64 ? quad / 2u : D == 128 ? quad : 2u * (quad & 1u);
#pragma unroll
        for (int j = 0; j < kQ; ++j)
          k[h][j] = fp4x8_to_bf16x8(*reinterpret_cast<const uint32_t*>(key + D / 8u * quad + 4u * j),
                                    power_of(mine_of >> 8u * (at + j / 4) & 0xffu));
      } else if constexpr (kFp8) {
#pragma unroll
        for (int j = 0; j < kQ / 2; ++j) {
          const uint4 v = *reinterpret_cast<const uint4*>(key + 64u * j + 16u * quad);
          k[h][2 * j] = fp8x8_to_bf16x8_paired(make_uint2(v.x, v.y));
          k[h][2 * j + 1] = fp8x8_to_bf16x8_paired(make_uint2(v.z, v.w));
        }
      } else {
#pragma unroll
        for (int j = 0; j < kQ; ++j) k[h][j] = *reinterpret_cast<const uint4*>(key + 64u * j + 16u * quad);
      }
    }
    float by[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) by[e] = kFp8 ? __shfl(scale, 16 * (e / 4) + 4 * quad + e % 4, kWave) * a.scale : a.scale;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    for (uint32_t sub = 0; sub < rows; sub += 16u) {
      const char* from = rows_tile + (sub + col) * kRow;
      const float2 of = row_of[sub + col];
      const uint32_t sees = __float_as_uint(of.y);
      floatx4 x[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
      for (int j = 0; j < kQ; ++j) {
        const uint32_t d = kFp4   ? D / 4u * quad + 8u * j
                           : kFp8 ? 64u * (j / 2) + 16u * quad + 8u * (j % 2)
                                  : 32u * j + 8u * quad;
        const uint4 q = *reinterpret_cast<const uint4*>(from + 2u * d);
        x[0] = mfma_16x16x32(Tag{}, k[0][j], q, x[0]);
        x[1] = mfma_16x16x32(Tag{}, k[1][j], q, x[1]);
      }
      const bool partly = __any(sees < key0 + kStep);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float p = exp2_fast(fmaf(x[e / 4][e % 4], by[e], -of.x));
        if (partly) p = key0 + 16u * (e / 4) + 4u * quad + e % 4 < sees ? p : 0.f;
        sum[e] += p;
      }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[e] = row16_sum(sum[e]);
    if (col < 8u) {
      float v = sum[0];
#pragma unroll
      for (int e = 1; e < 8; ++e) v = col == (uint32_t)e ? sum[e] : v;
      const uint32_t of = 16u * (col / 4u) + 4u * quad + col % 4u;  // the key that this lane adds to
      if (key0 + of < length)
        __hip_atomic_fetch_add(weights_of(w, g) + rows_at(step)[of], v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    wave_order();
  };
  for (bool first = true; tile0 < length; first = false, tile0 += w.few_slots * (4u * kStep * most)) {
    steps = min(most, (length - tile0 + 4u * kStep - 1u) / (4u * kStep));
    Tile t[kAhead];
    look(0);
    place(0);
#pragma unroll
    for (uint32_t i = 0; i < kAhead; ++i) load(t[i], min(i, steps - 1u));
    if (first) {
      for (uint32_t at = tid; at < rows * kRuns; at += 256u) {
        const uint32_t r = at / kRuns;
        const uint32_t i = w.by_group(r);
        *reinterpret_cast<u32x4*>(rows_tile + r * kRow + at % kRuns * 16u) =
            *reinterpret_cast<const u32x4*>(a.queries + (int64_t)(span.first + i) * a.query_stride +
                                            ((uint64_t)(g * a.group + r - i * a.group) * D + at % kRuns * 8u) * 2u);
      }
      if (tid < kStage) {
        const uint32_t r = min(tid, rows - 1u);
        const uint32_t i = w.by_group(r);
        const int64_t sees = a.causal ? before + i + 1 : (int64_t)length;
        const float lse = a.lse[(uint64_t)(span.first + i) * a.heads + g * a.group + r - i * a.group];
        row_of[tid] = make_float2(lse * kLog2E, __uint_as_float(tid < rows && lse != -INFINITY ? (uint32_t)max((int64_t)0, sees) : 0u));
      }
      __syncthreads();
    }
    for (uint32_t step0 = 0; step0 < steps; step0 += kAhead) {
#pragma unroll
      for (uint32_t i = 0; i < kAhead; ++i) {
        const uint32_t step = step0 + i;
        const uint32_t group = step / kGroup + 1u;
        if (group * kGroup < steps) {
          if (step % kGroup == 0) look(group);
          if (step % kGroup == 3) place(group);
        }
        char* mine = key_tile[wave];
#pragma unroll
        for (int p = 0; p < kPasses; ++p)
#pragma unroll
          for (int j = 0; j < kLoads; ++j)
            *reinterpret_cast<u32x4*>(mine + (kRows * p + load_row) * kKeyRow + (kLanes * j + load_chunk) * 16u) = t[i].k[p][j];
        const float scale = t[i].scale;
        uint32_t power[kPowerWords];
#pragma unroll
        for (int p = 0; p < kPowerWords; ++p) power[p] = t[i].power[p];
        wave_order();
        load(t[i], min(step + kAhead, steps - 1u));
        __builtin_amdgcn_sched_barrier(0);
        if (step < steps) compute(step, scale, power);
      }
    }
  }
}

// Adds the pieces of each key, a key a thread: of a batch's tiles, or of the listed
// sequences'.
__global__ __launch_bounds__(kTile) void paged_weights_join_kernel(WeightArgs w) {
  const PagedAttentionArgs& a = w.batch;
  const uint32_t heads = a.cache.kv_heads;
  const uint32_t g = blockIdx.x % heads, at = blockIdx.x / heads;
  uint32_t sequence, tile, pieces;
  uint64_t part;
  if (w.chunks) {
    pieces = w.chunks->pieces;
    if (pieces == 1u || at >= w.chunks->tiles) return;
    const ChunkTile t = chunk_tile(w.chunks, at);
    sequence = t.sequence, tile = t.tile;
    part = ((uint64_t)at * heads + g) * pieces;
  } else {
    sequence = at % a.sequences, tile = at / a.sequences;
    const Cut cut = cut_of(w, sequence);
    pieces = cut.pieces;
    if (pieces == 1u || tile >= cut.tiles) return;
    part = ((uint64_t)sequence * heads + g) * w.share + tile * pieces;
  }
  const uint32_t key = tile * kTile + threadIdx.x;
  if (key >= keys_of(a, sequence)) return;
  const float* from = w.parts + part * kTile + threadIdx.x;
  float sum = 0.f;
#pragma unroll 4
  for (uint32_t p = 0; p < pieces; ++p) sum += from[(uint64_t)p * kTile];
  add_weight(w, a.page_table + (int64_t)sequence * a.table_stride, g, key, sum);
}

struct WeightPlan {
  bool few, mixed;
  int64_t share, slots, few_share, few_slots;
  int64_t pieces;  // of a tile's rows, at most
  int64_t chunk_workgroups, list_bytes, part_bytes;
  int64_t bytes() const { return list_bytes + part_bytes; }
};

WeightPlan weight_plan(const dsa_paged_cache* cache, int64_t sequences, int64_t tokens, int64_t heads, int64_t capacity,
                       bool uniform) {
  const int64_t group = heads / cache->kv_heads, pairs = sequences * cache->kv_heads;
  WeightPlan p = {};
  // With `starts` each sequence has the kernel of its own rows.  (us, so / as a call for the
  // single tokens and one for the others, 32 heads on 8 of 128 dims, bf16: 256 tokens over
  // 4096 keys each and a chunk of 2048 over as many 509 / 433 + 75; 8 over 32K and a prompt
  // of 4096 203 / 110 + 95.  A batch that has no single tokens pays for the list: 4 x 150
  // tokens over 4096 keys each 49, without `starts` 46; 4 prompts of 150 19 and 15.)
  p.mixed = !uniform && sequences > 1 && tokens * group > kStage;
  p.few = p.mixed || tokens * group <= kStage * sequences;
  // Workgroups by what keeps the GPU busy; for sequences of more keys than that has tiles
  // for, as many as the page table's room asks for, while their starts cost little.  What
  // each does follows from the keys that its sequence has.  (Prompt of 4096 tokens, bf16,
  // in a table with room for 128K keys: 95 us as in one without, and 365 cut by the room.)
  const int64_t tiles = (capacity + kTile - 1) / kTile;
  auto slots = [&](int64_t share, int64_t of_room) {
    return std::max(share, std::min(of_room, 4 * kManyWorkgroups / pairs));
  };
  if (p.few) {
    p.few_share = (kFewWorkgroups + pairs - 1) / pairs;
    p.few_slots = std::min(slots(p.few_share, (2 * tiles + kMostSteps - 1) / kMostSteps), 2 * tiles);
  }
  if (p.mixed) {
    // What can be listed: sequences of more than kStage rows, pieces of 4 kStage each.
    const int64_t listed = std::min(sequences, tokens * group / (kStage + 1));
    p.pieces = std::min(kManyWorkgroups, (tokens * group + 4 * kStage - 1) / (4 * kStage));
    // (12 sequences of 240 rows over 116K keys of 64 dims, 5460 tiles, by 2048 workgroups
    // 115 us, by 4096 109; nothing listed, no difference.)
    p.chunk_workgroups = std::min(2 * kManyWorkgroups, listed * tiles * cache->kv_heads * p.pieces);
    p.list_bytes = (16 + sequences * 8 + 15) / 16 * 16;
    if (p.pieces > 1) p.part_bytes = 2 * kManyWorkgroups * kTile * 4;  // several pieces are fewer than twice the workgroups
  } else if (!p.few) {
    // As many pieces of every tile's rows, a causal tile's fewer rows in shorter ones:
    // the longest come first, and the short ones fill what they leave.  (Prompt of 4096
    // tokens over as many 4-bit keys, 32 heads on 8, us: 16 pieces a tile 92, 8 98;
    // pieces of one length, twice or four times what runs at a time, 120 and 108.)
    const int64_t rows = tokens / sequences * group;  // of a sequence: all have as many, or there is one
    p.share = (kManyWorkgroups + pairs - 1) / pairs;
    p.slots = slots(p.share, tiles);
    p.pieces = std::min(p.share, (rows + 4 * kStage - 1) / (4 * kStage));
    if (p.pieces > 1) p.part_bytes = pairs * p.share * kTile * 4;
  }
  return p;
}

template <class Tag, Store kStore, int D>
void launch_dim(const WeightArgs& w, uint32_t grid, uint32_t chunk_grid, hipStream_t s) {
  if (w.chunks) {
    hipLaunchKernelGGL((paged_weights_few_kernel<Tag, kStore, D>), dim3(grid + 1u), dim3(256), 0, s, w);
    hipLaunchKernelGGL((paged_weights_chunks_kernel<Tag, kStore, D>), dim3(chunk_grid), dim3(256), 0, s, w);
  } else if (w.few_share)
    hipLaunchKernelGGL((paged_weights_few_kernel<Tag, kStore, D>), dim3(grid), dim3(256), 0, s, w);
  else
    hipLaunchKernelGGL((paged_weights_kernel<Tag, kStore, D>), dim3(grid), dim3(256), 0, s, w);
}

template <class Tag, Store kStore>
void launch_weights(const WeightArgs& w, int32_t dim, uint32_t grid, uint32_t chunk_grid, hipStream_t s) {
  if (dim == 64)
    launch_dim<Tag, kStore, 64>(w, grid, chunk_grid, s);
  else if (dim == 128)
    launch_dim<Tag, kStore, 128>(w, grid, chunk_grid, s);
  else
    launch_dim<Tag, kStore, 256>(w, grid, chunk_grid, s);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int64_t dsa_paged_weights_workspace_bytes(const dsa_paged_cache* cache, int64_t sequences, int64_t tokens,
                                                     int32_t heads, int64_t columns, int32_t uniform) {
  if (!cache || cache->kv_heads <= 0 || heads <= 0 || heads % cache->kv_heads || sequences <= 0 || tokens <= 0 ||
      columns <= 0 || cache->page_size <= 0)
    return 0;
  return weight_plan(cache, sequences, tokens, heads, columns * cache->page_size, uniform != 0).bytes();
}

extern "C" int dsa_paged_weights(const dsa_paged_cache* cache, const void* queries, int64_t query_stride,
                                 const int32_t* page_table, int64_t table_stride, int64_t columns,
                                 const int32_t* lengths, const int32_t* starts, int64_t sequences, int64_t tokens,
                                 int32_t heads, int32_t dtype, float scale, int32_t causal, const float* lse,
                                 float* weights, void* workspace, int64_t workspace_bytes, void* stream) {
  WeightArgs w = {};
  if (int st = check_paged_batch(cache, queries, query_stride, page_table, table_stride, columns, lengths, starts,
                                 sequences, tokens, heads, dtype, scale, queries, w.batch))
    return st;
  DSA_REQUIRE(lse && weights, "null pointer argument");
  if (tokens == 0) return 0;
  DSA_REQUIRE(tokens * w.batch.group < (1LL << 31), "too many rows for one call");
  const int64_t capacity = columns * cache->page_size;
  const WeightPlan p = weight_plan(cache, sequences, tokens, heads, capacity, !starts);
  if (p.bytes() && (!workspace || workspace_bytes < p.bytes() || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(DSA_STATUS_WORKSPACE_TOO_SMALL, "paged weights need %lld bytes of 16-byte aligned workspace",
                (long long)p.bytes());
  w.by_group = quotient_by(w.batch.group);
  w.batch.causal = causal != 0;
  w.batch.lse = const_cast<float*>(lse);
  w.weights = weights;
  w.chunks = p.mixed ? static_cast<Chunks*>(workspace) : nullptr;
  w.parts = reinterpret_cast<float*>(static_cast<char*>(workspace) + p.list_bytes);
  w.share = (uint32_t)p.share;
  w.slots = (uint32_t)p.slots;
  w.few_share = (uint32_t)p.few_share;
  w.few_slots = (uint32_t)p.few_slots;
  w.row_count = (uint64_t)cache->pages * cache->page_size;
  const int64_t pairs = sequences * cache->kv_heads;
  const int64_t grid = pairs * (p.few ? p.few_slots : p.slots);
  DSA_REQUIRE(grid < (1LL << 24), "too many sequences for one call");
  DSA_REQUIRE((capacity + kTile - 1) / kTile * pairs < (1LL << 30), "too many keys for one call");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->dtype == kFP4E2M1)
    launch_weights<Bf16Tag, kE2M1>(w, cache->head_dim, (uint32_t)grid, (uint32_t)p.chunk_workgroups, s);
  else if (cache->dtype == kFP8E4M3)
    launch_weights<Bf16Tag, kE4M3>(w, cache->head_dim, (uint32_t)grid, (uint32_t)p.chunk_workgroups, s);
  else if (cache->dtype == kBF16)
    launch_weights<Bf16Tag, k16Bit>(w, cache->head_dim, (uint32_t)grid, (uint32_t)p.chunk_workgroups, s);
  else
    launch_weights<F16Tag, k16Bit>(w, cache->head_dim, (uint32_t)grid, (uint32_t)p.chunk_workgroups, s);
  if (int st = check_launch("paged_weights_kernel")) return st;
  if (p.pieces <= 1) return 0;
  // A workgroup a tile and head that has several pieces.
  const int64_t join = p.mixed ? kManyWorkgroups : pairs * (p.share / 2);
  hipLaunchKernelGGL(paged_weights_join_kernel, dim3((unsigned)join), dim3(kTile), 0, s, w);
  return check_launch("paged_weights_join_kernel");
}
