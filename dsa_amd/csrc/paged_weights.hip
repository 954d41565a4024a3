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
// Few rows (a decoded token) are bound by reading the keys, many by the exponentials
// and the products.  Where the keys are too few workgroups for many rows, the rows are
// cut into pieces, whose sums a second kernel adds in order.
#include "paged_attention.hpp"

namespace dsa {
namespace {

constexpr uint32_t kStage = 64;  // rows in LDS at a time
constexpr int64_t kManyWorkgroups = 2048;  // that rows are cut for: about four rounds of what runs at a time

struct WeightArgs {
  PagedAttentionArgs batch;
  float* weights;     // [kv_heads][cache rows]
  float* parts;       // of several pieces: [sequences][kv_heads][pieces][tiles * keys of a tile]
  uint32_t tiles;     // of keys, of the longest sequence that the page table has room for
  uint32_t pieces;    // of each tile's rows
  uint64_t row_count;
};

// Adds to a weight.  (An atomic, since sequences may share a page; else each weight is
// added to once.)
__device__ __forceinline__ void add_weight(const WeightArgs& a, const int32_t* pages, uint32_t g, uint32_t key, float v) {
  float* to = a.weights + g * a.row_count + cache_row(a.batch, pages, key);
  __hip_atomic_fetch_add(to, v, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

template <class Tag, Store kStore, int D, int kSets>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_weights_kernel(WeightArgs w) {
  const PagedAttentionArgs& a = w.batch;
  constexpr bool kFp8 = kStore == kE4M3;
  constexpr bool kFp4 = kStore == kE2M1;
  constexpr int kQ = D / 32;               // products of a tile of scores
  constexpr uint32_t kKeys = 16 * kSets;   // of a wave
  constexpr uint32_t kRow = 2 * D + 16;    // bytes of a row in LDS
  constexpr uint32_t kRuns = D / 8;        // 16-byte runs of a row
  constexpr uint32_t kLoads = kStage * kRuns / 256;
  __shared__ __attribute__((aligned(16))) char rows_tile[2][kStage * kRow];
  __shared__ float2 row_of[2][kStage];     // {log2 sum, keys that the row sees (as bits)}
  const uint32_t tid = threadIdx.x, lane = lane_id(), wave = tid / kWave, col = lane & 15u, quad = lane >> 4;

  // Heads vary fastest, then pieces, then tiles: a causal chunk's first keys, which
  // most rows see, come first.
  uint32_t id = blockIdx.x;
  const uint32_t g = id % a.cache.kv_heads;
  id /= a.cache.kv_heads;
  const uint32_t piece = id % w.pieces;
  id /= w.pieces;
  const uint32_t sequence = id % a.sequences;
  const uint32_t tile = id / a.sequences;
  const uint32_t length = keys_of(a, sequence);
  const uint32_t tile0 = tile * 4u * kKeys;
  if (tile0 >= length) return;
  const Span span = tokens_of(a, sequence);
  // The first token that sees the tile's first key, and this piece's rows from there on.
  const int64_t before = (int64_t)length - span.count;  // keys that token 0 sees, less its own
  const uint32_t first = a.causal ? (uint32_t)min((int64_t)span.count, max((int64_t)0, (int64_t)tile0 - before)) : 0u;
  const uint32_t rows_all = (span.count - first) * a.group;
  const uint32_t each = ((rows_all + w.pieces - 1u) / w.pieces + kStage - 1u) / kStage * kStage;
  const uint32_t begin = min(piece * each, rows_all), end = min(begin + each, rows_all);
  const uint32_t key0 = tile0 + wave * kKeys;
  const int32_t* pages = a.page_table + (int64_t)sequence * a.table_stride;

  float sum[kSets][4];
#pragma unroll
  for (int s = 0; s < kSets; ++s)
#pragma unroll
    for (int i = 0; i < 4; ++i) sum[s][i] = 0.f;

  if (begin < end) {
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

    uint4 staged[kLoads];
    float2 staged_of;
    auto load = [&](uint32_t r0) {
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) {
        const uint32_t at = tid + 256u * i;
        const uint32_t r = min(r0 + at / kRuns, end - 1u);
        const uint64_t token = span.first + first + r / a.group;
        staged[i] = *reinterpret_cast<const uint4*>(a.queries + (int64_t)token * a.query_stride +
                                                    ((uint64_t)(g * a.group + r % a.group) * D + at % kRuns * 8u) * 2u);
      }
      if (tid < kStage) {
        const uint32_t r = min(r0 + tid, end - 1u);
        const uint32_t t = first + r / a.group;
        const int64_t sees = a.causal ? before + t + 1 : (int64_t)length;
        const float lse = a.lse[(uint64_t)(span.first + t) * a.heads + g * a.group + r % a.group];
        staged_of = make_float2(lse * kLog2E, __uint_as_float(r0 + tid < end ? (uint32_t)max((int64_t)0, sees) : 0u));
      }
    };
    auto stage = [&](uint32_t slot) {
#pragma unroll
      for (uint32_t i = 0; i < kLoads; ++i) {
        const uint32_t at = tid + 256u * i;
        *reinterpret_cast<uint4*>(rows_tile[slot] + at / kRuns * kRow + at % kRuns * 16u) = staged[i];
      }
      if (tid < kStage) row_of[slot][tid] = staged_of;
    };
    load(begin);
    stage(0);
    __syncthreads();
    uint32_t slot = 0;
    for (uint32_t r0 = begin; r0 < end; r0 += kStage, slot ^= 1u) {
      const bool more = r0 + kStage < end;
      if (more) load(r0 + kStage);
      for (uint32_t sub = 0; sub < kStage && r0 + sub < end; sub += 16u) {
        const char* row = rows_tile[slot] + (sub + col) * kRow;
        const float2 of = row_of[slot][sub + col];
        const uint32_t sees = __float_as_uint(of.y);
        floatx4 x[kSets];
#pragma unroll
        for (int s = 0; s < kSets; ++s) x[s] = floatx4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int j = 0; j < kQ; ++j) {
          const uint32_t d = kFp4   ? D / 4u * quad + 8u * j
                             : kFp8 ? 64u * (j / 2) + 16u * quad + 8u * (j % 2)
                                    : 32u * j + 8u * quad;
          const uint4 q = *reinterpret_cast<const uint4*>(row + 2u * d);
#pragma unroll
          for (int s = 0; s < kSets; ++s) x[s] = mfma_16x16x32(Tag{}, k[s][j], q, x[s]);
        }
        const bool partly = __any(sees < key0 + kKeys);
#pragma unroll
        for (int s = 0; s < kSets; ++s)
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float p = exp2_fast(fmaf(x[s][i], kFp8 ? by[kFp8 ? s : 0][i] : a.scale, -of.x));
            if (partly) p = key0 + 16u * s + 4u * quad + i < sees ? p : 0.f;
            sum[s][i] += p;
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
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int off = 1; off < 16; off <<= 1) sum[s][i] += __shfl_xor(sum[s][i], off, kWave);
    if (col < 4u) {
      const float v = col == 0 ? sum[s][0] : col == 1 ? sum[s][1] : col == 2 ? sum[s][2] : sum[s][3];
      const uint32_t key = key0 + 16u * s + 4u * quad + col;
      if (w.pieces > 1u) {
        w.parts[(((uint64_t)sequence * a.cache.kv_heads + g) * w.pieces + piece) * (w.tiles * 4u * kKeys) + key] = v;
      } else if (key < length && begin < end) {
        add_weight(w, pages, g, key, v);
      }
    }
  }
}

// Adds the pieces of each key, a key a thread.
__global__ __launch_bounds__(256) void paged_weights_join_kernel(WeightArgs w, uint32_t keys) {
  const PagedAttentionArgs& a = w.batch;
  const uint32_t key = blockIdx.x * 256u + threadIdx.x;
  const uint32_t g = blockIdx.y, sequence = blockIdx.z;
  if (key >= keys_of(a, sequence)) return;
  const float* from = w.parts + ((uint64_t)sequence * a.cache.kv_heads + g) * w.pieces * keys + key;
  float sum = 0.f;
  for (uint32_t p = 0; p < w.pieces; ++p) sum += from[(uint64_t)p * keys];
  add_weight(w, a.page_table + (int64_t)sequence * a.table_stride, g, key, sum);
}

struct WeightPlan {
  int sets;
  int64_t tiles, pieces, part_bytes;
};

WeightPlan weight_plan(const dsa_paged_cache* cache, int64_t sequences, int64_t tokens, int64_t heads, int64_t capacity,
                       bool uniform) {
  const int64_t group = heads / cache->kv_heads;
  const int64_t rows = (uniform ? tokens / sequences : tokens) * group;  // of a sequence, at most
  WeightPlan p = {};
  const int64_t wide = (capacity + 255) / 256 * cache->kv_heads * sequences;
  p.sets = rows <= 64 && wide < 512 ? 1 : 4;
  p.tiles = (capacity + 64 * p.sets - 1) / (64 * p.sets);
  const int64_t most = (rows + 4 * kStage - 1) / (4 * kStage);
  p.pieces = (kManyWorkgroups + wide - 1) / wide;
  if (p.pieces > most) p.pieces = most;
  if (p.pieces < 1) p.pieces = 1;
  if (p.pieces > 1) p.part_bytes = sequences * cache->kv_heads * p.pieces * p.tiles * 64 * p.sets * 4;
  return p;
}

template <class Tag, Store kStore, int kSets>
void launch_weights(const WeightArgs& w, int32_t dim, uint32_t grid, hipStream_t s) {
  if (dim == 64)
    hipLaunchKernelGGL((paged_weights_kernel<Tag, kStore, 64, kSets>), dim3(grid), dim3(256), 0, s, w);
  else if (dim == 128)
    hipLaunchKernelGGL((paged_weights_kernel<Tag, kStore, 128, kSets>), dim3(grid), dim3(256), 0, s, w);
  else
    hipLaunchKernelGGL((paged_weights_kernel<Tag, kStore, 256, kSets>), dim3(grid), dim3(256), 0, s, w);
}

template <int kSets>
void launch_weights(const WeightArgs& w, const dsa_paged_cache* cache, uint32_t grid, hipStream_t s) {
  if (cache->dtype == kFP4E2M1)
    launch_weights<Bf16Tag, kE2M1, kSets>(w, cache->head_dim, grid, s);
  else if (cache->dtype == kFP8E4M3)
    launch_weights<Bf16Tag, kE4M3, kSets>(w, cache->head_dim, grid, s);
  else if (cache->dtype == kBF16)
    launch_weights<Bf16Tag, k16Bit, kSets>(w, cache->head_dim, grid, s);
  else
    launch_weights<F16Tag, k16Bit, kSets>(w, cache->head_dim, grid, s);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int64_t dsa_paged_weights_workspace_bytes(const dsa_paged_cache* cache, int64_t sequences, int64_t tokens,
                                                     int32_t heads, int64_t columns, int32_t uniform) {
  if (!cache || cache->kv_heads <= 0 || heads <= 0 || heads % cache->kv_heads || sequences <= 0 || tokens <= 0 ||
      columns <= 0 || cache->page_size <= 0)
    return 0;
  return weight_plan(cache, sequences, tokens, heads, columns * cache->page_size, uniform != 0).part_bytes;
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
  const int64_t capacity = columns * cache->page_size;
  const WeightPlan p = weight_plan(cache, sequences, tokens, heads, capacity, !starts);
  if (p.part_bytes && (!workspace || workspace_bytes < p.part_bytes || reinterpret_cast<uintptr_t>(workspace) % 16))
    return fail(DSA_STATUS_WORKSPACE_TOO_SMALL, "paged weights need %lld bytes of 16-byte aligned workspace",
                (long long)p.part_bytes);
  w.batch.causal = causal != 0;
  w.batch.lse = const_cast<float*>(lse);
  w.weights = weights;
  w.parts = static_cast<float*>(workspace);
  w.tiles = (uint32_t)p.tiles;
  w.pieces = (uint32_t)p.pieces;
  w.row_count = (uint64_t)cache->pages * cache->page_size;
  const int64_t grid = p.tiles * sequences * p.pieces * cache->kv_heads;
  DSA_REQUIRE(grid < (1LL << 24), "too many keys for one call");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (p.sets == 1)
    launch_weights<1>(w, cache, (uint32_t)grid, s);
  else
    launch_weights<4>(w, cache, (uint32_t)grid, s);
  if (int st = check_launch("paged_weights_kernel")) return st;
  if (p.pieces == 1) return 0;
  const uint32_t keys = (uint32_t)(p.tiles * 64 * p.sets);
  DSA_REQUIRE(sequences < 65536, "too many sequences for one call");
  const dim3 join((keys + 255) / 256, (unsigned)cache->kv_heads, (unsigned)sequences);
  hipLaunchKernelGGL(paged_weights_join_kernel, join, dim3(256), 0, s, w, keys);
  return check_launch("paged_weights_join_kernel");
}
