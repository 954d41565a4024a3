// Attention over a paged key/value cache: many query rows, as in a prefill or a
// chunk of a prompt, on the matrix cores.
//
// A workgroup takes 32 (token, head) rows of one kv head per wave against one
// piece of the keys, 64 keys at a time.  Keys and values of a tile go through
// registers into LDS, the next tile's loads in flight under this one's
// products; every wave reads all of them for its own rows.
//   scores^T = K Q^T   v_mfma_f32_32x32x16, keys the A operand: a lane holds 32
//                      scores of one row, so maximum, weights and sum need no
//                      other lane (the two halves of a wave meet only when the
//                      running maximum is raised, and at the end)
//   out^T += V^T P^T   the weights are the B operand as they stand, values read
//                      transposed by ds_read_b64_tr_b16
// Rescaling a row is one factor per lane for the same reason.
#include "paged_attention.hpp"

namespace dsa {
namespace {

constexpr int kTileKeys = 64;

typedef float floatx16 __attribute__((ext_vector_type(16)));

__device__ __forceinline__ floatx16 mfma_32x32x16(Bf16Tag, uint4 a, uint4 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ floatx16 mfma_32x32x16(F16Tag, uint4 a, uint4 b, floatx16 c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// LDS places of 16-byte chunk `chunk` of a row.  Keys are read 16 rows at one
// chunk at a time, values 4 rows x 4 chunks: each fills 256 bytes of banks.
template <int D>
__device__ __forceinline__ uint32_t key_place(uint32_t row, uint32_t chunk) {
  const uint32_t x = D == 64 ? (row >> 1) & 7u : row & 15u;
  return row * (D * 2) + ((chunk ^ x) << 4);
}
template <int D>
__device__ __forceinline__ uint32_t tile_value_place(uint32_t row, uint32_t chunk) {
  const uint32_t x = D == 64 ? ((row >> 1) & 1u) << 2 : (row & 3u) << 2;
  return row * (D * 2) + ((chunk ^ x) << 4);
}

template <class Tag, bool kFp8, int D, int kWaves>
__global__ __launch_bounds__(64 * kWaves, D == 256 ? kWaves / 4 : 2) void paged_chunk_kernel(PagedAttentionArgs a) {
  constexpr uint32_t kThreads = 64 * kWaves;
  constexpr uint32_t kRows = 32 * kWaves;
  constexpr uint32_t kChunks = kFp8 ? D / 16 : D / 8;       // 16-byte loads per cache row
  constexpr uint32_t kPass = kThreads / kChunks;            // cache rows per pass of the workgroup
  constexpr int kLoads = kTileKeys / kPass;                 // passes per tile
  constexpr int kTileBytes = kTileKeys * D * 2;
  static_assert(kLoads >= 1 && kTileKeys % kPass == 0, "a tile is whole passes");
  __shared__ __attribute__((aligned(16))) char key_tile[2][kTileBytes];
  __shared__ __attribute__((aligned(16))) char value_tile[2][kTileBytes];
  __shared__ __attribute__((aligned(16))) int32_t table[4][kTileKeys];  // cache rows of tiles t .. t + 2
  __shared__ __attribute__((aligned(16))) float scales[2][2][kTileKeys];
  const uint32_t tid = threadIdx.x;
  const uint32_t lane = lane_id();
  const uint32_t wave = tid / kWave;
  const uint32_t col = lane & 31u;
  const uint32_t half = lane >> 5;

  const uint32_t g = blockIdx.x % a.cache.kv_heads;
  const uint32_t rest = blockIdx.x / a.cache.kv_heads;
  const uint32_t piece = rest % a.splits;
  RowTile tile;
  if (!find_row_tile(a, rest / a.splits, kRows, tile)) return;
  const uint32_t length = keys_of(a, tile.sequence);
  const uint32_t rows = tile.span.count * a.group;
  // The last tile of a sequence first: a causal chunk's last rows see most.
  const uint32_t row0 = ((rows + kRows - 1u) / kRows - 1u - tile.index) * kRows;

  // Row r sees keys below `seen(r)`.
  auto seen = [&](uint32_t r) {
    return a.causal ? (uint32_t)max(0, (int32_t)(length - tile.span.count + r / a.group + 1u)) : length;
  };
  const uint32_t visible = seen(min(row0 + kRows, rows) - 1u);
  const uint32_t chunk = max(256u, ((visible + a.splits - 1u) / a.splits + kTileKeys - 1u) & ~(kTileKeys - 1u));
  const uint32_t begin = min(piece * chunk, visible);
  const uint32_t end = min(begin + chunk, visible);
  const uint32_t wave_row = min(row0 + 32u * wave, rows - 1u);
  const uint32_t my_row = min(row0 + 32u * wave + col, rows - 1u);
  const uint32_t my_token = tile.span.first + my_row / a.group;
  const uint32_t my_head = g * a.group + my_row % a.group;
  const uint32_t sees = min(seen(my_row), end);
  const uint32_t all_see = min(seen(wave_row), end);                          // every row of the wave sees these
  const uint32_t some_see = row0 + 32u * wave < rows ? min(seen(min(wave_row + 31u, rows - 1u)), end) : 0u;

  uint4 q[D / 16];
  {
    const char* p = a.queries + (int64_t)my_token * a.query_stride + (uint64_t)my_head * D * 2 + 16u * half;
#pragma unroll
    for (int j = 0; j < D / 16; ++j) q[j] = *reinterpret_cast<const uint4*>(p + 32 * j);
  }
  floatx16 o[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float reference = 0.f;  // set by the first tile: a row that sees any key of the piece sees its first
  float total = 0.f;

  const int32_t* pages = a.page_table + (int64_t)tile.sequence * a.table_stride;
  const uint32_t load_row = tid / kChunks;
  const uint32_t load_chunk = tid % kChunks;
  const char* key_base = a.cache.keys + g * a.cache.key_head + 16u * load_chunk;
  const char* value_base = a.cache.values + g * a.cache.value_head + 16u * load_chunk;

  u32x4 kr[kLoads], vr[kLoads];
  float sr = 0.f;
  auto load = [&](uint32_t t) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t row = (uint32_t)table[t & 3u][load_row + kPass * i];
      kr[i] = *reinterpret_cast<const u32x4*>(key_base + a.cache.key_offset(row));
      vr[i] = *reinterpret_cast<const u32x4*>(value_base + a.cache.value_offset(row));
    }
    if constexpr (kFp8) {
      if (tid < 2u * kTileKeys) {
        const uint32_t row = (uint32_t)table[t & 3u][tid % kTileKeys];
        sr = (tid < kTileKeys ? a.cache.key_scales : a.cache.value_scales)[(uint64_t)row * a.cache.kv_heads + g];
      }
    }
  };
  auto stage = [&](uint32_t t) {
    char* keys = key_tile[t & 1u];
    char* values = value_tile[t & 1u];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t row = load_row + kPass * i;
      if constexpr (kFp8) {
        *reinterpret_cast<uint4*>(keys + key_place<D>(row, 2u * load_chunk)) = fp8x8_to_bf16x8_paired(make_uint2(kr[i].x, kr[i].y));
        *reinterpret_cast<uint4*>(keys + key_place<D>(row, 2u * load_chunk + 1u)) = fp8x8_to_bf16x8_paired(make_uint2(kr[i].z, kr[i].w));
        *reinterpret_cast<uint4*>(values + tile_value_place<D>(row, 2u * load_chunk)) = fp8x8_to_bf16x8_paired(make_uint2(vr[i].x, vr[i].y));
        *reinterpret_cast<uint4*>(values + tile_value_place<D>(row, 2u * load_chunk + 1u)) = fp8x8_to_bf16x8_paired(make_uint2(vr[i].z, vr[i].w));
      } else {
        *reinterpret_cast<u32x4*>(keys + key_place<D>(row, load_chunk)) = kr[i];
        *reinterpret_cast<u32x4*>(values + tile_value_place<D>(row, load_chunk)) = vr[i];
      }
    }
    if constexpr (kFp8) {
      if (tid < 2u * kTileKeys) scales[t & 1u][tid / kTileKeys][tid % kTileKeys] = sr;
    }
  };
  // Places of this lane in a transposed read of 16 keys x 32 dims, by 32-dim block.
  uint32_t tr_place[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
    tr_place[i] = tile_value_place<D>(4u * half + ((lane & 15u) >> 2), 4u * i + 2u * ((lane >> 4) & 1u) + ((lane & 3u) >> 1)) +
                  8u * (lane & 1u);

  auto compute = [&](uint32_t t) {
    const uint32_t key0 = begin + t * kTileKeys;
    if (key0 >= some_see) return;
    const char* keys = key_tile[t & 1u];
    const char* values = value_tile[t & 1u];
    floatx16 x[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x[s][e] = 0.f;
#pragma unroll
      for (int j = 0; j < D / 16; ++j)
        x[s] = mfma_32x32x16(Tag{}, *reinterpret_cast<const uint4*>(keys + key_place<D>(32u * s + col, 2u * j + half)), q[j], x[s]);
    }
    // x[s][4 a + i]: key 32 s + 8 a + 4 half + i
    if constexpr (kFp8) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const floatx4 ks = *reinterpret_cast<const floatx4*>(&scales[t & 1u][0][32 * s + 8 * b + 4 * half]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[s][4 * b + i] *= ks[i];
        }
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int e = 0; e < 16; ++e) x[s][e] = fmaf(x[s][e], a.scale, -reference);
    if (key0 + kTileKeys > all_see) {
#pragma unroll
      for (int s = 0; s < 2; ++s)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[s][e] = key0 + 32u * s + 8u * (e / 4) + 4u * half + (e % 4) < sees ? x[s][e] : -INFINITY;
    }
    float most = fmaxf(x[0][0], x[1][0]);
#pragma unroll
    for (int e = 1; e < 16; ++e) most = fmaxf(most, fmaxf(x[0][e], x[1][e]));
    if (t == 0 || __any(most > kLift + kSlack)) {
      most = fmaxf(most, __shfl_xor(most, 32, kWave)) - kLift;
      const float raise = t == 0 ? (most == -INFINITY ? 0.f : most) : fmaxf(most, 0.f);
      reference += raise;
      const float shrink = exp2_fast(-raise);
      total *= shrink;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] *= shrink;
#pragma unroll
      for (int s = 0; s < 2; ++s) x[s] -= raise;
    }
    uint4 p[4];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        x[s][e] = exp2_fast(x[s][e]);
        total += x[s][e];
      }
      if constexpr (kFp8) {
#pragma unroll
        for (int b = 0; b < 4; ++b) {
          const floatx4 vs = *reinterpret_cast<const floatx4*>(&scales[t & 1u][1][32 * s + 8 * b + 4 * half]);
#pragma unroll
          for (int i = 0; i < 4; ++i) x[s][4 * b + i] *= vs[i];
        }
      }
#pragma unroll
      for (int u = 0; u < 2; ++u)
        p[2 * s + u] = make_uint4(pack2(Tag{}, x[s][8 * u], x[s][8 * u + 1]), pack2(Tag{}, x[s][8 * u + 2], x[s][8 * u + 3]),
                                  pack2(Tag{}, x[s][8 * u + 4], x[s][8 * u + 5]), pack2(Tag{}, x[s][8 * u + 6], x[s][8 * u + 7]));
    }
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int u = 0; u < 4; ++u) {
        const uint2 lo = read_transposed(values + tr_place[i] + (16 * u) * D * 2);
        const uint2 hi = read_transposed(values + tr_place[i] + (16 * u + 8) * D * 2);
        o[i] = mfma_32x32x16(Tag{}, make_uint4(lo.x, lo.y, hi.x, hi.y), p[u], o[i]);
      }
  };

  if (begin < end) {
    const uint32_t tiles = (end - begin + kTileKeys - 1u) / kTileKeys;
    auto look_up = [&](uint32_t t) { return (int32_t)cache_row(a, pages, min(begin + t * kTileKeys + tid % kTileKeys, end - 1u)); };
    if (tid < 2u * kTileKeys) table[tid / kTileKeys][tid % kTileKeys] = look_up(tid / kTileKeys);
    __syncthreads();
    load(0);
    stage(0);
    __syncthreads();
    for (uint32_t t = 0; t < tiles; ++t) {
      load(t + 1u);  // past the end: the last key again
      int32_t next = 0;
      if (tid < (uint32_t)kTileKeys) next = look_up(t + 2u);
      compute(t);
      stage(t + 1u);
      if (tid < (uint32_t)kTileKeys) table[(t + 2u) & 3u][tid] = next;
      __syncthreads();
    }
  }

  total += __shfl_xor(total, 32, kWave);
  if (total == 0.f) reference = kNoKeys;
  if (row0 + 32u * wave + col >= rows) return;
  const uint64_t my_out = (uint64_t)my_token * a.heads + my_head;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const uint32_t dim = 32u * i + 8u * b + 4u * half;
      const floatx4 part = {o[i][4 * b], o[i][4 * b + 1], o[i][4 * b + 2], o[i][4 * b + 3]};
      if (a.splits > 1) {
        const uint64_t at = my_out * a.splits + piece;
        *reinterpret_cast<floatx4*>(a.part_out + at * D + dim) = part;
        if (dim == 0) a.part_sum[at] = make_float2(reference, total);
      } else {
        store_out<Tag, D>(a, my_out, dim, part, reference, total);
      }
    }
}

}  // namespace

template <class Tag, bool kFp8>
static void launch_dim(const PagedAttentionArgs& a, int32_t dim, uint32_t grid, hipStream_t s) {
  constexpr int kThreads = 2 * kChunkRows;
  if (dim == 64)
    hipLaunchKernelGGL((paged_chunk_kernel<Tag, kFp8, 64, kChunkRows / 32>), dim3(grid), dim3(kThreads), 0, s, a);
  else if (dim == 128)
    hipLaunchKernelGGL((paged_chunk_kernel<Tag, kFp8, 128, kChunkRows / 32>), dim3(grid), dim3(kThreads), 0, s, a);
  else
    hipLaunchKernelGGL((paged_chunk_kernel<Tag, kFp8, 256, kChunkRows / 32>), dim3(grid), dim3(kThreads), 0, s, a);
}

int launch_paged_chunk(const PagedAttentionArgs& a, int32_t dim, int32_t cache_dtype, uint32_t grid, hipStream_t s) {
  if (cache_dtype == kFP8E4M3)
    launch_dim<Bf16Tag, true>(a, dim, grid, s);
  else if (cache_dtype == kBF16)
    launch_dim<Bf16Tag, false>(a, dim, grid, s);
  else
    launch_dim<F16Tag, false>(a, dim, grid, s);
  return check_launch("paged_chunk_kernel");
}

}  // namespace dsa
