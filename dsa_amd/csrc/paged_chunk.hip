// Attention over a paged key/value cache: some query rows, as in the chunks of a
// mixed batch, on the matrix cores.
//
// A workgroup takes 128 (token, head) rows of one kv head, 32 a wave, against one
// piece of the keys, 64 keys at a time.  Keys and values of a tile go through
// registers into LDS, the next tile's loads in flight under this one's products;
// every wave reads all of them for its own rows.
//   scores^T = K Q^T   v_mfma_f32_32x32x16, keys the A operand: a lane holds 32
//                      scores of one row, so maximum, weights and sum need no
//                      other lane (the two halves of a wave meet only when the
//                      running maximum is raised, and at the end)
//   out^T += V^T P^T   the weights are the B operand as they stand, values read
//                      transposed by ds_read_b64_tr_b16
// Rescaling a row is one factor per lane for the same reason.  Two workgroups a CU
// (three at head_dim 64) hide each other's waits; at few rows that reads the cache at
// 3.9 TB/s (20 rows a kv head of 64K bf16 keys, 268 MB: 68 us), at 128 it makes 440
// TFLOP/s, and from there on the prefill kernel is the faster one.
#include "paged_attention.hpp"

namespace dsa {
namespace {

constexpr uint32_t kLeastTiles = kLeastChunkKeys / kTileKeys;  // of a piece

// Keeps a value's computation where it stands: the compiler would move it past
// the next branch, away from the products that it is to run under.
__device__ __forceinline__ void pin(float& v) { asm volatile("" : "+v"(v)); }

// The scheduling of the instructions so far in the block: `others` arithmetic ones
// after each of `products` matrix ones.
#define interleave(products, others)                          \
  _Pragma("unroll") for (int n_ = 0; n_ < (products); ++n_) { \
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);        \
    __builtin_amdgcn_sched_group_barrier(0x402, (others), 0); \
  }

template <class Tag, bool kFp8, int D>
__global__ __launch_bounds__(256, 2) void paged_chunk_kernel(PagedAttentionArgs a) {
  constexpr uint32_t kThreads = 256;
  constexpr uint32_t kRows = kChunkRows;
  constexpr uint32_t kChunks = kFp8 ? D / 16 : D / 8;       // 16-byte loads per cache row
  constexpr uint32_t kPass = kThreads / kChunks;            // cache rows per pass of the workgroup
  constexpr int kLoads = kTileKeys / kPass;                 // passes per tile
  constexpr int kKeyBytes = kTileKeys * kKeyRow<D>;
  constexpr int kValueBytes = kTileKeys * kValueRow<D>;
  static_assert(kLoads >= 1 && kTileKeys % kPass == 0, "a tile is whole passes");
  __shared__ __attribute__((aligned(16))) char key_tile[2][kKeyBytes];
  __shared__ __attribute__((aligned(16))) char value_tile[2][kValueBytes];
  // Places in the cache of tiles t .. t + 2: offsets of the keys' and the values'
  // row, and for fp8 the row itself.
  __shared__ ulong2 table[4][kTileKeys];
  __shared__ uint32_t table_row[4][kFp8 ? kTileKeys : 1];
  __shared__ __attribute__((aligned(16))) float scales[2][2][kTileKeys];
  // Whether a value was staged as 0 for not being finite: in the last row's padding.
  uint32_t& dropped = *reinterpret_cast<uint32_t*>(key_tile[0] + kTileKeys * kKeyRow<D> - 16u);
  const uint32_t tid = threadIdx.x;
  const uint32_t lane = lane_id();
  const uint32_t wave = tid / kWave;
  const uint32_t col = lane & 31u;
  const uint32_t half = lane >> 5;

  // Heads vary fastest: workgroups go round-robin over the XCDs, so that a kv
  // head's keys meet all of its rows in few L2s.
  const uint32_t g = blockIdx.x % a.cache.kv_heads;
  clear_unowned<D, kThreads>(a);
  Piece piece;
  if (!find_piece<kRows, kTileKeys, kLeastTiles>(a, blockIdx.x / a.cache.kv_heads, piece)) return;
  const Span span = piece.span;
  const uint32_t length = piece.keys;
  const uint32_t rows = span.count * a.group;
  // The last tile of a sequence first: a causal chunk's last rows see most.
  const uint32_t row0 = ((rows + kRows - 1u) / kRows - 1u - piece.tile) * kRows;

  // Row r sees keys below `seen(r)`.
  auto seen = [&](uint32_t r) {
    return a.causal ? (uint32_t)max(0, (int32_t)(length - span.count + r / a.group + 1u)) : length;
  };
  const uint32_t visible = seen(min(row0 + kRows, rows) - 1u);
  const uint32_t begin = (uint32_t)min((uint64_t)piece.index * piece.units * kTileKeys, (uint64_t)visible);
  const uint32_t end = (uint32_t)min((uint64_t)begin + (uint64_t)piece.units * kTileKeys, (uint64_t)visible);
  const uint32_t wave_row = min(row0 + 32u * wave, rows - 1u);
  const uint32_t my_row = min(row0 + 32u * wave + col, rows - 1u);
  const uint32_t my_token = span.first + my_row / a.group;
  const uint32_t my_head = g * a.group + my_row % a.group;
  const uint32_t sees = min(seen(my_row), end);
  const uint32_t all_see = min(seen(wave_row), end);  // every row of the wave sees these
  const uint32_t all_rows_see = seen(row0);  // of the workgroup
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
  float reference = 0.f;  // set by the row's first keys whose scores are not all -inf
  uint64_t fresh = __ballot(sees > begin);  // lanes whose row has no reference yet
  float total = 0.f;

  const int32_t* pages = a.page_table + (int64_t)piece.sequence * a.table_stride;
  const uint32_t load_row = tid / kChunks;
  const uint32_t load_chunk = tid % kChunks;
  const char* key_base = a.cache.keys + g * a.cache.key_head + 16u * load_chunk;
  const char* value_base = a.cache.values + g * a.cache.value_head + 16u * load_chunk;

  u32x4 kr[kLoads], vr[kLoads];
  float sr = 0.f;
  auto load = [&](uint32_t t) {
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const ulong2 at = table[t & 3u][load_row + kPass * i];
      kr[i] = *reinterpret_cast<const u32x4*>(key_base + at.x);
      vr[i] = *reinterpret_cast<const u32x4*>(value_base + at.y);
    }
    if constexpr (kFp8) {
      if (tid < 2u * kTileKeys) {
        const uint32_t row = table_row[t & 3u][tid % kTileKeys];
        sr = (tid < kTileKeys ? a.cache.key_scales : a.cache.value_scales)[(uint64_t)row * a.cache.kv_heads + g];
      }
    }
  };
  auto stage = [&](uint32_t t) {
    const uint32_t key0 = begin + t * kTileKeys;
    if (key0 + kTileKeys > all_rows_see) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        if (key0 + load_row + kPass * i >= all_rows_see && drop_nonfinite<Tag, kFp8>(vr[i])) dropped = 1;
      if (kFp8 && tid >= kTileKeys && key0 + tid - kTileKeys >= all_rows_see && !is_finite(sr)) {
        sr = 0.f;
        dropped = 1;
      }
    }
    char* keys = key_tile[t & 1u];
    char* values = value_tile[t & 1u];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      const uint32_t row = load_row + kPass * i;
      if constexpr (kFp8) {
        *reinterpret_cast<uint4*>(keys + row * kKeyRow<D> + 32u * load_chunk) = fp8x8_to_bf16x8_paired(make_uint2(kr[i].x, kr[i].y));
        *reinterpret_cast<uint4*>(keys + row * kKeyRow<D> + 32u * load_chunk + 16u) = fp8x8_to_bf16x8_paired(make_uint2(kr[i].z, kr[i].w));
        *reinterpret_cast<uint4*>(values + row * kValueRow<D> + 32u * load_chunk) = fp8x8_to_bf16x8_paired(make_uint2(vr[i].x, vr[i].y));
        *reinterpret_cast<uint4*>(values + row * kValueRow<D> + 32u * load_chunk + 16u) = fp8x8_to_bf16x8_paired(make_uint2(vr[i].z, vr[i].w));
      } else {
        *reinterpret_cast<u32x4*>(keys + row * kKeyRow<D> + 16u * load_chunk) = kr[i];
        *reinterpret_cast<u32x4*>(values + row * kValueRow<D> + 16u * load_chunk) = vr[i];
      }
    }
    if constexpr (kFp8) {
      if (tid < 2u * kTileKeys) scales[t & 1u][tid / kTileKeys][tid % kTileKeys] = sr;
    }
  };
  // This lane's places: keys row `col`, chunk `half`; values in a transposed read
  // of 16 keys x 32 dims.
  const uint32_t key_at = col * kKeyRow<D> + 16u * half;
  const uint32_t value_at = (4u * half + ((lane & 15u) >> 2)) * kValueRow<D> + 32u * ((lane >> 4) & 1u) + 8u * (lane & 3u);

  // One tile for the wave's rows, 32 keys at a time, so that the products of one
  // half run under the exponentials of the other: a dependent product holds up
  // the wave, but between two of them other instructions issue.  Operands are
  // read from LDS a batch ahead of their products.
  auto compute = [&](uint32_t t) {
    const uint32_t key0 = begin + t * kTileKeys;
    if (key0 >= some_see) return;
    const char* keys = key_tile[t & 1u] + key_at;
    const char* values = value_tile[t & 1u] + value_at;
    constexpr int kSteps = D / 16;
    uint4 ka[kSteps], kb[kSteps];
    floatx16 x[2];
    auto read_key = [&](uint32_t s, uint32_t step) {
      return *reinterpret_cast<const uint4*>(keys + 32u * s * kKeyRow<D> + 32u * step);
    };
    // x[s][4 b + i]: key 32 s + 8 b + 4 half + i.  Scores less the reference, in
    // powers of two, hidden ones -inf, and their maximum.
    auto scores = [&](uint32_t s) {
      float most = -INFINITY;
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        floatx4 by = {a.scale, a.scale, a.scale, a.scale};
        if constexpr (kFp8) by *= *reinterpret_cast<const floatx4*>(&scales[t & 1u][0][32 * s + 8 * b + 4 * half]);
#pragma unroll
        for (int i = 0; i < 4; ++i) x[s][4 * b + i] = fmaf(x[s][4 * b + i], by[i], -reference);
      }
      if (key0 + 32u * s + 32u > all_see) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          x[s][e] = key0 + 32u * s + 8u * (e / 4) + 4u * half + (e % 4) < sees ? x[s][e] : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < 16; e += 2) most = fmaxf(fmaxf(most, x[s][e]), x[s][e + 1]);
      return most;
    };
    auto raises = [&](float most) { return (__ballot(most > kLift + kSlack) | fresh) != 0; };
    auto raise_by = [&](float most) {
      most = fmaxf(most, __shfl_xor(most, 32, kWave)) - kLift;
      const float raise = most > (fresh >> lane & 1u ? -INFINITY : 0.f) ? most : 0.f;
      fresh &= __ballot(most == -INFINITY);
      reference += raise;
      // (the first raise may be below zero, by any amount: its sums are 0 and must stay so)
      const float shrink = exp2_fast(fminf(-raise, 0.f));
      total *= shrink;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] *= shrink;
      return raise;
    };
    float weight[2][16];
    auto weigh = [&](uint32_t s) {
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        weight[s][e] = exp2_fast(x[s][e]);
        total += weight[s][e];
      }
    };
    auto packed = [&](uint32_t s, uint32_t u) {
      const float* p = &weight[s][8 * u];
      floatx4 w[2] = {{p[0], p[1], p[2], p[3]}, {p[4], p[5], p[6], p[7]}};
      if constexpr (kFp8) {
#pragma unroll
        for (int b = 0; b < 2; ++b)
          w[b] *= *reinterpret_cast<const floatx4*>(&scales[t & 1u][1][32 * s + 16 * u + 8 * b + 4 * half]);
      }
      return make_uint4(pack2(Tag{}, w[0][0], w[0][1]), pack2(Tag{}, w[0][2], w[0][3]), pack2(Tag{}, w[1][0], w[1][1]),
                        pack2(Tag{}, w[1][2], w[1][3]));
    };
    auto read_value = [&](uint32_t u, uint32_t i) {
      const uint2 lo = read_transposed(values + 16u * u * kValueRow<D> + 64u * i);
      const uint2 hi = read_transposed(values + (16u * u + 8u) * kValueRow<D> + 64u * i);
      return make_uint4(lo.x, lo.y, hi.x, hi.y);
    };

#pragma unroll
    for (int j = 0; j < kSteps; ++j) ka[j] = read_key(0, j);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int e = 0; e < 16; ++e) x[0][e] = x[1][e] = 0.f;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) {
      kb[j] = read_key(1, j);
      x[0] = mfma_32x32x16(Tag{}, ka[j], q[j], x[0]);
    }
    __builtin_amdgcn_sched_barrier(0);
    const float most0 = scores(0);
    if (raises(most0)) x[0] -= raise_by(most0);
#pragma unroll
    for (int j = 0; j < kSteps; ++j) x[1] = mfma_32x32x16(Tag{}, kb[j], q[j], x[1]);
    weigh(0);
    uint4 va[D / 32], vb[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) va[i] = read_value(0, i);
    interleave(kSteps, 48 / kSteps);
#pragma unroll
    for (int e = 0; e < 16; ++e) pin(weight[0][e]);
    const float most1 = scores(1);
    if (raises(most1)) {
      const float raise = raise_by(most1);
      const float shrink = exp2_fast(fminf(-raise, 0.f));
#pragma unroll
      for (int e = 0; e < 16; ++e) weight[0][e] *= shrink;
      x[1] -= raise;
    }
    {
      const uint4 p0 = packed(0, 0), p1 = packed(0, 1);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        vb[i] = read_value(1, i);
        o[i] = mfma_32x32x16(Tag{}, va[i], p0, o[i]);
      }
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        va[i] = read_value(2, i);
        o[i] = mfma_32x32x16(Tag{}, vb[i], p1, o[i]);
      }
      weigh(1);
    }
    {
      const uint4 p0 = packed(1, 0), p1 = packed(1, 1);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        vb[i] = read_value(3, i);
        o[i] = mfma_32x32x16(Tag{}, va[i], p0, o[i]);
      }
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] = mfma_32x32x16(Tag{}, vb[i], p1, o[i]);
    }
  };

  if (begin < end) {
    if (tid == 0) dropped = 0;
    const uint32_t tiles = (end - begin + kTileKeys - 1u) / kTileKeys;
    // The look-up of a tile's cache rows, by its first 64 threads: the page id's
    // load two tiles ahead of the rows' and before them, its use after the tile.
    auto key_of = [&](uint32_t t) { return min(begin + t * kTileKeys + tid % kTileKeys, end - 1u); };
    auto look_page = [&](uint32_t t) { return (uint32_t)pages[key_of(t) >> a.cache.shift]; };
    auto place = [&](uint32_t t, uint32_t page) {
      const uint32_t row = (min(page, a.cache.pages - 1u) << a.cache.shift) | (key_of(t) & ((1u << a.cache.shift) - 1u));
      table[t & 3u][tid % kTileKeys] = ulong2{a.cache.key_offset(row), a.cache.value_offset(row)};
      if constexpr (kFp8) table_row[t & 3u][tid % kTileKeys] = row;
    };
    if (tid < 2u * kTileKeys) place(tid / kTileKeys, look_page(tid / kTileKeys));
    __syncthreads();
    load(0);
    stage(0);
    __syncthreads();
    for (uint32_t t = 0; t < tiles; ++t) {
      uint32_t page = 0;
      if (wave == 0) page = look_page(t + 2u);
      __builtin_amdgcn_sched_barrier(0);
      load(t + 1u);  // past the end: the last key again
      __builtin_amdgcn_sched_barrier(0);
      compute(t);
      stage(t + 1u);
      if (wave == 0) {
        asm volatile("" : "+v"(page));  // nothing of what follows, and so no wait, moves up to the load
        place(t + 2u, page);
      }
      __syncthreads();
    }
  }

  if (begin < end && all_rows_see < end && dropped) {
    for (uint32_t k = max(begin, all_rows_see); k < end; ++k)
      if (k < sees) {
        const uint32_t row = cache_row(a, pages, k);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int b = 0; b < 4; ++b) {
            float back[4] = {0.f, 0.f, 0.f, 0.f};
            add_nonfinite<Tag, kFp8>(a, row, g, 32u * i + 8u * b + 4u * half, back);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[i][4 * b + e] += back[e];
            __builtin_amdgcn_sched_barrier(0);  // few loads at a time: no registers for more
          }
      }
  }

  total += __shfl_xor(total, 32, kWave);
  if (total == 0.f) reference = kNoKeys;
  if (row0 + 32u * wave + col >= rows) return;
  const uint64_t my_out = (uint64_t)my_token * a.heads + my_head;
  const uint64_t part = ((uint64_t)(piece.slot + piece.index) * a.cache.kv_heads + g) * kRows + 32u * wave + col;
  if (half == 0 && a.cuts) {
    if (piece.index == 0) a.part_of[my_out] = make_uint2((uint32_t)part, piece.count);
    if (piece.count > 1u) a.part_sum[part] = make_float2(reference, total);
  }
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const uint32_t dim = 32u * i + 8u * b + 4u * half;
      const floatx4 v = {o[i][4 * b], o[i][4 * b + 1], o[i][4 * b + 2], o[i][4 * b + 3]};
      if (piece.count > 1u)
        *reinterpret_cast<floatx4*>(a.part_out + part * D + dim) = v;
      else
        store_out<Tag, D>(a, my_out, dim, v, reference, total);
    }
}

}  // namespace

template <class Tag, bool kFp8>
static void launch_dim(const PagedAttentionArgs& a, int32_t dim, uint32_t grid, hipStream_t s) {
  if (dim == 64)
    hipLaunchKernelGGL((paged_chunk_kernel<Tag, kFp8, 64>), dim3(grid), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((paged_chunk_kernel<Tag, kFp8, 128>), dim3(grid), dim3(256), 0, s, a);
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
