// Attention over a paged key/value cache: many query rows, as in a prefill.
//
// The chunk kernel's products and layouts (paged_chunk.hip) at 256 rows a workgroup:
// eight waves of 32 rows share a tile of 64 keys (four at head_dim 256, whose 128
// output registers a lane leave room for one wave a SIMD).  A wave's own arithmetic
// fills the time of its matrix instructions, in two phases a tile:
//   scores of the NEXT tile   under   this tile's exponentials, sums and packing
//   output of this tile       under   the next tile's scaling and maximum
// so that between two matrix instructions stand others that wait for neither.  Keys
// are in LDS a tile ahead of the values.
//
// Bound by power: 2048 tokens over 32K keys (1.06 TFLOP) take 965 us, 1.1 PFLOP/s,
// the matrix pipes busy 54 % of the time at the 1.88 GHz that the card then holds
// (2.1 GHz in the chunk kernel, 1120 us); a plain 8192^3 product of the library makes
// 1.44 PFLOP/s.  Operands read further ahead, half of the waves half a tile behind
// the others, and wave priorities changed nothing; 64 rows a wave spill.
#include "paged_attention.hpp"

namespace dsa {
namespace {

constexpr uint32_t kLeastTiles = kLeastChunkKeys / kTileKeys;  // of a piece

template <class Tag, bool kFp8, int D, int kWaves>
__global__ __launch_bounds__(64 * kWaves, kWaves / 4) void paged_prefill_kernel(PagedAttentionArgs a) {
  constexpr uint32_t kThreads = 64 * kWaves;
  constexpr uint32_t kRows = 32 * kWaves;
  constexpr uint32_t kChunks = kFp8 ? D / 16 : D / 8;  // 16-byte loads per cache row
  constexpr uint32_t kPass = kThreads / kChunks;       // cache rows per pass of the workgroup
  constexpr bool kPart = kPass > kTileKeys;            // fewer loads than threads
  constexpr int kLoads = kPart ? 1 : kTileKeys / kPass;  // passes per tile
  constexpr int kSteps = D / 16;                       // of a 32 x 32 block of scores
  constexpr int kBlocks = D / 32;                      // of an output row
  constexpr int kRing = 4;                             // operands read ahead of their products, and one at work
  static_assert(kPart || kTileKeys % kPass == 0, "a tile is whole passes");
  __shared__ __attribute__((aligned(16))) char key_tile[2][kTileKeys * kKeyRow<D>];
  __shared__ __attribute__((aligned(16))) char value_tile[2][kTileKeys * kValueRow<D>];
  // Places in the cache of tiles t + 1 .. t + 3: offsets of the keys' and the
  // values' row, and for fp8 the row itself.
  __shared__ ulong2 table[4][kTileKeys];
  __shared__ uint32_t table_row[4][kFp8 ? kTileKeys : 1];
  __shared__ __attribute__((aligned(16))) float scales[2][4][kTileKeys];
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
  const uint32_t wave_row = row0 + 32u * wave;
  const uint32_t my_row = min(wave_row + col, rows - 1u);
  const uint32_t my_token = span.first + my_row / a.group;
  const uint32_t my_head = g * a.group + my_row % a.group;
  const uint32_t sees = min(seen(my_row), end);
  const uint32_t all_see = min(seen(min(wave_row, rows - 1u)), end);  // every row of the wave sees these
  const uint32_t all_rows_see = seen(row0);  // of the workgroup
  const uint32_t some_see = wave_row < rows ? min(seen(min(wave_row + 32u, rows) - 1u), end) : 0u;

  uint4 q[kSteps];
  {
    const char* from = a.queries + (int64_t)my_token * a.query_stride + (uint64_t)my_head * D * 2 + 16u * half;
#pragma unroll
    for (int j = 0; j < kSteps; ++j) q[j] = *reinterpret_cast<const uint4*>(from + 32 * j);
  }
  floatx16 o[kBlocks];
#pragma unroll
  for (int i = 0; i < kBlocks; ++i)
#pragma unroll
    for (int e = 0; e < 16; ++e) o[i][e] = 0.f;
  float reference = 0.f;  // set by the row's first tile whose scores are not all -inf
  uint64_t fresh = __ballot(sees > begin);  // lanes whose row has no reference yet
  float total = 0.f;

  const int32_t* pages = a.page_table + (int64_t)piece.sequence * a.table_stride;
  const uint32_t load_row = tid / kChunks;
  const uint32_t load_chunk = tid % kChunks;
  const char* key_base = a.cache.keys + g * a.cache.key_head + 16u * load_chunk;
  const char* value_base = a.cache.values + g * a.cache.value_head + 16u * load_chunk;
  u32x4 kr[kLoads], vr[kLoads];
  float ks = 0.f, vs = 0.f;
  auto load_keys = [&](uint32_t t) {
    if (kPart && load_row >= kTileKeys) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      kr[i] = *reinterpret_cast<const u32x4*>(key_base + table[t & 3u][load_row + kPass * i].x);
    if constexpr (kFp8) {
      if (tid < kTileKeys) ks = a.cache.key_scales[(uint64_t)table_row[t & 3u][tid] * a.cache.kv_heads + g];
    }
  };
  auto load_values = [&](uint32_t t) {
    if (kPart && load_row >= kTileKeys) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i)
      vr[i] = *reinterpret_cast<const u32x4*>(value_base + table[t & 3u][load_row + kPass * i].y);
    if constexpr (kFp8) {
      if (tid < kTileKeys) vs = a.cache.value_scales[(uint64_t)table_row[t & 3u][tid] * a.cache.kv_heads + g];
    }
  };
  auto put = [&](char* row, const u32x4& v) {
    if constexpr (kFp8) {
      *reinterpret_cast<uint4*>(row + 32u * load_chunk) = fp8x8_to_bf16x8_paired(make_uint2(v.x, v.y));
      *reinterpret_cast<uint4*>(row + 32u * load_chunk + 16u) = fp8x8_to_bf16x8_paired(make_uint2(v.z, v.w));
    } else {
      *reinterpret_cast<u32x4*>(row + 16u * load_chunk) = v;
    }
  };
  auto stage_keys = [&](uint32_t t) {
    if (kPart && load_row >= kTileKeys) return;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) put(key_tile[t & 1u] + (load_row + kPass * i) * kKeyRow<D>, kr[i]);
    if constexpr (kFp8) {
      if (tid < kTileKeys) scales[0][t & 3u][tid] = ks;
    }
  };
  auto stage_values = [&](uint32_t t) {
    if (kPart && load_row >= kTileKeys) return;  // these threads have loaded nothing
    const uint32_t key0 = begin + t * kTileKeys;
    if (key0 + kTileKeys > all_rows_see) {
#pragma unroll
      for (int i = 0; i < kLoads; ++i)
        if (key0 + load_row + kPass * i >= all_rows_see && drop_nonfinite<Tag, kFp8>(vr[i])) dropped = 1;
      if (kFp8 && tid < kTileKeys && key0 + tid >= all_rows_see && !is_finite(vs)) {
        vs = 0.f;
        dropped = 1;
      }
    }
#pragma unroll
    for (int i = 0; i < kLoads; ++i) put(value_tile[t & 1u] + (load_row + kPass * i) * kValueRow<D>, vr[i]);
    if constexpr (kFp8) {
      if (tid < kTileKeys) scales[1][t & 3u][tid] = vs;
    }
  };
  // The look-up of a tile's cache rows, a key a thread.
  auto key_of = [&](uint32_t t) { return min(begin + t * kTileKeys + tid % kTileKeys, end - 1u); };
  auto look_page = [&](uint32_t t) { return (uint32_t)pages[key_of(t) >> a.cache.shift]; };
  auto place = [&](uint32_t t, uint32_t page) {
    const uint32_t row = (min(page, a.cache.pages - 1u) << a.cache.shift) | (key_of(t) & ((1u << a.cache.shift) - 1u));
    table[t & 3u][tid % kTileKeys] = ulong2{a.cache.key_offset(row), a.cache.value_offset(row)};
    if constexpr (kFp8) table_row[t & 3u][tid % kTileKeys] = row;
  };

  // This lane's places: keys row `col`, chunk `half`; values in a transposed read
  // of 16 keys x 32 dims.
  const uint32_t key_at = col * kKeyRow<D> + 16u * half;
  const uint32_t value_at = (4u * half + ((lane & 15u) >> 2)) * kValueRow<D> + 32u * ((lane >> 4) & 1u) + 8u * (lane & 3u);
  struct Scores {
    floatx16 s[2];  // s[h][4 b + i]: key 32 h + 8 b + 4 half + i
    float most;
  };
  auto read_key = [&](uint32_t t, int n) {  // keys 32 (n / kSteps) .., step n % kSteps
    return *reinterpret_cast<const uint4*>(key_tile[t & 1u] + key_at + 32u * (n / kSteps) * kKeyRow<D> + 32u * (n % kSteps));
  };
  auto read_value = [&](uint32_t t, int n) {  // block n / 4, keys 16 (n % 4) ..
    const char* at = value_tile[t & 1u] + value_at + 16u * (n % 4) * kValueRow<D> + 64u * (n / 4);
    const uint2 lo = read_transposed(at);
    const uint2 hi = read_transposed(at + 8u * kValueRow<D>);
    return make_uint4(lo.x, lo.y, hi.x, hi.y);
  };
  // Score e less the reference, in powers of two.
  auto scale_score = [&](Scores& x, uint32_t t, int e) {
    float by = a.scale;
    if constexpr (kFp8) by *= scales[0][t & 3u][32 * (e / 16) + 8 * (e % 16 / 4) + 4 * half + e % 4];
    x.s[e / 16][e % 16] = fmaf(x.s[e / 16][e % 16], by, -reference);
  };
  // Hides what the row does not see, and raises the reference if a score passes it.
  auto settle = [&](Scores& x, uint32_t t, bool first) {
    const uint32_t key0 = begin + t * kTileKeys;
    if (key0 + kTileKeys > all_see) {
      x.most = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
          x.s[h][e] = key0 + 32u * h + 8u * (e / 4) + 4u * half + (e % 4) < sees ? x.s[h][e] : -INFINITY;
          x.most = fmaxf(x.most, x.s[h][e]);
        }
    }
    if (first || (__ballot(x.most > kLift + kSlack) | fresh) != 0) {
      const float top = fmaxf(x.most, __shfl_xor(x.most, 32, kWave)) - kLift;
      const float raise = top > (fresh >> lane & 1u ? -INFINITY : 0.f) ? top : 0.f;
      fresh &= __ballot(top == -INFINITY);
      reference += raise;
      // (the first raise may be below zero, by any amount: its sums are 0 and must stay so)
      const float shrink = exp2_fast(fminf(-raise, 0.f));
      total *= shrink;
#pragma unroll
      for (int i = 0; i < kBlocks; ++i) o[i] *= shrink;
#pragma unroll
      for (int h = 0; h < 2; ++h) x.s[h] -= raise;
    }
  };

  // The two phases, product by product: what stands between two barriers of the
  // scheduler is one matrix instruction, the LDS read of a later one's operand and
  // the arithmetic that runs under it.
  constexpr int kProducts = 2 * kSteps;         // of either phase
  constexpr int kEach = 32 / kProducts;         // scores that go with a product
  static_assert(kProducts == 4 * kBlocks && kEach >= 1, "both phases have as many products");
  uint4 p[4];  // weights of a tile, packed
  // The scores of tile t + 1 into y, under the weights of tile t: x its settled
  // scores, which end packed in p.
  auto weigh = [&](uint32_t t, const Scores& x, Scores& y) {
    uint4 k[kRing];
#pragma unroll
    for (int n = 0; n < kRing - 1; ++n) k[n] = read_key(t + 1u, n);
#pragma unroll
    for (int e = 0; e < 16; ++e) y.s[0][e] = y.s[1][e] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
    float weight[32];
    uint32_t words[16];
#pragma unroll
    for (int n = 0; n < kProducts; ++n) {
      if (n + kRing - 1 < kProducts) k[(n + kRing - 1) % kRing] = read_key(t + 1u, n + kRing - 1);
      y.s[n / kSteps] = mfma_32x32x16(Tag{}, k[n % kRing], q[n % kSteps], y.s[n / kSteps]);
#pragma unroll
      for (int e = kEach * n; e < kEach * n + kEach; ++e) {
        weight[e] = exp2_fast(x.s[e / 16][e % 16]);
        total += weight[e];
        if constexpr (kFp8) weight[e] *= scales[1][t & 3u][32 * (e / 16) + 8 * (e % 16 / 4) + 4 * half + e % 4];
        if (e % 2) {
          words[e / 2] = pack2(Tag{}, weight[e - 1], weight[e]);
          asm volatile("" : "+v"(words[e / 2]), "+v"(total));  // here, not where they are used
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) p[u] = make_uint4(words[4 * u], words[4 * u + 1], words[4 * u + 2], words[4 * u + 3]);
  };
  // The output of tile t, under the scaling and maximum of y, the scores of t + 1.
  auto add_output = [&](uint32_t t, Scores& y) {
    uint4 v[kRing];
#pragma unroll
    for (int n = 0; n < kRing - 1; ++n) v[n] = read_value(t, n);
    __builtin_amdgcn_sched_barrier(0);
    float most = -INFINITY;
#pragma unroll
    for (int n = 0; n < kProducts; ++n) {
      if (n + kRing - 1 < kProducts) v[(n + kRing - 1) % kRing] = read_value(t, n + kRing - 1);
      o[n / 4] = mfma_32x32x16(Tag{}, v[n % kRing], p[n % 4], o[n / 4]);
#pragma unroll
      for (int e = kEach * n; e < kEach * n + kEach; ++e) {
        scale_score(y, t + 1u, e);
        if (e % 2) most = fmaxf(fmaxf(most, y.s[e / 16][e % 16 - 1]), y.s[e / 16][e % 16]);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    y.most = most;
    settle(y, t + 1u, false);
  };

  if (begin < end) {
    if (tid == 0) dropped = 0;
    const uint32_t tiles = (end - begin + kTileKeys - 1u) / kTileKeys;
    const uint32_t mine = some_see > begin ? (some_see - begin + kTileKeys - 1u) / kTileKeys : 0u;  // tiles the wave sees
    if (tid < 3u * kTileKeys) place(tid / kTileKeys, look_page(tid / kTileKeys));
    __syncthreads();
    load_keys(0);
    load_values(0);
    stage_keys(0);
    stage_values(0);
    load_keys(1);
    stage_keys(1);
    __syncthreads();
    Scores x, y;
    if (mine > 0) {
#pragma unroll
      for (int e = 0; e < 16; ++e) x.s[0][e] = x.s[1][e] = 0.f;
#pragma unroll
      for (int n = 0; n < kProducts; ++n)
        x.s[n / kSteps] = mfma_32x32x16(Tag{}, read_key(0, n), q[n % kSteps], x.s[n / kSteps]);
      x.most = -INFINITY;
#pragma unroll
      for (int e = 0; e < 32; ++e) {
        scale_score(x, 0, e);
        x.most = fmaxf(x.most, x.s[e / 16][e % 16]);
      }
      settle(x, 0, true);
    }
    __syncthreads();  // every wave has read the first tile's keys
    auto turn = [&](uint32_t t, Scores& now, Scores& next) {
      uint32_t page = 0;
      if (wave == 0) page = look_page(t + 3u);
      __builtin_amdgcn_sched_barrier(0);
      load_keys(t + 2u);  // past the end: the last key again
      load_values(t + 1u);
      __builtin_amdgcn_sched_barrier(0);
      if (t < mine) {
        weigh(t, now, next);
        add_output(t, next);
      }
      stage_keys(t + 2u);
      stage_values(t + 1u);
      if (wave == 0) {
        asm volatile("" : "+v"(page));  // nothing of what follows, and so no wait, moves up to the load
        place(t + 3u, page);
      }
      __syncthreads();
    };
    for (uint32_t t = 0; t < tiles; t += 2u) {
      turn(t, x, y);
      if (t + 1u < tiles) turn(t + 1u, y, x);
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
  if (wave_row + col >= rows) return;
  const uint64_t out = (uint64_t)my_token * a.heads + my_head;
  const uint64_t part = ((uint64_t)(piece.slot + piece.index) * a.cache.kv_heads + g) * kRows + 32u * wave + col;
  if (half == 0 && a.cuts) {
    if (piece.index == 0) a.part_of[out] = make_uint2((uint32_t)part, piece.count);
    if (piece.count > 1u) a.part_sum[part] = make_float2(reference, total);
  }
#pragma unroll
  for (int i = 0; i < kBlocks; ++i)
#pragma unroll
    for (int b = 0; b < 4; ++b) {
      const uint32_t dim = 32u * i + 8u * b + 4u * half;
      const floatx4 v = {o[i][4 * b], o[i][4 * b + 1], o[i][4 * b + 2], o[i][4 * b + 3]};
      if (piece.count > 1u)
        *reinterpret_cast<floatx4*>(a.part_out + part * D + dim) = v;
      else
        store_out<Tag, D>(a, out, dim, v, reference, total);
    }
}

template <class Tag, bool kFp8>
void launch_dim(const PagedAttentionArgs& a, int32_t dim, uint32_t grid, hipStream_t s) {
  if (dim == 64)
    hipLaunchKernelGGL((paged_prefill_kernel<Tag, kFp8, 64, 8>), dim3(grid), dim3(512), 0, s, a);
  else if (dim == 128)
    hipLaunchKernelGGL((paged_prefill_kernel<Tag, kFp8, 128, 8>), dim3(grid), dim3(512), 0, s, a);
  else
    hipLaunchKernelGGL((paged_prefill_kernel<Tag, kFp8, 256, 4>), dim3(grid), dim3(256), 0, s, a);
}

}  // namespace

int launch_paged_prefill(const PagedAttentionArgs& a, int32_t dim, int32_t cache_dtype, uint32_t grid, hipStream_t s) {
  if (cache_dtype == kFP8E4M3)
    launch_dim<Bf16Tag, true>(a, dim, grid, s);
  else if (cache_dtype == kBF16)
    launch_dim<Bf16Tag, false>(a, dim, grid, s);
  else
    launch_dim<F16Tag, false>(a, dim, grid, s);
  return check_launch("paged_prefill_kernel");
}

}  // namespace dsa
