// Attention over a paged key/value cache: a few query rows against many keys.
//
//   s_j = scale q . k_j,  o = sum_j exp(s_j) v_j / sum_j exp(s_j)
//
// over the keys a row sees: its sequence's first ones up to its own position,
// or the positions its index list names.  One pass over the keys with the
// running maximum and sum of the softmax; scores, weights' sum and output stay
// in fp32, and the weights are rounded to the queries' type for the second
// product, whose error then is of the output's own rounding.
//
// A workgroup takes 16 rows, which are (token, head) pairs of one kv head,
// against one piece of the keys; its four waves take steps of 32 keys each.
// Keys are the A operand of v_mfma_f32_16x16x32 and queries the B operand, so a
// lane ends with eight scores of ONE row (lane & 15) and those are, as they
// stand, the B operand of the second product: its k index is any order of the
// 32 keys that both operands share, and here is the order the scores have.  The
// values' transposed operand is read from LDS by ds_read_b64_tr_b16.  Every row
// of the cache is read once, as 16-byte loads of 64 contiguous bytes a row.
#include "paged_attention.hpp"

namespace dsa {
namespace {

constexpr int kSpan = 2048;  // keys whose cache rows are looked up at a time
constexpr int kStep = 32;    // keys per wave and step
constexpr int kMostSplits = 256;
constexpr int kMostTiles = 1024;  // row tiles x kv heads that are split (each has a counter)

// LDS that the lanes of one wave share: a wave's LDS accesses are served in
// order, so only the compiler has to keep them so.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

// Place of 16-byte chunk `chunk` of row `row` in a wave's value tile: the 8 rows
// x 2 chunks of half a transposed read, and the 16 rows of a store, fall on
// different banks.
template <int D>
__device__ __forceinline__ uint32_t value_place(uint32_t row, uint32_t chunk) {
  const uint32_t x = D == 64 ? (((row >> 1) & 3u) << 1) | ((row >> 3) & 1u) : ((row & 7u) << 1) | ((row >> 3) & 1u);
  return row * (D * 2) + ((chunk ^ x) << 4);
}

template <bool kFp8, int D>
struct Tile {
  static constexpr int kLoads = kFp8 ? D / 64 : D / 32;  // 16-byte loads per lane and 16-key tile
  uint4 k[2][kLoads];
  uint4 v[2][kLoads];
  float scale;  // fp8: lane l < 32 the key scale of key l, else the value scale of key l - 32
};

template <class Tag, bool kFp8, int D, bool kSelected>
__global__ __launch_bounds__(256, D == 256 ? 1 : 2) void paged_stream_kernel(PagedAttentionArgs a) {
  constexpr int kLoads = Tile<kFp8, D>::kLoads;
  constexpr int kQ = D / 32;  // k-steps of the first product
  constexpr int kO = D / 16;  // dim tiles of the second
  __shared__ __attribute__((aligned(16))) char values[4][kStep * D * 2];  // a wave's value tile; its output at the end
  __shared__ __attribute__((aligned(16))) int32_t table[kSpan];
  __shared__ __attribute__((aligned(16))) float scales[4][64];
  __shared__ float2 sums[4][16];
  __shared__ uint32_t last_piece;
  const uint32_t lane = lane_id();
  const uint32_t wave = threadIdx.x / kWave;
  const uint32_t col = lane & 15u;
  const uint32_t quad = lane >> 4;

  // Heads vary fastest: workgroups go round-robin over the XCDs, so a kv head's
  // rows meet in few L2s.
  const uint32_t g = blockIdx.x % a.cache.kv_heads;
  const uint32_t rest = blockIdx.x / a.cache.kv_heads;
  const uint32_t piece = rest % a.splits;
  const uint32_t item = rest / a.splits;

  uint32_t sequence, token0, row0, rows, length, visible, seen0 = 0;
  if constexpr (kSelected) {
    // item: a tile of a token's heads
    const uint32_t tiles = (a.group + 15u) / 16u;
    token0 = item / tiles;
    row0 = item % tiles * 16u;
    rows = a.group;
    sequence = sequence_of(a, token0);
    length = keys_of(a, sequence);
    visible = length ? a.k : 0u;
  } else {
    // item: a tile of some sequence's (token, head) rows, counted over the sequences
    RowTile tile;
    if (!find_row_tile(a, item, 16u, tile)) return;
    sequence = tile.sequence;
    const Span span = tile.span;
    token0 = span.first;
    row0 = tile.index * 16u;
    rows = span.count * a.group;
    length = keys_of(a, sequence);
    // row r sees keys below seen0 + r / group + 1 of a causal chunk
    seen0 = a.causal ? length - span.count : length;  // may wrap below zero: see `sees`
    const uint32_t last = min(row0 + 15u, rows - 1u) / a.group;
    visible = a.causal ? (uint32_t)max(0, (int32_t)(length - span.count + last + 1u)) : length;
  }

  // This lane's row, and the keys it sees.
  const uint32_t my_row = min(row0 + col, rows - 1u);
  const uint32_t my_token = kSelected ? token0 : token0 + my_row / a.group;
  const uint32_t my_head = g * a.group + (kSelected ? my_row : my_row % a.group);
  const uint32_t sees = kSelected || !a.causal ? visible : (uint32_t)max(0, (int32_t)(seen0 + my_row / a.group + 1u));
  const uint32_t all_see = kSelected || !a.causal ? visible : (uint32_t)max(0, (int32_t)(seen0 + row0 / a.group + 1u));

  const uint32_t chunk = max(128u, ((visible + a.splits - 1u) / a.splits + 31u) & ~31u);
  const uint32_t begin = min(piece * chunk, visible);
  const uint32_t end = min(begin + chunk, visible);

  uint4 q[kQ];
  {
    const char* p = a.queries + (int64_t)my_token * a.query_stride + (uint64_t)my_head * D * 2;
#pragma unroll
    for (int j = 0; j < kQ; ++j) {
      const uint32_t d = kFp8 ? 64u * (j / 2) + 16u * quad + 8u * (j % 2) : 32u * j + 8u * quad;
      q[j] = *reinterpret_cast<const uint4*>(p + d * 2);
    }
  }
  const char* key_base = a.cache.keys + g * a.cache.key_head + 16u * quad;
  const char* value_base = a.cache.values + g * a.cache.value_head + 16u * quad;
  const int32_t* pages = a.page_table + (int64_t)sequence * a.table_stride;
  const int64_t* list = kSelected ? a.indices + (int64_t)token0 * a.index_stride : nullptr;

  floatx4 o[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i) o[i] = floatx4{0.f, 0.f, 0.f, 0.f};
  float reference = kNoKeys;
  float total = 0.f;  // of this lane's keys
  char* mine = values[wave];
  uint32_t tr_place[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i)
    tr_place[i] = value_place<D>(4u * quad + (col >> 2), 2u * i + ((col & 3u) >> 1)) + 8u * (col & 1u);

  auto load = [&](Tile<kFp8, D>& t, uint32_t step) {
    const int32_t* at = table + step * kStep;
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const uint32_t row = (uint32_t)at[16 * h + col] & 0x7fffffffu;
      const char* kp = key_base + a.cache.key_offset(row);
      const char* vp = value_base + a.cache.value_offset(row);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) t.k[h][j] = *reinterpret_cast<const uint4*>(kp + 64 * j);
#pragma unroll
      for (int j = 0; j < kLoads; ++j) t.v[h][j] = *reinterpret_cast<const uint4*>(vp + 64 * j);
    }
    if constexpr (kFp8) {
      const uint32_t row = (uint32_t)at[lane & 31u] & 0x7fffffffu;
      t.scale = (lane < 32u ? a.cache.key_scales : a.cache.value_scales)[(uint64_t)row * a.cache.kv_heads + g];
    }
  };

  auto compute = [&](const Tile<kFp8, D>& t, uint32_t step, uint32_t base) {
    const int32_t* at = table + step * kStep;
    // Values to LDS, rows as they are.
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      bool drop = false;
      if constexpr (kSelected) drop = at[16 * h + col] < 0;  // padding's weight is 0, which NaN would survive
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        uint4 v = t.v[h][j];
        if (kSelected && drop) v = make_uint4(0u, 0u, 0u, 0u);
        if constexpr (kFp8) {
          const uint32_t c = 2u * (4u * j + quad);
          *reinterpret_cast<uint4*>(mine + value_place<D>(16u * h + col, c)) = fp8x8_to_bf16x8(make_uint2(v.x, v.y));
          *reinterpret_cast<uint4*>(mine + value_place<D>(16u * h + col, c + 1u)) = fp8x8_to_bf16x8(make_uint2(v.z, v.w));
        } else {
          *reinterpret_cast<uint4*>(mine + value_place<D>(16u * h + col, 4u * j + quad)) = v;
        }
      }
    }
    if constexpr (kFp8) scales[wave][lane] = t.scale;
    wave_order();
    // Scores of keys 16 h + 4 quad + i, in powers of two.
    float x[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      floatx4 s = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int j = 0; j < kLoads; ++j) {
        const uint4 k = t.k[h][j];
        if constexpr (kFp8) {
          s = mfma_16x16x32(Tag{}, fp8x8_to_bf16x8(make_uint2(k.x, k.y)), q[2 * j], s);
          s = mfma_16x16x32(Tag{}, fp8x8_to_bf16x8(make_uint2(k.z, k.w)), q[2 * j + 1], s);
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
      if constexpr (kSelected) {
        const int4 r = *reinterpret_cast<const int4*>(&at[16 * h + 4 * quad]);
        x[4 * h] = r.x < 0 ? -INFINITY : x[4 * h];
        x[4 * h + 1] = r.y < 0 ? -INFINITY : x[4 * h + 1];
        x[4 * h + 2] = r.z < 0 ? -INFINITY : x[4 * h + 2];
        x[4 * h + 3] = r.w < 0 ? -INFINITY : x[4 * h + 3];
      }
    }
    const uint32_t key0 = base + step * kStep;
    if (!kSelected && key0 + kStep > min(all_see, end)) {
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

  for (uint32_t base = begin; base < end; base += kSpan) {
    const uint32_t n = min((uint32_t)kSpan, end - base);
    const uint32_t steps = (n + kStep - 1) / kStep;
    if (base != begin) __syncthreads();
    for (uint32_t i = threadIdx.x; i < steps * kStep; i += 256u) {
      if constexpr (kSelected) {
        const int64_t key = i < n ? list[base + i] : -1;
        const bool named = key >= 0 && key < (int64_t)length;
        const uint32_t row = cache_row(a, pages, named ? (uint32_t)key : 0u);
        table[i] = (int32_t)(row | (named ? 0u : 0x80000000u));
      } else {
        table[i] = (int32_t)cache_row(a, pages, min(base + i, end - 1u));
      }
    }
    __syncthreads();
    Tile<kFp8, D> t0, t1;
    uint32_t step = wave;
    if (step < steps) {
      load(t0, step);
      while (true) {
        // the next step's loads run under this one's products; past the end they repeat the last
        load(t1, min(step + 4u, steps - 1u));
        compute(t0, step, base);
        step += 4u;
        if (step >= steps) break;
        load(t0, min(step + 4u, steps - 1u));
        compute(t1, step, base);
        step += 4u;
        if (step >= steps) break;
      }
    }
  }

  // Join the four waves: every wave scales its sums to the largest reference.
  total += __shfl_xor(total, 16, kWave);
  total += __shfl_xor(total, 32, kWave);
  if (quad == 0) sums[wave][col] = make_float2(reference, total);
  __syncthreads();
  float most = sums[0][col].x;
#pragma unroll
  for (int w = 1; w < 4; ++w) most = fmaxf(most, sums[w][col].x);
  const float shrink = exp2_fast(reference - most);
#pragma unroll
  for (int i = 0; i < kO; ++i)
    *reinterpret_cast<floatx4*>(mine + col * (D * 4) + (((4u * i + quad) ^ col) << 4)) = o[i] * shrink;
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < 16u * (D / 4); i += 256u) {
    const uint32_t r = i / (D / 4);
    const uint32_t c = i % (D / 4);
    if (row0 + r >= rows) break;
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
    float top = sums[0][r].x;
#pragma unroll
    for (int w = 1; w < 4; ++w) top = fmaxf(top, sums[w][r].x);
    float weight = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w) {
      sum += *reinterpret_cast<const floatx4*>(values[w] + r * (D * 4) + ((c ^ r) << 4));
      weight += sums[w][r].y * exp2_fast(sums[w][r].x - top);
    }
    const uint32_t token = kSelected ? token0 : token0 + (row0 + r) / a.group;
    const uint32_t head = g * a.group + (kSelected ? row0 + r : (row0 + r) % a.group);
    if (a.splits > 1)
      store_part<D, true>(a, token, head, piece, 4u * c, sum, top, weight);
    else
      store_out<Tag, D>(a, token, head, 4u * c, sum, top, weight);
  }
  if (a.splits == 1) return;

  // The tile's last piece to finish joins them all, in the order of the pieces:
  // the same bits whichever it is.  The pieces are stored and loaded past the
  // XCDs' own L2s, so no cache is written back or dropped (a release and an
  // acquire of agent scope here took 140 us of a 385 us step): each wave waits for
  // its stores, the counter is raised after all four waves have, and what the
  // last workgroup loads depends on the counter it read.
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __syncthreads();
  if (threadIdx.x == 0) {
    uint32_t* arrived = a.arrived + (item * a.cache.kv_heads + g);
    const uint32_t before = __hip_atomic_fetch_add(arrived, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    last_piece = before + 1u == a.splits;
    if (before + 1u == a.splits) __hip_atomic_store(arrived, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
  __syncthreads();
  if (!last_piece) return;
  const uint32_t live = min(16u, rows - row0);
  auto row_of = [&](uint32_t r) {
    const uint64_t token = kSelected ? token0 : token0 + (row0 + r) / a.group;
    return token * a.heads + g * a.group + (kSelected ? row0 + r : (row0 + r) % a.group);
  };
  float* weights = reinterpret_cast<float*>(values[0]);  // [16][splits]
  static_assert(sizeof(values) >= 16 * kMostSplits * sizeof(float), "weights of the pieces");
  {
    const uint32_t r = threadIdx.x / 16u;
    float top = kNoKeys;
    float sum = 0.f;
    if (r < live) {
      const float2* part = a.part_sum + row_of(r) * a.splits;
      for (uint32_t p = threadIdx.x % 16u; p < a.splits; p += 16u) top = fmaxf(top, load_shared(part + p).x);
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) top = fmaxf(top, __shfl_xor(top, off, kWave));
      for (uint32_t p = threadIdx.x % 16u; p < a.splits; p += 16u) {
        const float2 s = load_shared(part + p);
        const float w = exp2_fast(s.x - top);
        weights[r * a.splits + p] = w;
        sum += s.y * w;
      }
#pragma unroll
      for (int off = 8; off > 0; off >>= 1) sum += __shfl_xor(sum, off, kWave);
      if (threadIdx.x % 16u == 0) sums[0][r] = make_float2(top, sum);
    }
  }
  __syncthreads();
  for (uint32_t i = threadIdx.x; i < live * (D / 4); i += 256u) {
    const uint32_t r = i / (D / 4);
    const uint32_t c = i % (D / 4);
    const uint64_t row = row_of(r);
    const float* part = a.part_out + row * a.splits * D + 4u * c;
    floatx4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 8
    for (uint32_t p = 0; p < a.splits; ++p) {
      const float2* o2 = reinterpret_cast<const float2*>(part + (uint64_t)p * D);
      const float2 lo = load_shared(o2);
      const float2 hi = load_shared(o2 + 1);
      sum += floatx4{lo.x, lo.y, hi.x, hi.y} * weights[r * a.splits + p];
    }
    store_out<Tag, D>(a, (uint32_t)(row / a.heads), (uint32_t)(row % a.heads), 4u * c, sum, sums[0][r].x, sums[0][r].y);
  }
}

// The chunk kernel's pieces of one (token, head) row: references to their maximum, sums
// and outputs scaled to it and added in the order of the pieces.
template <class Tag, int D>
__global__ __launch_bounds__(256) void paged_combine_kernel(PagedAttentionArgs a) {
  constexpr uint32_t kLanes = D / 4;
  constexpr uint32_t kGroups = 256 / kLanes;
  __shared__ floatx4 sums[256];
  const uint32_t lane = lane_id();
  const uint64_t row = blockIdx.x;
  if (a.starts) {  // a mixed batch: the stream kernel's rows are not in these pieces
    const uint32_t rows = tokens_of(a, sequence_of(a, blockIdx.x / a.heads)).count * a.group;
    if (rows < a.least_rows) return;
  }
  const float2* part = a.part_sum + row * a.splits;
  float top = kNoKeys;
  for (uint32_t p = lane; p < a.splits; p += kWave) top = fmaxf(top, part[p].x);
  top = wave_max(top);
  float total = 0.f;
  for (uint32_t p = lane; p < a.splits; p += kWave) total += part[p].y * exp2_fast(part[p].x - top);
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, kWave);
  const uint32_t c = threadIdx.x % kLanes;
  floatx4 o = {0.f, 0.f, 0.f, 0.f};
  for (uint32_t p = threadIdx.x / kLanes; p < a.splits; p += kGroups) {
    const float2 s = part[p];
    if (s.y == 0.f) continue;
    o += *reinterpret_cast<const floatx4*>(a.part_out + (row * a.splits + p) * D + 4u * c) * exp2_fast(s.x - top);
  }
  sums[threadIdx.x] = o;
  __syncthreads();
  if (threadIdx.x >= kLanes) return;
  for (uint32_t i = 1; i < kGroups; ++i) o += sums[i * kLanes + c];
  store_out<Tag, D>(a, (uint32_t)(row / a.heads), (uint32_t)(row % a.heads), 4u * c, o, top, total);
}

template <class Tag, bool kFp8, bool kSelected>
void launch_stream(const PagedAttentionArgs& a, int32_t dim, uint32_t grid, hipStream_t s) {
  if (dim == 64)
    hipLaunchKernelGGL((paged_stream_kernel<Tag, kFp8, 64, kSelected>), dim3(grid), dim3(256), 0, s, a);
  else if (dim == 128)
    hipLaunchKernelGGL((paged_stream_kernel<Tag, kFp8, 128, kSelected>), dim3(grid), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((paged_stream_kernel<Tag, kFp8, 256, kSelected>), dim3(grid), dim3(256), 0, s, a);
}

template <class Tag>
void launch_combine(const PagedAttentionArgs& a, int32_t dim, hipStream_t s) {
  const dim3 grid(a.tokens * a.heads);
  if (dim == 64)
    hipLaunchKernelGGL((paged_combine_kernel<Tag, 64>), grid, dim3(256), 0, s, a);
  else if (dim == 128)
    hipLaunchKernelGGL((paged_combine_kernel<Tag, 128>), grid, dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((paged_combine_kernel<Tag, 256>), grid, dim3(256), 0, s, a);
}

int combine(const PagedAttentionArgs& a, int32_t dim, int32_t dtype, hipStream_t s) {
  if (a.splits == 1) return 0;
  if (dtype == kBF16)
    launch_combine<Bf16Tag>(a, dim, s);
  else
    launch_combine<F16Tag>(a, dim, s);
  return check_launch("paged_combine_kernel");
}

template <bool kSelected>
int launch(const PagedAttentionArgs& a, const dsa_paged_cache* cache, int32_t dtype, int64_t items, hipStream_t s) {
  const int64_t grid = items * a.splits * a.cache.kv_heads;
  DSA_REQUIRE(grid < (1LL << 31), "too many tokens for one call");
  const int32_t dim = cache->head_dim;
  if (cache->dtype == kFP8E4M3)
    launch_stream<Bf16Tag, true, kSelected>(a, dim, (uint32_t)grid, s);
  else if (dtype == kBF16)
    launch_stream<Bf16Tag, false, kSelected>(a, dim, (uint32_t)grid, s);
  else
    launch_stream<F16Tag, false, kSelected>(a, dim, (uint32_t)grid, s);
  return check_launch("paged_stream_kernel");
}

// Pieces of each row's keys: enough workgroups to fill the GPU `rounds` times,
// none of fewer than `least` keys.
uint32_t splits_for(int64_t workgroups, int64_t want_workgroups, int64_t most_keys, int64_t least) {
  const int64_t want = (want_workgroups + workgroups - 1) / workgroups;
  const int64_t most = (most_keys + least - 1) / least;
  const int64_t splits = want < most ? want : most;
  return (uint32_t)(splits < 1 ? 1 : splits > kMostSplits ? kMostSplits : splits);
}

// Counters first, at one place for every shape, then the pieces.
int64_t part_bytes(int64_t rows, int64_t splits, int64_t dim) {
  return splits > 1 ? kMostTiles * 4 + rows * splits * (dim + 2) * 4 : 0;
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
  DSA_REQUIRE(columns > 0 && columns < (1LL << 31) && columns * cache->page_size < (1LL << 31) && table_stride >= columns,
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

int take_workspace(PagedAttentionArgs& a, int64_t dim, void* workspace, int64_t bytes) {
  if (a.splits == 1) return 0;
  const int64_t rows = (int64_t)a.tokens * a.heads;
  if (!workspace || bytes < part_bytes(rows, a.splits, dim) || reinterpret_cast<uintptr_t>(workspace) % 16)
    return fail(DSA_STATUS_WORKSPACE_TOO_SMALL, "paged attention needs %lld bytes of 16-byte aligned workspace",
                (long long)part_bytes(rows, a.splits, dim));
  a.arrived = static_cast<uint32_t*>(workspace);
  a.part_out = reinterpret_cast<float*>(a.arrived + kMostTiles);
  a.part_sum = reinterpret_cast<float2*>(a.part_out + rows * a.splits * dim);
  return 0;
}

constexpr int64_t kStreamRows = 16;  // most rows of a sequence that the stream kernel takes

struct Plan {
  int64_t stream_items, chunk_items;  // 0: no sequence of that kind
  uint32_t stream_splits, chunk_splits;
};

Plan dense_plan(int64_t sequences, int64_t tokens, int64_t heads, int64_t kv_heads, int64_t capacity, bool uniform) {
  const int64_t group = heads / kv_heads;
  Plan p = {0, 0, 1, 1};
  const int64_t each = tokens / sequences * group;
  if (!uniform || each <= kStreamRows) p.stream_items = uniform ? sequences : (tokens < sequences ? tokens : sequences);
  if (!uniform || each > kStreamRows) p.chunk_items = row_tiles(sequences, tokens, group, uniform, kChunkRows);
  if (p.stream_items) p.stream_splits = splits_for(p.stream_items * kv_heads, kMostTiles, capacity, 128);
  if (p.chunk_items) p.chunk_splits = splits_for(p.chunk_items * kv_heads, 512, capacity, 256);
  return p;
}

struct SelectedPlan {
  int64_t items;
  uint32_t splits;
};

SelectedPlan selected_plan(int64_t tokens, int64_t heads, int64_t kv_heads, int64_t k) {
  const int64_t items = tokens * ((heads / kv_heads + 15) / 16);
  return {items, splits_for(items * kv_heads, kMostTiles, k, 128)};
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
  const Plan p = dense_plan(sequences, tokens, heads, cache->kv_heads, columns * cache->page_size, uniform != 0);
  return part_bytes(tokens * heads, p.stream_splits > p.chunk_splits ? p.stream_splits : p.chunk_splits, cache->head_dim);
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
  const Plan p = dense_plan(sequences, tokens, heads, cache->kv_heads, columns * cache->page_size, !starts);
  a.causal = causal != 0;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  hipStream_t s = static_cast<hipStream_t>(stream);
  // A sequence of few rows (one decoded token, a few drafted ones) is bound by
  // reading its cache, one of many by the products: a mixed batch has both.
  if (p.stream_items) {
    a.splits = p.stream_splits;
    a.least_rows = 1;
    a.most_rows = kStreamRows;
    if (int st = take_workspace(a, cache->head_dim, workspace, workspace_bytes)) return st;
    if (int st = launch<false>(a, cache, dtype, p.stream_items, s)) return st;
  }
  if (p.chunk_items) {
    a.splits = p.chunk_splits;
    a.least_rows = kStreamRows + 1;
    a.most_rows = 0xffffffffu;
    if (int st = take_workspace(a, cache->head_dim, workspace, workspace_bytes)) return st;
    const int64_t grid = p.chunk_items * a.splits * a.cache.kv_heads;
    DSA_REQUIRE(grid < (1LL << 31), "too many tokens for one call");
    if (int st = launch_paged_chunk(a, cache->head_dim, cache->dtype, (uint32_t)grid, s)) return st;
    return combine(a, cache->head_dim, dtype, s);
  }
  return 0;
}

extern "C" int64_t dsa_paged_selected_workspace_bytes(const dsa_paged_cache* cache, int64_t tokens, int32_t heads,
                                                      int64_t k) {
  if (!sizes_valid(cache, 1, tokens, heads)) return 0;
  const SelectedPlan p = selected_plan(tokens, heads, cache->kv_heads, k);
  return part_bytes(tokens * heads, p.splits, cache->head_dim);
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
  const SelectedPlan p = selected_plan(tokens, heads, cache->kv_heads, k);
  a.splits = p.splits;
  a.indices = indices;
  a.index_stride = index_stride;
  a.k = (uint32_t)k;
  a.out = static_cast<char*>(out);
  a.lse = lse;
  if (int st = take_workspace(a, cache->head_dim, workspace, workspace_bytes)) return st;
  return launch<true>(a, cache, dtype, p.items, static_cast<hipStream_t>(stream));
}
