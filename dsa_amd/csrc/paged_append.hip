// Appending new tokens to a paged key/value cache, positions rotated on the way.
//
// Pair (i, i + half) of a key's first rope_dim = 2 half dims is turned by the
// angle a = position * theta^(-i / half):
//   x'[i] = x[i] cos a - x[i + half] sin a
//   x'[i + half] = x[i + half] cos a + x[i] sin a
// in fp32, rounded once to the cache's type; values are stored as they are.
// An e4m3 cache takes s = max(max|x| / 448, 2^-126) of each head and stores
// rn(x / s) and s.  The queries' heads can be turned by the same angles in the
// same launch.  The angle's turns are taken in double and reduced there: in fp32
// an angle near 10^5 is off by 0.01.
#include <math.h>

#include "paged.hpp"

namespace dsa {

int make_paged_view(const dsa_paged_cache* c, PagedView& v) {
  DSA_REQUIRE(c && c->keys && c->values, "the paged cache has no keys or values");
  DSA_REQUIRE(c->dtype == kBF16 || c->dtype == kF16 || c->dtype == kFP8E4M3,
              "a paged cache is bf16, fp16 or fp8 e4m3 (got %d)", c->dtype);
  const bool fp8 = c->dtype == kFP8E4M3;
  DSA_REQUIRE(!fp8 || (c->key_scales && c->value_scales), "an fp8 paged cache needs key and value scales");
  DSA_REQUIRE(c->page_size > 0 && (c->page_size & (c->page_size - 1)) == 0, "page_size %d must be a power of two",
              c->page_size);
  DSA_REQUIRE(c->head_dim == 64 || c->head_dim == 128 || c->head_dim == 256, "head_dim %d must be 64, 128 or 256",
              c->head_dim);
  DSA_REQUIRE(c->kv_heads > 0 && c->kv_heads <= 1024, "kv_heads %d out of range", c->kv_heads);
  DSA_REQUIRE(c->pages > 0 && c->pages * (int64_t)c->page_size < (1LL << 31), "pages * page_size must be in 1..2^31 - 1");
  const int64_t e = fp8 ? 1 : 2;
  const int64_t strides[6] = {c->key_page_stride, c->key_slot_stride, c->key_head_stride,
                              c->value_page_stride, c->value_slot_stride, c->value_head_stride};
  for (int i = 0; i < 6; ++i) {
    DSA_REQUIRE(strides[i] >= 0 && strides[i] * e % 16 == 0, "paged cache strides must be non-negative multiples of 16 bytes");
    DSA_REQUIRE(i % 3 == 2 || strides[i] * e < (1LL << 32), "page and slot strides must be below 4 GiB");
  }
  DSA_REQUIRE(reinterpret_cast<uintptr_t>(c->keys) % 16 == 0 && reinterpret_cast<uintptr_t>(c->values) % 16 == 0,
              "the paged cache must be 16-byte aligned");
  v.keys = static_cast<char*>(c->keys);
  v.values = static_cast<char*>(c->values);
  v.key_scales = fp8 ? c->key_scales : nullptr;
  v.value_scales = fp8 ? c->value_scales : nullptr;
  v.key_page = (uint32_t)(c->key_page_stride * e);
  v.key_slot = (uint32_t)(c->key_slot_stride * e);
  v.key_head = (uint64_t)(c->key_head_stride * e);
  v.value_page = (uint32_t)(c->value_page_stride * e);
  v.value_slot = (uint32_t)(c->value_slot_stride * e);
  v.value_head = (uint64_t)(c->value_head_stride * e);
  v.pages = (uint32_t)c->pages;
  v.shift = (uint32_t)__builtin_ctz((unsigned)c->page_size);
  v.kv_heads = (uint32_t)c->kv_heads;
  return 0;
}

namespace {

constexpr float kE4M3Most = 448.f;
constexpr float kLeastScale = 0x1p-126f;

struct AppendArgs {
  PagedView cache;
  const char* keys;     // [tokens][kv_heads][dim], rows key_stride bytes apart
  const char* values;
  const char* queries;  // nullable: [tokens][heads][dim]
  char* out_queries;    // [tokens][heads][dim] dense
  int64_t key_stride, value_stride, query_stride;
  const int64_t* rows;
  const int64_t* positions;
  int64_t row_limit;
  uint32_t kv_heads, heads;
  uint32_t units;       // per token: 16 elements each of every key, value and query head
  uint32_t pack;        // tokens per workgroup
  int64_t tokens;
  uint32_t rope_dim;
  double octaves;       // log2(theta) / half
};

// A thread serves a unit, 16 elements of one head: two 8-element runs that turn
// into each other (i.. and i + half..), or 16 consecutive ones where nothing turns.
// So it loads and stores 16 bytes at a time, and a head's D/16 units are
// neighbouring lanes, which share its largest magnitude by shuffles.  A workgroup
// takes 256 units of one token, or as many whole tokens as it has threads for.
// HBM bound: 8192 tokens of 48 bf16 heads, 202 MB, 39 us (5.1 TB/s).
template <class Tag, bool kFp8, int D>
__global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a) {
  constexpr uint32_t kUnits = D / 16;
  __shared__ float2 turn[1024];  // [tokens of the workgroup][half], at most 256 / (2 kUnits) of D / 2
  const uint32_t half = a.rope_dim / 2;
  const uint32_t my = a.pack > 1u ? threadIdx.x / a.units : 0u;
  const uint32_t unit = a.pack > 1u ? threadIdx.x % a.units : blockIdx.y * 256u + threadIdx.x;
  const int64_t first = (int64_t)blockIdx.x * a.pack;
  const bool live = unit < a.units && my < a.pack && first + my < a.tokens;
  const int64_t token = live ? first + my : first;
  const uint32_t head = unit / kUnits;
  const uint32_t c = unit % kUnits;
  const int64_t row = a.rows[token];
  const bool is_key = head < a.kv_heads;
  const bool is_value = !is_key && head < 2 * a.kv_heads;
  const uint32_t h = is_key ? head : is_value ? head - a.kv_heads : head - 2 * a.kv_heads;
  const bool turned = !is_value && 8 * c < half;
  const uint32_t d0 = turned ? 8 * c : is_value ? 16 * c : a.rope_dim + 16 * (c - half / 8);
  const uint32_t d1 = turned ? d0 + half : d0 + 8;
  const char* from = is_key ? a.keys + token * a.key_stride
                     : is_value ? a.values + token * a.value_stride
                                : a.queries + token * a.query_stride;
  uint4 raw[2] = {};
  if (live) {
    raw[0] = *reinterpret_cast<const uint4*>(from + ((uint64_t)h * D + d0) * 2);
    raw[1] = *reinterpret_cast<const uint4*>(from + ((uint64_t)h * D + d1) * 2);
  }
  for (uint32_t i = threadIdx.x; i < a.pack * half; i += 256u) {
    const uint32_t at = i / half;
    const int64_t position = a.positions[min(first + at, (int64_t)a.tokens - 1)];
    const double turns = (double)position * exp2(-a.octaves * (double)(i - at * half)) * 0.15915494309189535;
    float s, co;
    sincospif((float)(2.0 * (turns - rint(turns))), &s, &co);
    turn[i] = make_float2(co, s);
  }
  __syncthreads();
  if (!live) return;
  float x[16];
#pragma unroll
  for (int p = 0; p < 2; ++p) {
    const uint32_t w[4] = {raw[p].x, raw[p].y, raw[p].z, raw[p].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float2 f = unpack2(Tag{}, w[i]);
      x[8 * p + 2 * i] = f.x;
      x[8 * p + 2 * i + 1] = f.y;
    }
  }
  if (turned) {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float2 t = turn[my * half + 8 * c + i];
      const float first = x[i], second = x[8 + i];
      x[i] = first * t.x - second * t.y;
      x[8 + i] = second * t.x + first * t.y;
    }
  }
  const bool in_cache = row >= 0 && row < a.row_limit;
  if (is_key || is_value) {
    const uint32_t r = in_cache ? (uint32_t)row : 0u;
    char* to = is_key ? a.cache.keys + a.cache.key_offset(r) + h * a.cache.key_head
                      : a.cache.values + a.cache.value_offset(r) + h * a.cache.value_head;
    if constexpr (kFp8) {
      float most = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(x[i]));
#pragma unroll
      for (int off = kUnits / 2; off > 0; off >>= 1) most = fmaxf(most, __shfl_xor(most, off, kWave));
      const float scale = fmaxf(most / kE4M3Most, kLeastScale);
      // The quotients by one reciprocal and a correction each: a third of the
      // instructions of sixteen divisions, which were as long as the memory's time.
      const float inverse = 1.f / scale;
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float q = x[i] * inverse;
        x[i] = fmaf(fmaf(-q, scale, x[i]), inverse, q);
      }
      uint32_t code[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        int v = __builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i], x[4 * i + 1], 0, false);
        code[i] = (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(x[4 * i + 2], x[4 * i + 3], v, true);
      }
      if (!in_cache) return;
      *reinterpret_cast<uint2*>(to + d0) = make_uint2(code[0], code[1]);
      *reinterpret_cast<uint2*>(to + d1) = make_uint2(code[2], code[3]);
      if (c == 0) (is_key ? a.cache.key_scales : a.cache.value_scales)[(uint64_t)r * a.kv_heads + h] = scale;
      return;
    }
    if (!in_cache) return;
    *reinterpret_cast<uint4*>(to + 2 * d0) = make_uint4(pack2(Tag{}, x[0], x[1]), pack2(Tag{}, x[2], x[3]),
                                                        pack2(Tag{}, x[4], x[5]), pack2(Tag{}, x[6], x[7]));
    *reinterpret_cast<uint4*>(to + 2 * d1) = make_uint4(pack2(Tag{}, x[8], x[9]), pack2(Tag{}, x[10], x[11]),
                                                        pack2(Tag{}, x[12], x[13]), pack2(Tag{}, x[14], x[15]));
    return;
  }
  char* to = a.out_queries + ((uint64_t)token * a.heads + h) * D * 2;
  *reinterpret_cast<uint4*>(to + 2 * d0) = make_uint4(pack2(Tag{}, x[0], x[1]), pack2(Tag{}, x[2], x[3]),
                                                      pack2(Tag{}, x[4], x[5]), pack2(Tag{}, x[6], x[7]));
  *reinterpret_cast<uint4*>(to + 2 * d1) = make_uint4(pack2(Tag{}, x[8], x[9]), pack2(Tag{}, x[10], x[11]),
                                                      pack2(Tag{}, x[12], x[13]), pack2(Tag{}, x[14], x[15]));
}

template <class Tag, bool kFp8>
void launch_append(const AppendArgs& a, int32_t dim, dim3 grid, hipStream_t stream) {
  if (dim == 64)
    hipLaunchKernelGGL((paged_append_kernel<Tag, kFp8, 64>), grid, dim3(256), 0, stream, a);
  else if (dim == 128)
    hipLaunchKernelGGL((paged_append_kernel<Tag, kFp8, 128>), grid, dim3(256), 0, stream, a);
  else
    hipLaunchKernelGGL((paged_append_kernel<Tag, kFp8, 256>), grid, dim3(256), 0, stream, a);
}

bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_paged_append(const dsa_paged_cache* cache, const void* keys, int64_t key_stride, const void* values,
                                int64_t value_stride, const void* queries, int64_t query_stride, void* out_queries,
                                int32_t heads, int32_t dtype, const int64_t* rows, const int64_t* positions,
                                int64_t tokens, int32_t rope_dim, double theta, void* stream) {
  AppendArgs a = {};
  if (int st = make_paged_view(cache, a.cache)) return st;
  DSA_REQUIRE(tokens >= 0 && tokens <= 0x7fffffffLL, "tokens out of range");
  if (tokens == 0) return 0;
  DSA_REQUIRE(keys && values && rows && positions, "null pointer argument");
  DSA_REQUIRE(!queries == !out_queries && (!queries || (heads > 0 && heads <= 65536)),
              "queries need an output and 1..65536 heads");
  DSA_REQUIRE(dtype == kBF16 || dtype == kF16, "appended rows are bf16 or fp16 (got %d)", dtype);
  DSA_REQUIRE(dtype == (cache->dtype == kFP8E4M3 ? kBF16 : cache->dtype),
              "appended rows must have the cache's type (bf16 for an fp8 cache)");
  const int32_t dim = cache->head_dim;
  DSA_REQUIRE(rope_dim >= 0 && rope_dim <= dim && rope_dim % 16 == 0, "rope_dim %d must be a multiple of 16 up to head_dim",
              rope_dim);
  DSA_REQUIRE(theta > 0 && isfinite(theta), "theta must be positive");
  const int64_t row = (int64_t)cache->kv_heads * dim;
  DSA_REQUIRE(key_stride >= row && value_stride >= row && key_stride % 8 == 0 && value_stride % 8 == 0 &&
                  (!queries || (query_stride >= (int64_t)heads * dim && query_stride % 8 == 0)),
              "token strides must cover the heads and be multiples of 8");
  DSA_REQUIRE(aligned16(keys) && aligned16(values) && aligned16(queries) && aligned16(out_queries),
              "appended rows must be 16-byte aligned");
  a.keys = static_cast<const char*>(keys);
  a.values = static_cast<const char*>(values);
  a.queries = static_cast<const char*>(queries);
  a.out_queries = static_cast<char*>(out_queries);
  a.key_stride = key_stride * 2;
  a.value_stride = value_stride * 2;
  a.query_stride = query_stride * 2;
  a.rows = rows;
  a.positions = positions;
  a.row_limit = cache->pages * cache->page_size;
  a.kv_heads = (uint32_t)cache->kv_heads;
  a.heads = queries ? (uint32_t)heads : 0u;
  a.units = (2 * a.kv_heads + a.heads) * (uint32_t)(dim / 16);
  a.rope_dim = (uint32_t)rope_dim;
  a.octaves = rope_dim ? log2(theta) / (rope_dim / 2) : 0.0;
  a.pack = a.units < 256 ? 256 / a.units : 1;
  a.tokens = tokens;
  const dim3 grid((unsigned)((tokens + a.pack - 1) / a.pack), (a.units + 255) / 256);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->dtype == kFP8E4M3)
    launch_append<Bf16Tag, true>(a, dim, grid, s);
  else if (dtype == kBF16)
    launch_append<Bf16Tag, false>(a, dim, grid, s);
  else
    launch_append<F16Tag, false>(a, dim, grid, s);
  return check_launch("paged_append_kernel");
}
