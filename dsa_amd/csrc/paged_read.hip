// What rows of a paged cache stand for, in the type that rows are appended in.
//
// e4m3: code * scale, rounded once; e2m1: code * power, exact in bf16; 16 bits: the
// row itself.  A thread takes 8 elements of a key or value, so that the stores, four
// fifths of an e2m1 cache's bytes, are 16 neighbouring bytes a lane.
#include "paged.hpp"

namespace dsa {
namespace {

struct ReadArgs {
  PagedView cache;
  const int64_t* rows;
  int64_t count;
  uint32_t row_limit;
  char* out[2];  // keys, values; nullable
  Quotient by_units;
};

constexpr uint32_t kEach = 2;  // runs of a thread, of keys and of values each

template <Store kStore, int D>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadArgs a) {
  constexpr uint32_t kUnits = D / 8;
  const uint32_t units = a.cache.kv_heads * kUnits;
  const uint32_t all = (uint32_t)a.count * units;
  const uint32_t at = blockIdx.x * (256u * kEach) + threadIdx.x;
  uint32_t row[kEach], head[kEach];
  bool inside[kEach];
#pragma unroll
  for (uint32_t e = 0; e < kEach; ++e) {
    const uint32_t i = min(at + 256u * e, all - 1u);
    const uint32_t index = a.by_units(i);
    head[e] = (i - index * units) / kUnits;
    const int64_t named = a.rows[index];
    inside[e] = named >= 0 && named < (int64_t)a.row_limit;
    row[e] = inside[e] ? (uint32_t)named : 0u;
  }
  const uint32_t c = threadIdx.x % kUnits;  // (a workgroup starts on a head)
  u32x4 v[2][kEach];
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (!a.out[which]) continue;
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
      const char* from = which ? a.cache.values + a.cache.value_offset(row[e]) + head[e] * a.cache.value_head
                               : a.cache.keys + a.cache.key_offset(row[e]) + head[e] * a.cache.key_head;
      if constexpr (kStore == kE2M1) {
        const uint8_t* powers = which ? a.cache.value_powers : a.cache.key_powers;
        v[which][e][0] = *reinterpret_cast<const uint32_t*>(from + 4u * c);
        v[which][e][1] = powers[a.cache.power_offset<D>(row[e], head[e]) + c / 4u];
      } else if constexpr (kStore == kE4M3) {
        const float* scales = which ? a.cache.value_scales : a.cache.key_scales;
        const u32x2 w = *reinterpret_cast<const u32x2*>(from + 8u * c);
        v[which][e][0] = w[0], v[which][e][1] = w[1];
        v[which][e][2] = __float_as_uint(scales[(uint64_t)row[e] * a.cache.kv_heads + head[e]]);
      } else {
        v[which][e] = *reinterpret_cast<const u32x4*>(from + 16u * c);
      }
    }
  }
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (!a.out[which]) continue;
#pragma unroll
    for (uint32_t e = 0; e < kEach; ++e) {
      u32x4 x = v[which][e];
      if constexpr (kStore == kE2M1) {
        x = __builtin_bit_cast(u32x4, fp4x8_to_bf16x8(x[0], power_of(x[1])));
      } else if constexpr (kStore == kE4M3) {
        const float scale = __uint_as_float(x[2]);
        auto two = [&](uint32_t bits, bool high) {
          const floatx2 f = high ? __builtin_amdgcn_cvt_pk_f32_fp8((int)bits, true) : __builtin_amdgcn_cvt_pk_f32_fp8((int)bits, false);
          return pack2(Bf16Tag{}, f[0] * scale, f[1] * scale);
        };
        x = u32x4{two(x[0], false), two(x[0], true), two(x[1], false), two(x[1], true)};
      }
      if (!inside[e]) x = u32x4{0u, 0u, 0u, 0u};
      if (at + 256u * e < all) *reinterpret_cast<u32x4*>(a.out[which] + (uint64_t)(at + 256u * e) * 16u) = x;
    }
  }
}

template <Store kStore>
void launch_read(const ReadArgs& a, int32_t dim, uint32_t grid, hipStream_t s) {
  if (dim == 64)
    hipLaunchKernelGGL((paged_read_kernel<kStore, 64>), dim3(grid), dim3(256), 0, s, a);
  else if (dim == 128)
    hipLaunchKernelGGL((paged_read_kernel<kStore, 128>), dim3(grid), dim3(256), 0, s, a);
  else
    hipLaunchKernelGGL((paged_read_kernel<kStore, 256>), dim3(grid), dim3(256), 0, s, a);
}

}  // namespace
}  // namespace dsa

using namespace dsa;

extern "C" int dsa_paged_read(const dsa_paged_cache* cache, const int64_t* rows, int64_t count, void* out_keys,
                              void* out_values, void* stream) {
  ReadArgs a = {};
  if (int st = make_paged_view(cache, a.cache)) return st;
  DSA_REQUIRE(count >= 0 && count <= 0x7fffffffLL, "rows out of range");
  const int64_t units = cache->kv_heads * (int64_t)(cache->head_dim / 8);
  if (count == 0 || (!out_keys && !out_values)) return 0;
  DSA_REQUIRE(rows, "null pointer argument");
  DSA_REQUIRE(reinterpret_cast<uintptr_t>(out_keys) % 16 == 0 && reinterpret_cast<uintptr_t>(out_values) % 16 == 0,
              "outputs must be 16-byte aligned");
  a.rows = rows;
  a.count = count;
  a.row_limit = (uint32_t)(cache->pages * cache->page_size);
  a.out[0] = static_cast<char*>(out_keys);
  a.out[1] = static_cast<char*>(out_values);
  DSA_REQUIRE(count * units < (1LL << 31) - 512, "too many rows for one call");  // 32 GiB of keys
  a.by_units = quotient_by((uint32_t)units);
  const int64_t grid = (count * units + 256 * kEach - 1) / (256 * kEach);
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->dtype == kFP4E2M1)
    launch_read<kE2M1>(a, cache->head_dim, (uint32_t)grid, s);
  else if (cache->dtype == kFP8E4M3)
    launch_read<kE4M3>(a, cache->head_dim, (uint32_t)grid, s);
  else
    launch_read<k16Bit>(a, cache->head_dim, (uint32_t)grid, s);
  return check_launch("paged_read_kernel");
}
