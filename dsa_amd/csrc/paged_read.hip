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
};

template <Store kStore, int D>
__global__ __launch_bounds__(256) void paged_read_kernel(ReadArgs a) {
  constexpr uint32_t kUnits = D / 8;
  const uint32_t units = a.cache.kv_heads * kUnits;
  const uint64_t at = (uint64_t)blockIdx.x * 256u + threadIdx.x;
  const uint64_t index = at / units;
  const uint32_t unit = (uint32_t)(at % units);
  if (index >= (uint64_t)a.count) return;
  const uint32_t head = unit / kUnits, c = unit % kUnits;
  const int64_t named = a.rows[index];
  const bool inside = named >= 0 && named < (int64_t)a.row_limit;
  const uint32_t row = inside ? (uint32_t)named : 0u;
#pragma unroll
  for (int which = 0; which < 2; ++which) {
    if (!a.out[which]) continue;
    const char* from = which ? a.cache.values + a.cache.value_offset(row) + head * a.cache.value_head
                             : a.cache.keys + a.cache.key_offset(row) + head * a.cache.key_head;
    uint4 v;
    if constexpr (kStore == kE2M1) {
      const uint8_t* powers = which ? a.cache.value_powers : a.cache.key_powers;
      const uint32_t power = powers[a.cache.power_offset<D>(row, head) + c / 4u];
      v = fp4x8_to_bf16x8(*reinterpret_cast<const uint32_t*>(from + 4u * c), power_of(power));
    } else if constexpr (kStore == kE4M3) {
      const float* scales = which ? a.cache.value_scales : a.cache.key_scales;
      const float scale = scales[(uint64_t)row * a.cache.kv_heads + head];
      const uint2 w = *reinterpret_cast<const uint2*>(from + 8u * c);
      auto two = [&](uint32_t bits) {
        const floatx2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)bits, false);
        const floatx2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)bits, true);
        return make_uint2(pack2(Bf16Tag{}, lo[0] * scale, lo[1] * scale), pack2(Bf16Tag{}, hi[0] * scale, hi[1] * scale));
      };
      const uint2 lo = two(w.x), hi = two(w.y);
      v = make_uint4(lo.x, lo.y, hi.x, hi.y);
    } else {
      v = *reinterpret_cast<const uint4*>(from + 16u * c);
    }
    if (!inside) v = make_uint4(0u, 0u, 0u, 0u);
    *reinterpret_cast<uint4*>(a.out[which] + at * 16u) = v;
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
  if (count == 0 || (!out_keys && !out_values)) return 0;
  DSA_REQUIRE(rows, "null pointer argument");
  DSA_REQUIRE(reinterpret_cast<uintptr_t>(out_keys) % 16 == 0 && reinterpret_cast<uintptr_t>(out_values) % 16 == 0,
              "outputs must be 16-byte aligned");
  a.rows = rows;
  a.count = count;
  a.row_limit = (uint32_t)(cache->pages * cache->page_size);
  a.out[0] = static_cast<char*>(out_keys);
  a.out[1] = static_cast<char*>(out_values);
  const int64_t grid = (count * cache->kv_heads * (cache->head_dim / 8) + 255) / 256;
  DSA_REQUIRE(grid < (1LL << 24), "too many rows for one call");
  hipStream_t s = static_cast<hipStream_t>(stream);
  if (cache->dtype == kFP4E2M1)
    launch_read<kE2M1>(a, cache->head_dim, (uint32_t)grid, s);
  else if (cache->dtype == kFP8E4M3)
    launch_read<kE4M3>(a, cache->head_dim, (uint32_t)grid, s);
  else
    launch_read<k16Bit>(a, cache->head_dim, (uint32_t)grid, s);
  return check_launch("paged_read_kernel");
}
