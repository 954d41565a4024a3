// The paged key/value cache as the kernels see it (append, attention).
//
// A cache row is one token's keys or values of every kv head; row r is slot
// r % page_size of page r / page_size.  Position p of a sequence is row
// page_table[p / page_size] * page_size + p % page_size.  Heads are contiguous
// runs of head_dim elements, 16-byte aligned; pages, slots and heads lie at any
// strides.  e4m3 caches keep one fp32 scale per (page, slot, head), contiguous.
#pragma once

#include <float.h>

#include "common.hpp"
#include "dsa_amd.h"
#include "status.hpp"

namespace dsa {

struct PagedView {
  char* keys;
  char* values;
  float* key_scales;
  float* value_scales;
  uint64_t key_head, value_head;  // bytes between heads
  uint32_t key_page, key_slot;    // bytes between pages and slots
  uint32_t value_page, value_slot;
  uint32_t pages;
  uint32_t shift;  // page_size = 1 << shift
  uint32_t kv_heads;

  __device__ __forceinline__ uint64_t key_offset(uint32_t row) const {
    return (uint64_t)(row >> shift) * key_page + (uint64_t)(row & ((1u << shift) - 1u)) * key_slot;
  }
  __device__ __forceinline__ uint64_t value_offset(uint32_t row) const {
    return (uint64_t)(row >> shift) * value_page + (uint64_t)(row & ((1u << shift) - 1u)) * value_slot;
  }
};

// Checks a descriptor and fills the device view of it.
int make_paged_view(const dsa_paged_cache* cache, PagedView& view);

// 2^x by the hardware instruction (results below the normal range become 0).
__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

struct Low {
  static constexpr bool value = false;
};
struct High {
  static constexpr bool value = true;
};

// 8 e4m3 codes to 8 bf16, exactly: two codes per instruction at a scale of 1.
__device__ __forceinline__ uint4 fp8x8_to_bf16x8_paired(uint2 v) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  auto two = [](uint32_t w, auto high) {
    const pair p = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8((int)w, 1.0f, decltype(high)::value);
    return __builtin_bit_cast(uint32_t, p);
  };
  return make_uint4(two(v.x, Low{}), two(v.x, High{}), two(v.y, Low{}), two(v.y, High{}));
}

// Two fp32 rounded to nearest-even bf16 or fp16, packed.
__device__ __forceinline__ uint32_t pack2(Bf16Tag, float lo, float hi) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  const floatx2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pair));
}
__device__ __forceinline__ uint32_t pack2(F16Tag, float lo, float hi) {
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
  const floatx2 v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, pair));
}
__device__ __forceinline__ float2 unpack2(Bf16Tag, uint32_t v) {
  return make_float2(__uint_as_float(v << 16), __uint_as_float(v & 0xffff0000u));
}
__device__ __forceinline__ float2 unpack2(F16Tag, uint32_t v) {
  typedef _Float16 pair __attribute__((ext_vector_type(2)));
  const pair p = __builtin_bit_cast(pair, v);
  return make_float2((float)p[0], (float)p[1]);
}

}  // namespace dsa
