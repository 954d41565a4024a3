// The paged key/value cache as the kernels see it (append, attention).
//
// A cache row is one token's keys or values of every kv head; row r is slot
// r % page_size of page r / page_size.  Position p of a sequence is row
// page_table[p / page_size] * page_size + p % page_size.  Heads are contiguous
// runs of head_dim elements, 16-byte aligned; pages, slots and heads lie at any
// strides.  e4m3 caches keep one fp32 scale per (page, slot, head), contiguous.
// e2m1 caches hold two codes a byte, the first in the low half, and one power of
// two (e8m0, the byte less 127; 255: the block is NaN) per kPowerDims of them in
// contiguous [pages][kv_heads][page_size][head_dim / kPowerDims]: a page's of one
// head lie together, as one workgroup reads them.
#pragma once

#include <float.h>

#include "common.hpp"
#include "dsa_amd.h"
#include "status.hpp"

namespace dsa {

// How a cache holds its elements.
enum Store { k16Bit, kE4M3, kE2M1 };
constexpr int kPowerDims = 32;  // dims that share a power of two of an e2m1 cache
template <Store kStore, int D>
constexpr int kRowBytes = kStore == kE2M1 ? D / 2 : kStore == kE4M3 ? D : 2 * D;  // of a head's keys or values

// Quotients of numbers below 2^31 by one divisor: a product and a shift.
struct Quotient {
  uint32_t factor, shift;
  __device__ __forceinline__ uint32_t operator()(uint32_t x) const { return (uint32_t)((uint64_t)x * factor >> shift); }
};

inline Quotient quotient_by(uint32_t divisor) {
  uint32_t shift = 31;
  while ((1ull << (shift - 31)) < divisor) ++shift;
  return {(uint32_t)(((1ull << shift) + divisor - 1) / divisor), shift};
}

struct PagedView {
  char* keys;
  char* values;
  float* key_scales;
  float* value_scales;
  uint8_t* key_powers;
  uint8_t* value_powers;
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
  // Of a head's first power of two.
  template <int D>
  __device__ __forceinline__ uint64_t power_offset(uint32_t row, uint32_t head) const {
    return ((((uint64_t)(row >> shift) * kv_heads + head) << shift) | (row & ((1u << shift) - 1u))) * (D / kPowerDims);
  }
};

// Checks a descriptor and fills the device view of it.
int make_paged_view(const dsa_paged_cache* cache, PagedView& view);

// The type of a cache's queries, and of the rows appended to it.
inline int32_t row_type(int32_t cache_dtype) {
  return cache_dtype == kFP8E4M3 || cache_dtype == kFP4E2M1 ? (int32_t)kBF16 : cache_dtype;
}

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

// 8 e2m1 codes times a power of two to 8 bf16, exactly (NaN for a power of NaN; infinite
// from 2^128 on, which powers from 2^126 on reach).
__device__ __forceinline__ uint4 fp4x8_to_bf16x8(uint32_t w, float power) {
  typedef __bf16 pair __attribute__((ext_vector_type(2)));
  const pair p0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 0);
  const pair p1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 1);
  const pair p2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 2);
  const pair p3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, power, 3);
  return make_uint4(__builtin_bit_cast(uint32_t, p0), __builtin_bit_cast(uint32_t, p1), __builtin_bit_cast(uint32_t, p2),
                    __builtin_bit_cast(uint32_t, p3));
}
__device__ __forceinline__ float power_of(uint32_t byte) { return __uint_as_float(byte << 23); }
// Codes of 8 whose values bf16 does not hold (4 and 6 under a power of 2^126, those from 2
// on under 2^127, all of a block that is NaN) become 0; whether there were any.
__device__ __forceinline__ bool drop_nonfinite_codes(uint32_t& codes, uint32_t power) {
  if (power < 253u) return false;
  uint32_t found = 0x11111111u;
  if (power < 255u) found &= (codes >> 2) & (power == 254u ? 0xffffffffu : codes >> 1);
  codes &= ~(found * 15u);
  return found != 0;
}

// LDS that the lanes of one wave share: a wave's LDS accesses are served in
// order, so only the compiler has to keep them so.
__device__ __forceinline__ void wave_order() {
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
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
