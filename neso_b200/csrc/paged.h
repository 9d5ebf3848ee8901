// Pieces shared by the kernels of the paged key-value cache: the cache's
// layout, 16-bit element types and host-side checks of the caches' arguments.
#pragma once

#include <cuda_bf16.h>

#include "runtime.h"

namespace neso {

// One half of a paged cache: element (page, head, token, d) lies at
// page * page_stride + head * head_stride + token * token_stride + d. All
// strides are in elements and 64-bit: a cache passes 2^31 elements easily.
struct PagedCache {
  void* base;
  int64_t page_stride;
  int64_t head_stride;
  int64_t token_stride;
};

// Elements are 16 bits wide and move as 16-byte vectors, so the base and
// every stride have to be multiples of 16 bytes.
inline int check_cache(const PagedCache& c, const char* name) {
  if (c.base == nullptr) return fail(NESO_ERR_INVALID_ARG, "%s is a null pointer", name);
  if (!aligned16(c.base) || c.page_stride % 8 != 0 || c.head_stride % 8 != 0 || c.token_stride % 8 != 0) {
    return fail(NESO_ERR_MISALIGNED, "%s and its page, head and token strides must be multiples of 16 bytes", name);
  }
  if (c.page_stride < 0 || c.head_stride < 0 || c.token_stride < 0) {
    return fail(NESO_ERR_INVALID_ARG, "%s has a negative stride", name);
  }
  return NESO_OK;
}

// A page size as a divisor of token indexes, which are below 2^31. With
// 2^shift >= size and mul = ceil(2^(32+shift) / size) = (2^(32+shift) + e) /
// size, e < size, t * mul / 2^(32+shift) exceeds t / size by
// t * e / (size * 2^(32+shift)) < 2^31 / 2^(32+shift) <= 1 / (2 size): too
// little to reach the next integer, so the shifted product is the quotient.
struct PageDivisor {
  uint32_t size;
  uint32_t shift;
  uint64_t mul;
};

inline PageDivisor page_divisor(uint32_t size) {
  PageDivisor d{size, 0, 0};
  while ((1ull << d.shift) < size) ++d.shift;
  d.mul = ((1ull << (32 + d.shift)) + size - 1) / size;
  return d;
}

__device__ __forceinline__ uint32_t page_of(const PageDivisor& d, uint32_t token) {
  // mul < 2^33: its bit 32 is token itself, the rest is a 32 x 32 product.
  const uint64_t lo = (static_cast<uint64_t>(token) * static_cast<uint32_t>(d.mul)) >> 32;
  const uint64_t hi = (d.mul >> 32) ? token : 0u;
  return static_cast<uint32_t>((hi + lo) >> d.shift);
}

// The two 16-bit types: pack with one rounding, unpack exactly.
template <bool kBf16>
__device__ __forceinline__ uint32_t pack16(float lo, float hi) {
  if (kBf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&h);
  }
  return pack_half2(lo, hi);
}
template <bool kBf16>
__device__ __forceinline__ float2 unpack16(uint32_t x) {
  if (kBf16) return make_float2(__uint_as_float(x << 16), __uint_as_float(x & 0xffff0000u));
  return __half22float2(*reinterpret_cast<const __half2*>(&x));
}
}  // namespace neso
