// What the kernels of the paged key / value cache share: where a position lies, and the 8-bit form of a page.
//
// e4m3 keeps three bits behind the point at every size, so a power of two as a page's scale costs no precision: it only moves the range. What a page
// holds when later tokens need a larger one is brought to it by that power of two, which leaves every value as it was but those that come out below
// 2^-6, the least with all three bits.
#pragma once
#include "common.cuh"
#include "kernels_api.h"

namespace mdb {

// the page of a position of sequence b, or -1 where the table or the page number ends before it
__device__ __forceinline__ int page_of(const MdbPages& p, int b, int index) {
  if (index < 0 || index >= p.width) return -1;
  const int page = p.table[static_cast<long long>(b) * p.width + index];
  return page >= 0 && page < p.count ? page : -1;
}

// The scale of a page as a byte: the least power of two 2^(byte - 127) that brings `most` to 448 = 1.75 * 2^8 or less, and no denormal one
__device__ __forceinline__ int scale_byte(float most) {
  const uint32_t bits = __float_as_uint(most);
  return max(static_cast<int>(bits >> 23) - 8 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0), 1);
}
// 2^(byte - 127) and its inverse, for bytes of 1 to 253; a byte of 0 stands for 2^-127, of which fp32 without denormals makes nothing
__device__ __forceinline__ float scale_value(int byte) { return __uint_as_float(static_cast<uint32_t>(byte) << 23); }
__device__ __forceinline__ float scale_inverse(int byte) { return __uint_as_float(static_cast<uint32_t>(254 - byte) << 23); }

// two finite values or NaN in e4m3, rounded to nearest; the first in the low byte
__device__ __forceinline__ uint32_t pack_e4m3x2(float2 x) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(x.y), "f"(x.x));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {      // exact
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}
__device__ __forceinline__ float2 e4m3x2_to_float2(uint16_t v) {
  const uint32_t h = e4m3x2_to_f16x2(v);
  return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

}  // namespace mdb
