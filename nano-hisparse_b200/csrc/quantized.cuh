// What the kernels of an 8-bit cache share: the record of a row and its codes.
// include/hisparse_quantized.h has the layout and the formulas.
#pragma once

#include "common.cuh"
#include "hisparse_quantized.h"

namespace hs {

constexpr int kQuantMaxDim = 256;
constexpr int kLowestExponent = -100;  // of a scale: weights and sums stay inside fp32 (attend)

__host__ __device__ __forceinline__ int64_t record_bytes(int kv_heads, int head_dim) {
  return ((int64_t)kv_heads * (head_dim + 1) + 31) / 32 * 32;
}

// 2^e for e in -126 .. 127
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }
// The scale that a record's byte stands for.
__device__ __forceinline__ float scale_of(unsigned byte) { return __int_as_float((int)byte << 23); }

// The smallest e >= kLowestExponent with largest <= 448 * 2^e; 448 = 1.75 * 2^8, so it
// takes one more than the exponent's difference where the fraction is above 1.75. A
// subnormal (or 0) falls to the lowest.
__device__ __forceinline__ int exponent_of(float largest) {
  const int bits = __float_as_int(largest);
  const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
  return e < kLowestExponent ? kLowestExponent : e;
}

// Four e4m3 codes of four numbers, the first in the lowest byte; NaN becomes NaN.
__device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d) {
  uint32_t r;
  asm("{\n .reg .b16 lo, hi;\n cvt.rn.satfinite.e4m3x2.f32 lo, %2, %1;\n"
      " cvt.rn.satfinite.e4m3x2.f32 hi, %4, %3;\n mov.b32 %0, {lo, hi};\n}\n"
      : "=r"(r)
      : "f"(a), "f"(b), "f"(c), "f"(d));
  return r;
}
// Two fp16 pairs of four codes (every e4m3 number is one of fp16).
__device__ __forceinline__ uint2 decode4(uint32_t codes) {
  uint2 r;
  asm("{\n .reg .b16 lo, hi;\n mov.b32 {lo, hi}, %2;\n cvt.rn.f16x2.e4m3x2 %0, lo;\n"
      " cvt.rn.f16x2.e4m3x2 %1, hi;\n}\n"
      : "=r"(r.x), "=r"(r.y)
      : "r"(codes));
  return r;
}
__device__ __forceinline__ float4 decode4_f32(uint32_t codes) {
  const uint2 h = decode4(codes);
  const float2 lo = __half22float2(*reinterpret_cast<const __half2 *>(&h.x));
  const float2 hi = __half22float2(*reinterpret_cast<const __half2 *>(&h.y));
  return make_float4(lo.x, lo.y, hi.x, hi.y);
}
__device__ __forceinline__ float decode1(unsigned char code) {
  return decode4_f32((uint32_t)code).x;
}

__device__ __forceinline__ float max_nan(float a, float b) {  // NaN if one is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}

// log2 of the page size where it is a power of two, else -1
inline int page_shift_of(int page_size) {
  int shift = -1;
  if ((page_size & (page_size - 1)) == 0)
    for (int sh = 0; sh < 31; ++sh)
      if ((1 << sh) == page_size) shift = sh;
  return shift;
}
// Index among all records of physical row `row`'s K record (V: page_size further); -1
// for a row that is padding or outside the pool.
__device__ __forceinline__ int64_t record_index(int64_t row, int page_size, int page_shift,
                                                int64_t pool_blocks, int32_t *status) {
  if (row < 0) return -1;
  int64_t block, within;
  if (page_shift >= 0) {
    block = row >> page_shift;
    within = row & (page_size - 1);
  } else {
    block = row / page_size;
    within = row - block * page_size;
  }
  if (block >= pool_blocks) {
    flag(status, HS_DEV_ROW_OUT_OF_RANGE);
    return -1;
  }
  return block * 2 * page_size + within;
}

}  // namespace hs
