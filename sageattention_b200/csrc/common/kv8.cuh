// Element arithmetic of the paged 8-bit KV cache: e4m3 codes with one scale for each block of tokens and head.
//
// The scale of a block is the smallest power of two 2^e with max|x| <= 448 * 2^e.  A float format loses nothing by a scale
// that is a power of two (the codes keep their three mantissa bits whatever it is), and every step becomes exact but one:
// x * 2^-e is exact, the code is its one rounding, and code * 2^e is exact.  When a later token raises the scale of an
// open block, its older codes are rounded again to the new one, which changes only those that fall below 2^-6 * 2^e.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

namespace nvfp4 {

constexpr int kKv8MinExp = -110;   // of a block of zeros: the scale and its reciprocal stay normal floats

// 2^e for the block maximum whose float bits are `amax` (finite, >= 0).  448 = 1.75 * 2^8, so e is the exponent of amax
// less 8, one more where its mantissa is above 1.75.
__device__ __forceinline__ float kv8_scale(uint32_t amax) {
  int e = (int)(amax >> 23) - 127 - 8 + ((amax & 0x7FFFFFu) > 0x600000u ? 1 : 0);
  e = max(e, kKv8MinExp);           // zeros and subnormals
  return __uint_as_float((uint32_t)(e + 127) << 23);
}

// float bits of |x| where x is finite, else 0: an infinity takes the largest code and a NaN stays one, but neither makes a
// scale
__device__ __forceinline__ uint32_t kv8_magnitude(float x) {
  const uint32_t u = __float_as_uint(x) & 0x7FFFFFFFu;
  return u < 0x7F800000u ? u : 0u;
}

// the four e4m3 values of a word as two pairs of halves (exact)
__device__ __forceinline__ void half4_of_e4m3x4(uint32_t v, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 a, b;\n\t"
      "mov.b32 {a, b}, %2;\n\t"
      "cvt.rn.f16x2.e4m3x2 %0, a;\n\t"
      "cvt.rn.f16x2.e4m3x2 %1, b;\n\t}\n"
      : "=r"(lo), "=r"(hi)
      : "r"(v));
}

}  // namespace nvfp4
