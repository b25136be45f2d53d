// 8-bit floating point (e4m3: 4 bits of exponent, 3 of mantissa, largest number 448) with a scale for each block of 128.
//
// A block with the largest magnitude m has the scale s = max(m / 448, 2^-126) in fp32, and a number x of it the code nearest to 448 x / m (to
// 2^126 x below that), ties to even.  A block with an infinity or NaN has the scale NaN and codes of zero, so every product with it is NaN.
#pragma once
#include "common.cuh"

namespace kge {
namespace fp8 {
constexpr int kBlock = 128;
constexpr float kMax = 448.f;
constexpr float kLeast = 1.17549435e-38f;                  // 2^-126
inline int64_t blocks(int64_t n) { return (n + kBlock - 1) / kBlock; }

#ifdef __CUDACC__
// two numbers as codes, the first in the low byte
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ uint32_t pack4(float a, float b, float c, float d) { return pack2(a, b) | pack2(c, d) << 16; }

// A block's scale and what its numbers are multiplied with, from its largest magnitude; an infinity or NaN gives NaN and zero.
// The scale is m / 448 rounded once: a product with 1 / 448 and what is left of m, which one fma gives exactly.  The factor is off by 2^-22 at most (a
// reciprocal within a last place of m / 16, which keeps both of them normal numbers).  Two divisions were two thirds of an eight-lane block's instructions.
__device__ __forceinline__ void scale_of(float m, float& scale, float& factor) {
  const bool fine = m <= 3.402823466e38f;
  constexpr float c = 1.f / kMax;
  float q = m * c;
  q = fmaf(fmaf(-kMax, q, m), c, q);
  float inv;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(fmaxf(m, kMax * kLeast) * 0.0625f));
  scale = fine ? fmaxf(q, kLeast) : __int_as_float(0x7fffffff);
  factor = fine ? inv * (kMax * 0.0625f) : 0.f;
}
#endif
}  // namespace fp8
}  // namespace kge
