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

// fp32 numbers of a block as codes.  A product with the factor is off by a few 2^-24 and may lie on the other side of half a step than 448 h / m does.  So a number's code
// is taken from just below and just above it, and four numbers of which one has two codes (1 in 50000) are marked and settled exactly.
struct Rows32 {
  float m, factor, below, above;                             // (m: no less than the magnitude that has the smallest scale)
  // The factor within a rounding, 2^-24, by a Newton step; with that of `below` and of the product, three together, 2^-22 is enough between them.
  __device__ __forceinline__ Rows32(float top, float f) : m(fmaxf(top, kMax * kLeast)) {
    factor = fmaf(fmaf(-m, f, kMax) * (1.f / kMax), f, f);
    below = factor * (1.f - 0x1p-22f);
    above = factor * (1.f + 0x1p-22f);
  }
  __device__ __forceinline__ uint32_t codes4(float a, float b, float c, float d, uint32_t& marked, int at) const {
    const uint32_t lo = pack4(a * below, b * below, c * below, d * below), hi = pack4(a * above, b * above, c * above, d * above);
    if (lo != hi) marked |= 1u << at;
    return lo;
  }
  // A number on h's side of every half step, or on it.  Those and the codes have four bits behind the first at most: of such numbers the product's nearest, t,
  // is either no half step or the one next to 448 h / m, and 448 h - t m (33 and 29 bits) has the sign of what is between them.
  __device__ __forceinline__ float settled(float h) const {
    const uint32_t t = (__float_as_uint(h * factor) + 0x40000u) & ~0x7ffffu;
    const double r = fma(-(double)fabsf(__uint_as_float(t)), (double)m, 448.0 * (double)fabsf(h));
    return __uint_as_float(t + (r > 0.0) - (r < 0.0));
  }
  __device__ __forceinline__ uint32_t settled4(float a, float b, float c, float d) const { return pack4(settled(a), settled(b), settled(c), settled(d)); }
};
#endif
}  // namespace fp8
}  // namespace kge
