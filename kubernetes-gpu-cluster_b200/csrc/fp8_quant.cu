// Rows and matrices of 16 bits as 8-bit floating point with a scale for each block (fp8.cuh has the definition).
//
// Both are bound by their bytes, 2 in and 1 out for a number.  16-bit numbers x, m have at most 11 bits, so 448 x and t m (t half way between two
// codes, 5 bits) are integers of at most 17 bits on one grid: 448 x / m either is t or misses it by 2^-17 and more.  x fl(448 / m) is off by 2^-23
// at most, hence rounding it to 20 bits gives t where the quotient is t, and leaves it on its side of t elsewhere: one product and two integer
// operations in place of a division.
#include "fp8.cuh"
#include "kge.h"

namespace kge {
inline namespace KGE_ELT_NS {

#ifdef KGE_HALF
constexpr uint32_t kInf16 = 0x7c00u;
#else
constexpr uint32_t kInf16 = 0x7f80u;
#endif

__device__ __forceinline__ uint32_t mag2(uint4 v) {        // the largest magnitudes of the low and of the high halves
  constexpr uint32_t k = 0x7fff7fffu;
  return __vmaxu2(__vmaxu2(v.x & k, v.y & k), __vmaxu2(v.z & k, v.w & k));
}
// the largest magnitude of a block from that of its halves; infinity and NaN stay what they are
__device__ __forceinline__ float mag(uint32_t m2) { return bf_lo(max(m2 & 0xffffu, m2 >> 16)); }

__device__ __forceinline__ float scaled(float x, float factor) { return __uint_as_float((__float_as_uint(x * factor) + 8u) & ~15u); }
__device__ __forceinline__ uint2 codes8(uint4 v, float factor) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint32_t c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) c[k] = fp8::pack2(scaled(bf_lo(u[k]), factor), scaled(bf_hi(u[k]), factor));
  return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

// Eight lanes have a block of a row, 16 numbers each.
__global__ void __launch_bounds__(256)
fp8_quant_kernel(uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t scales_stride, const bf16* __restrict__ x, int64_t x_stride, const int32_t* __restrict__ rows,
                 int T, int K, int blocks) {
  pdl_launch_dependents();
  pdl_wait();
  const int64_t at = (int64_t)blockIdx.x * 32 + (threadIdx.x >> 3);      // which block of all
  const int t = (int)(at / blocks), b = (int)(at - (int64_t)t * blocks), k = b * fp8::kBlock + (threadIdx.x & 7) * 16;
  uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  const bool there = t < T && k < K;
  if (there) {
    const int64_t r = rows ? rows[t] : t;
    if (r >= 0) {
      const bf16* src = x + r * x_stride + k;
      v[0] = ld_nc_v4(src);
      v[1] = ld_nc_v4(src + 8);
    }
  }
  uint32_t m2 = __vmaxu2(mag2(v[0]), mag2(v[1]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m2 = __vmaxu2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
  if (!there) return;
  float scale, factor;
  fp8::scale_of(mag(m2), scale, factor);
  uint4 c = make_uint4(0, 0, 0, 0);
  if (factor > 0.f) {
    const uint2 lo = codes8(v[0], factor), hi = codes8(v[1], factor);
    c = make_uint4(lo.x, lo.y, hi.x, hi.y);
  }
  *reinterpret_cast<uint4*>(codes + (int64_t)t * K + k) = c;
  if ((threadIdx.x & 7) == 0) scales[b * scales_stride + t] = scale;
}

// A CTA has a block of 128 x 128, a thread 16 numbers of each of four rows (n, n + 32, ...).
__global__ void __launch_bounds__(256)
fp8_quant_weight_kernel(uint8_t* __restrict__ codes, float* __restrict__ scales, const bf16* __restrict__ w, int N, int K) {
  pdl_wait();
  __shared__ uint32_t part[8];
  const int k = blockIdx.x * fp8::kBlock + (threadIdx.x & 7) * 16, n0 = blockIdx.y * fp8::kBlock + (threadIdx.x >> 3);
  const int64_t base = (int64_t)blockIdx.z * N * K + k;
  uint4 v[4][2];
  uint32_t m2 = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + 32 * i;
    v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
    if (n < N && k < K) {
      const bf16* src = w + base + (int64_t)n * K;
      v[i][0] = ld_nc_v4(src);
      v[i][1] = ld_nc_v4(src + 8);
    }
    m2 = __vmaxu2(m2, __vmaxu2(mag2(v[i][0]), mag2(v[i][1])));
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m2 = __vmaxu2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = m2;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i) m2 = __vmaxu2(m2, part[i]);
  float scale, factor;
  fp8::scale_of(mag(m2), scale, factor);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int n = n0 + 32 * i;
    if (n < N && k < K) {
      uint4 c = make_uint4(0, 0, 0, 0);
      if (factor > 0.f) {
        const uint2 lo = codes8(v[i][0], factor), hi = codes8(v[i][1], factor);
        c = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
      *reinterpret_cast<uint4*>(codes + base + (int64_t)n * K) = c;
    }
  }
  if (threadIdx.x == 0) scales[((int64_t)blockIdx.z * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x] = scale;
}

static bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

}  // namespace KGE_ELT_NS
}  // namespace kge

using namespace kge;

extern "C" int KGE_API(kge_fp8_quant)(void* codes, float* scales, int scales_stride, const void* x, int x_stride, const int32_t* rows, int T, int K, void* stream) {
  KGE_REQUIRE(codes && scales && x, "kge_fp8_quant: null pointer");
  KGE_REQUIRE(K > 0 && K % 16 == 0, "kge_fp8_quant: K=%d must be a positive multiple of 16", K);
  KGE_REQUIRE(x_stride >= K && x_stride % 8 == 0, "kge_fp8_quant: rows of x %d apart (a multiple of 8, at least K = %d)", x_stride, K);
  KGE_REQUIRE(scales_stride >= T, "kge_fp8_quant: scales_stride=%d for %d rows", scales_stride, T);
  KGE_REQUIRE(aligned16(codes) && aligned16(x) && ((uintptr_t)scales & 3) == 0, "kge_fp8_quant: codes and x must be 16-byte aligned");
  if (T <= 0) return 0;
  const int blocks = (int)fp8::blocks(K);
  const int64_t ctas = ((int64_t)T * blocks + 31) / 32;
  KGE_REQUIRE(ctas < (1ll << 31), "kge_fp8_quant: %d rows of %d in one call", T, K);
  KGE_CUDA_OK(launch_pdl(fp8_quant_kernel, dim3((unsigned)ctas), dim3(256), 0, (cudaStream_t)stream, (uint8_t*)codes, scales, (int64_t)scales_stride, (const bf16*)x,
                         (int64_t)x_stride, rows, T, K, blocks));
  return 0;
}

extern "C" int KGE_API(kge_fp8_quant_weight)(void* codes, float* scales, const void* w, int E, int N, int K, void* stream) {
  KGE_REQUIRE(codes && scales && w, "kge_fp8_quant_weight: null pointer");
  KGE_REQUIRE(E > 0 && E <= 65535 && N > 0 && fp8::blocks(N) <= 65535, "kge_fp8_quant_weight: %d matrices of %d rows (up to 65535 of 65535 x 128)", E, N);
  KGE_REQUIRE(K > 0 && K % 16 == 0, "kge_fp8_quant_weight: K=%d must be a positive multiple of 16", K);
  KGE_REQUIRE(aligned16(codes) && aligned16(w) && ((uintptr_t)scales & 3) == 0, "kge_fp8_quant_weight: codes and w must be 16-byte aligned");
  KGE_CUDA_OK(launch_pdl(fp8_quant_weight_kernel, dim3((unsigned)fp8::blocks(K), (unsigned)fp8::blocks(N), E), dim3(256), 0, (cudaStream_t)stream, (uint8_t*)codes, scales,
                         (const bf16*)w, N, K));
  pdl_break_next();        // a product that is launched early reads weights before it waits for the kernel before it
  return 0;
}
