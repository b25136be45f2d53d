// Rows and matrices of 16 bits as 8-bit floating point with a scale for each block (fp8.cuh has the definition).
//
// Both are bound by their bytes, 2 in and 1 out for a number.  16-bit numbers x, m have at most 11 bits, so 448 x and t m (t half way between two
// codes, 5 bits) are integers of at most 17 bits on one grid: 448 x / m either is t or misses it by 2^-17 and more.  x times the factor is off by less
// than 2^-21, hence rounding it to 20 bits gives t where the quotient is t, and leaves it on its side of t elsewhere: one product and two integer
// operations in place of a division.
#include "fp8.cuh"
#include "kge.h"

namespace kge {
inline namespace KGE_ELT_NS {

// The larger magnitudes of the low and of the high halves, under signs that mean nothing; NaN above all.
__device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.NaN.xorsign.abs." KGE_MMA_ELT "x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}
__device__ __forceinline__ uint32_t mag2(uint4 v) { return max2(max2(v.x, v.y), max2(v.z, v.w)); }
// the largest magnitude of a block from that of its halves
__device__ __forceinline__ float mag(uint32_t m2) { return fabsf(bf_lo(max2(m2, m2 >> 16))); }

// x factor, rounded to 20 bits
__device__ __forceinline__ float scaled(float x, float factor) { return __uint_as_float((__float_as_uint(x * factor) + 8u) & ~15u); }
__device__ __forceinline__ uint2 codes8(uint4 v, float factor) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint32_t c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) c[k] = fp8::pack2(scaled(bf_lo(u[k]), factor), scaled(bf_hi(u[k]), factor));
  return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

// Eight lanes have a block of a row, 16 numbers each, and go on to another 32 blocks a CTA further: the next block's numbers and the one after's row are
// under way meanwhile.  Bound by instructions (13 a number), not by the bytes: 16384 rows of 2048 gathered from 2048 (43 MB, 6.6 us) 22.9 us, 8192 rows of
// 4096 (101 MB, 15.5 us) 27.1; a block a thread and no more 24.9 and 30.8, two blocks at a time in 64 registers 24.3 and 28.6.
__global__ void __launch_bounds__(256, 6)
fp8_quant_kernel(uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t scales_stride, const bf16* __restrict__ x, int64_t x_stride, const int32_t* __restrict__ rows,
                 uint32_t units, int K, uint32_t blocks) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t step = gridDim.x * 32, step_t = step / blocks, step_b = step - step_t * blocks;
  const int lane_k = (threadIdx.x & 7) * 16;
  struct Place { uint32_t at, t, b; int row; };            // block number, row, block of the row; the row of x, below 0 for zeros
  auto look = [&](Place& p) {
    if (p.at < units) p.row = rows ? rows[p.t] : (int)p.t;
  };
  auto on = [&](const Place& p) {
    Place n{p.at + step, p.t + step_t, p.b + step_b, -1};
    if (n.b >= blocks) { n.b -= blocks; ++n.t; }
    return n;
  };
  auto load = [&](const Place& p, uint4 (&v)[2]) {
    v[0] = v[1] = make_uint4(0, 0, 0, 0);
    const int k = p.b * fp8::kBlock + lane_k;
    if (p.at < units && p.row >= 0 && k < K) {
      const bf16* src = x + p.row * x_stride + k;
      v[0] = ld_nc_v4(src);
      v[1] = ld_nc_v4(src + 8);
    }
  };
  Place now{blockIdx.x * 32 + (threadIdx.x >> 3), 0, 0, -1};
  now.t = now.at / blocks;
  now.b = now.at - now.t * blocks;
  look(now);
  Place next = on(now);
  look(next);
  uint4 v[2];
  load(now, v);
  while (__any_sync(0xffffffffu, now.at < units)) {
    uint4 w[2];
    load(next, w);
    Place then = on(next);
    look(then);
    uint32_t m2 = max2(mag2(v[0]), mag2(v[1]));
#pragma unroll
    for (int o = 4; o > 0; o >>= 1) m2 = max2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
    float scale, factor;
    fp8::scale_of(mag(m2), scale, factor);
    const int k = now.b * fp8::kBlock + lane_k;
    if (now.at < units && k < K) {
      uint4 c = make_uint4(0, 0, 0, 0);
      if (factor > 0.f) {
        const uint2 lo = codes8(v[0], factor), hi = codes8(v[1], factor);
        c = make_uint4(lo.x, lo.y, hi.x, hi.y);
      }
      *reinterpret_cast<uint4*>(codes + (int64_t)now.t * K + k) = c;
      if ((threadIdx.x & 7) == 0) scales[now.b * scales_stride + now.t] = scale;
    }
    v[0] = w[0]; v[1] = w[1];
    now = next; next = then;
  }
}

// A CTA takes steps of 128 rows x 256 columns (two blocks), copied three steps ahead into shared memory: every access to memory is a whole 512-byte piece
// of a row, or 256 bytes of codes, and loads are under way all the time.  (A block a CTA, from registers, 28672 x 4096: 98 us, 55 % of the copy's rate.)
constexpr int kWThreads = 512, kWStages = 3, kWStage = 128 * 256 * 2;
__global__ void __launch_bounds__(kWThreads, 1)
fp8_quant_weight_kernel(uint8_t* __restrict__ codes, float* __restrict__ scales, const bf16* __restrict__ w, int N, int K, uint32_t steps, uint32_t steps_k, uint32_t steps_n) {
  pdl_wait();
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t part[2][2][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
  const int blocks_k = (K + 127) / 128, blocks_n = (N + 127) / 128;
  struct At { int64_t matrix; int n, k; };
  auto at_of = [&](uint32_t step) {                      // which matrix, its first row and column
    const uint32_t row = step / steps_k, e = row / steps_n;
    return At{(int64_t)e, (int)(row - e * steps_n) * 128, (int)(step - row * steps_k) * 256};
  };
  auto copy = [&](uint32_t step, int stage) {            // a warp takes rows warp, warp + 16, ..., a lane eight columns of each
    if (step < steps) {
      const At a = at_of(step);
      const int k = a.k + lane * 8;
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int n = a.n + warp + 16 * i;
        const bool there = n < N && k < K;
        const bf16* src = there ? w + (a.matrix * N + n) * K + k : w;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(base + stage * kWStage + (warp + 16 * i) * 512 + lane * 16), "l"(src), "r"(there ? 16 : 0) : "memory");
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kWStages; ++s) copy(blockIdx.x + s * gridDim.x, s);
  int stage = 0, turn = 0;
  for (uint32_t step = blockIdx.x; step < steps; step += gridDim.x) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kWStages - 1) : "memory");      // (a thread reads back what it has copied itself)
    uint4 v[8];
    uint32_t m2 = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      v[i] = *reinterpret_cast<const uint4*>(smem + stage * kWStage + (warp + 16 * i) * 512 + lane * 16);
      m2 = max2(m2, mag2(v[i]));
    }
    copy(step + kWStages * gridDim.x, stage);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m2 = max2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
    if ((lane & 15) == 0) part[turn][lane >> 4][warp] = m2;
    __syncthreads();
    m2 = part[turn][lane >> 4][lane & 15];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m2 = max2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
    float scale, factor;
    fp8::scale_of(mag(m2), scale, factor);
    const At a = at_of(step);
    const int k = a.k + lane * 8;
    if (k < K) {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int n = a.n + warp + 16 * i;
        if (n < N) *reinterpret_cast<uint2*>(codes + (a.matrix * N + n) * K + k) = factor > 0.f ? codes8(v[i], factor) : make_uint2(0, 0);
      }
      if (warp == 0 && (lane & 15) == 0) scales[(a.matrix * blocks_n + a.n / 128) * blocks_k + k / 128] = scale;
    }
    if (++stage == kWStages) stage = 0;
    turn ^= 1;
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
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
  const int64_t units = (int64_t)T * blocks;
  KGE_REQUIRE(units < (1ll << 31) - 64 * 148 * 32, "kge_fp8_quant: %d rows of %d in one call", T, K);
  const int64_t ctas = (units + 31) / 32, most = 148 * 6;
  KGE_CUDA_OK(launch_pdl(fp8_quant_kernel, dim3((unsigned)(ctas < most ? ctas : most)), dim3(256), 0, (cudaStream_t)stream, (uint8_t*)codes, scales, (int64_t)scales_stride,
                         (const bf16*)x, (int64_t)x_stride, rows, (uint32_t)units, K, (uint32_t)blocks));
  return 0;
}

extern "C" int KGE_API(kge_fp8_quant_weight)(void* codes, float* scales, const void* w, int E, int N, int K, void* stream) {
  KGE_REQUIRE(codes && scales && w, "kge_fp8_quant_weight: null pointer");
  KGE_REQUIRE(E > 0 && N > 0, "kge_fp8_quant_weight: %d matrices of %d rows", E, N);
  KGE_REQUIRE(K > 0 && K % 16 == 0, "kge_fp8_quant_weight: K=%d must be a positive multiple of 16", K);
  KGE_REQUIRE(aligned16(codes) && aligned16(w) && ((uintptr_t)scales & 3) == 0, "kge_fp8_quant_weight: codes and w must be 16-byte aligned");
  const int64_t steps_k = (K + 255) / 256, steps_n = fp8::blocks(N), steps = steps_k * steps_n * E;
  KGE_REQUIRE(steps < (1ll << 31) - 4 * 148, "kge_fp8_quant_weight: %d matrices of %d x %d in one call", E, N, K);
  const int smem = kWStages * kWStage;
  KGE_CUDA_OK(cudaFuncSetAttribute(fp8_quant_weight_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  KGE_CUDA_OK(launch_pdl(fp8_quant_weight_kernel, dim3((unsigned)(steps < 148 ? steps : 148)), dim3(kWThreads), (size_t)smem, (cudaStream_t)stream, (uint8_t*)codes, scales,
                         (const bf16*)w, N, K, (uint32_t)steps, (uint32_t)steps_k, (uint32_t)steps_n));
  pdl_break_next();        // a product that is launched early reads weights before it waits for the kernel before it
  return 0;
}
