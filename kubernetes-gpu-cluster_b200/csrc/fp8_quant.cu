// Rows and matrices of 16 bits as 8-bit floating point with a scale for each block (fp8.cuh has the definition).
//
// Both are bound by their bytes, 2 in and 1 out for a number.  16-bit numbers x, m have at most 11 bits, so 448 x and t m (t half way between two
// codes, 5 bits) are integers of at most 17 bits on one grid: 448 x / m either is t or misses it by 2^-17 and more.  x times the factor is off by less
// than 2^-21, hence rounding it to 20 bits gives t where the quotient is t, and leaves it on its side of t elsewhere: one product and two integer
// operations in place of a division.
#include "f32x2.cuh"
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

__device__ __forceinline__ float to_20_bits(float x) { return __uint_as_float((__float_as_uint(x) + 8u) & ~15u); }
__device__ __forceinline__ uint2 codes8(uint4 v, float factor) {
  const uint32_t u[4] = {v.x, v.y, v.z, v.w};
  uint32_t c[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    float a, b;
    upk(mul2(pk(bf_lo(u[k]), bf_hi(u[k])), pk(factor, factor)), a, b);
    c[k] = fp8::pack2(to_20_bits(a), to_20_bits(b));
  }
  return make_uint2(c[0] | c[1] << 16, c[2] | c[3] << 16);
}

// (zeros where the factor is zero: a block with an infinity or NaN)
__device__ __forceinline__ uint4 codes16(const uint4 (&v)[2], float factor) {
  if (!(factor > 0.f)) return make_uint4(0, 0, 0, 0);
  const uint2 lo = codes8(v[0], factor), hi = codes8(v[1], factor);
  return make_uint4(lo.x, lo.y, hi.x, hi.y);
}

// Few rows: eight lanes have a block of a row, 16 numbers each.
__global__ void __launch_bounds__(256)
fp8_quant_few_kernel(uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t scales_stride, const bf16* __restrict__ x, int64_t x_stride, const int32_t* __restrict__ rows,
                     uint32_t units, int K, uint32_t blocks) {
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t at = blockIdx.x * 32 + (threadIdx.x >> 3), t = at / blocks, b = at - t * blocks;
  const int k = b * fp8::kBlock + (threadIdx.x & 7) * 16;
  const bool there = at < units && k < K;
  uint4 v[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (there) {
    const int r = rows ? rows[t] : (int)t;
    if (r >= 0) {
      const bf16* src = x + r * x_stride + k;
      v[0] = ld_nc_v4(src);
      v[1] = ld_nc_v4(src + 8);
    }
  }
  uint32_t m2 = max2(mag2(v[0]), mag2(v[1]));
#pragma unroll
  for (int o = 4; o > 0; o >>= 1) m2 = max2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
  if (!there) return;
  float scale, factor;
  fp8::scale_of(mag(m2), scale, factor);
  *reinterpret_cast<uint4*>(codes + (int64_t)t * K + k) = codes16(v, factor);
  if ((threadIdx.x & 7) == 0) scales[b * scales_stride + t] = scale;
}

// Many rows: a warp takes 512 W columns of a row at a time, 16 W numbers a lane, one piece after the other of an equal share of all, copied ahead into a ring
// of its own in shared memory.  A copy is 512 bytes one behind the other; a lane reads back the 32 W that it turns into codes, from places exchanged so that
// eight lanes meet in no bank.  (Where a lane copied its own 32 bytes every sector was fetched twice: 18.3 us for 16 of 16384 rows of 2048.)
// Bound by instructions where rows lie in the L2, 12 a number with W = 1 and 9.5 with W = 2, else by memory.  us with W = 1 and 2: 16384 rows of 2048 gathered
// from 2048 (43 MB, 6.6 us at the copy's rate) 15.9 and 13.8, 8192 of 4096 (101 MB, 15.5 us) 21.0 and 20.2, 20000 of 7168 (434 MB) 86.4 and 80.6 (5.4 TB/s), of
// 2560 32.1 and 31.4, of 640 10.7 and 9.9; but where the last piece is half empty, 20000 of 512 7.6 and 9.3, 6000 of 1408 6.9 and 7.3: W = 2 with at most 5/8
// as many pieces.  With 16, 24 and 28 warps and as many more pieces ahead within 4 % of it.
constexpr int kRowWarps = 32, kRing = 6 * 1024;            // warps; bytes of a warp's ring
template <int W>
__global__ void __launch_bounds__(kRowWarps * 32, 1)
fp8_quant_kernel(uint8_t* __restrict__ codes, float* __restrict__ scales, int64_t scales_stride, const bf16* __restrict__ x, int64_t x_stride, const int32_t* __restrict__ rows,
                 uint32_t pieces, int K, uint32_t per_row) {
  constexpr int kColumns = 512 * W, kPiece = 2 * kColumns, kAhead = kRing / kPiece, kMine = 16 * W;      // of a piece: columns, bytes; pieces ahead; columns of a lane
  extern __shared__ __align__(16) uint8_t smem[];
  pdl_launch_dependents();
  pdl_wait();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t warps = gridDim.x * kRowWarps, me = blockIdx.x * kRowWarps + warp, each = pieces / warps, more = pieces - each * warps;
  const uint32_t first = each * me + min(me, more);
  int n = (int)(each + (me < more));
  if (n == 0) return;
  const uint32_t t0 = first / per_row, last = (first + n - 1) / per_row;
  const int k0 = (int)(first - t0 * per_row) * kColumns;
  // a piece's 16 bytes number c lie at c ^ (c / 8 % 2W)
  const uint8_t* ring = smem + warp * kRing;
  const int turned = W == 1 ? (lane >> 2) & 1 : (lane >> 1) & 3;
  const uint8_t* mine[2 * W];
#pragma unroll
  for (int j = 0; j < 2 * W; ++j) mine[j] = ring + (2 * W * lane + (j ^ turned)) * 16;
  const uint32_t to = (uint32_t)__cvta_generic_to_shared(ring) + ((lane ^ ((lane >> 3) & (2 * W - 1))) << 4), to_end = to + kAhead * kPiece;
  auto row_of = [&](uint32_t t) { return rows && t <= last ? rows[t] : (int)t; };
  // the copies' way through the share: row, column, source; and the row after that, asked for a row ahead
  uint32_t t = t0, slot_in = to;
  int k = k0 + lane * 8, r = row_of(t0), r_next = row_of(t0 + 1), left = n;
  const bf16* src = x + r * x_stride + k;
  auto copy = [&] {
    if (left > 0) {
      --left;
#pragma unroll
      for (int i = 0; i < 2 * W; ++i) {
        const bool there = r >= 0 && k + i * 256 < K;
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(slot_in + i * 512), "l"(there ? src + i * 256 : x), "r"(there ? 16u : 0u) : "memory");
      }
      k += kColumns;
      src += kColumns;
      if (k - lane * 8 >= K) {
        ++t;
        k = lane * 8;
        r = r_next;
        r_next = row_of(t + 1);
        src = x + r * x_stride + k;
      }
      if ((slot_in += kPiece) == to_end) slot_in = to;
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll 1
  for (int i = 0; i < kAhead; ++i) copy();
  int at = k0 + lane * kMine, slot = 0;
  const int64_t blocks_on = 4 * W * scales_stride, row_on = 1 - (int64_t)(per_row - 1) * blocks_on;      // from one piece's scales to the next's, to the next row's first
  uint8_t* dst = codes + (int64_t)t0 * K + at;
  float* sc = scales + (int64_t)(at / 128) * scales_stride + t0;
#pragma unroll 1
  for (; n > 0; --n) {
    asm volatile("cp.async.wait_group %0;" ::"n"(kAhead - 1) : "memory");
    __syncwarp();                                    // (a lane reads what others have copied)
    uint4 v[W][2];
#pragma unroll
    for (int j = 0; j < 2 * W; ++j) v[j / 2][j % 2] = *reinterpret_cast<const uint4*>(mine[j] + slot);
    __syncwarp();
    copy();
    if ((slot += kPiece) == kAhead * kPiece) slot = 0;
    uint32_t m2 = max2(mag2(v[0][0]), mag2(v[0][1]));
    if (W == 2) m2 = max2(m2, max2(mag2(v[W - 1][0]), mag2(v[W - 1][1])));
#pragma unroll
    for (int o = 4 / W; o > 0; o >>= 1) m2 = max2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
    float scale, factor;
    fp8::scale_of(mag(m2), scale, factor);
    if (at < K) {
      if constexpr (W == 1) {
        *reinterpret_cast<uint4*>(dst) = codes16(v[0], factor);
      } else {
        const uint4 a = codes16(v[0], factor), b = codes16(v[1], factor);
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x), "r"(b.y), "r"(b.z), "r"(b.w) : "memory");
      }
      if (lane % (8 / W) == 0) *sc = scale;
    }
    at += kColumns;
    dst += kColumns;
    if (at - lane * kMine < K) {
      sc += blocks_on;
    } else {
      dst += K - (at - lane * kMine);
      at = lane * kMine;
      sc += row_on;
    }
  }
  asm volatile("cp.async.wait_all;" ::: "memory");
}

// A CTA takes steps of 128 rows x 256 columns (two blocks), copied three steps ahead into shared memory: every access to memory is a whole 512-byte piece
// of a row, or 256 bytes of codes, and loads are under way all the time.  28672 x 4096 (352 MB) 65.5 us, 5.4 TB/s (a block a
// CTA, from registers, 98); 1024 threads 70.9.
constexpr int kWThreads = 512, kWStages = 3, kWStage = 128 * 256 * 2;
__global__ void __launch_bounds__(kWThreads, 1)
fp8_quant_weight_kernel(uint8_t* __restrict__ codes, float* __restrict__ scales, const bf16* __restrict__ w, int N, int K, uint32_t steps, uint32_t steps_k, uint32_t steps_n) {
  pdl_wait();
  extern __shared__ __align__(16) uint8_t smem[];
  __shared__ uint32_t part[2][2][16];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t base = (uint32_t)__cvta_generic_to_shared(smem);
  const int blocks_k = (K - 1) / 128 + 1, blocks_n = (N - 1) / 128 + 1;
  // a step's matrix, block row and pair of block columns; the CTA's next step is gridDim.x further
  const uint32_t dk = gridDim.x % steps_k, dr = gridDim.x / steps_k, dn = dr % steps_n, de = dr / steps_n;
  struct At { uint32_t e, n, k; };
  auto next = [&](At& a) {
    a.k += dk; a.n += dn; a.e += de;
    if (a.k >= steps_k) { a.k -= steps_k; ++a.n; }
    if (a.n >= steps_n) { a.n -= steps_n; ++a.e; }
  };
  const uint32_t row0 = blockIdx.x / steps_k;
  At in = {row0 / steps_n, row0 % steps_n, blockIdx.x % steps_k}, at = in;
  const int64_t rows16 = (int64_t)16 * K;
  uint32_t asked = blockIdx.x;
  auto copy = [&](int stage) {                           // a warp takes rows warp, warp + 16, ..., a lane eight columns of each
    if (asked < steps) {
      const int n = in.n * 128 + warp, k = in.k * 256 + lane * 8;
      const bf16* src = w + ((int64_t)in.e * N + n) * K + k;
      const uint32_t dst = base + stage * kWStage + warp * 512 + lane * 16;
      const int there = k < K ? N - n : 0;               // rows 16 i below that are
#pragma unroll
      for (int i = 0; i < 8; ++i, src += rows16)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst + i * 8192), "l"(16 * i < there ? src : w), "r"(16 * i < there ? 16 : 0) : "memory");
      asked += gridDim.x;
      next(in);
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kWStages; ++s) copy(s);
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
    copy(stage);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m2 = max2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
    if ((lane & 15) == 0) part[turn][lane >> 4][warp] = m2;
    __syncthreads();
    m2 = part[turn][lane >> 4][lane & 15];
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) m2 = max2(m2, __shfl_xor_sync(0xffffffffu, m2, o));
    float scale, factor;
    fp8::scale_of(mag(m2), scale, factor);
    const int n = at.n * 128 + warp, k = at.k * 256 + lane * 8, there = k < K ? N - n : 0;
    uint8_t* dst = codes + ((int64_t)at.e * N + n) * K + k;
#pragma unroll
    for (int i = 0; i < 8; ++i, dst += rows16)
      if (16 * i < there) *reinterpret_cast<uint2*>(dst) = factor > 0.f ? codes8(v[i], factor) : make_uint2(0, 0);
    if (warp == 0 && (lane & 15) == 0 && k < K) scales[((int64_t)at.e * blocks_n + at.n) * blocks_k + k / 128] = scale;
    next(at);
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
  KGE_REQUIRE(aligned16(codes) && aligned16(x) && ((uintptr_t)scales & 3) == 0 && ((uintptr_t)rows & 3) == 0,
              "kge_fp8_quant: codes and x must be 16-byte aligned, scales and rows to their types");
  if (T <= 0) return 0;
  const int blocks = (int)fp8::blocks(K);
  const int64_t units = (int64_t)T * blocks;
  KGE_REQUIRE(units < (1ll << 31) - 64 * 148 * 32 && K < 0x7fffffff - 1024, "kge_fp8_quant: %d rows of %d in one call", T, K);      // (columns are counted beyond K)
  const int64_t per_row = (K + 511) / 512;
  if (T * per_row < 2 * 148 * kRowWarps) {
    KGE_CUDA_OK(launch_pdl(fp8_quant_few_kernel, dim3((unsigned)((units + 31) / 32)), dim3(256), 0, (cudaStream_t)stream, (uint8_t*)codes, scales, (int64_t)scales_stride,
                           (const bf16*)x, (int64_t)x_stride, rows, (uint32_t)units, K, (uint32_t)blocks));
    return 0;
  }
  const bool wide = K % 32 == 0 && ((uintptr_t)codes & 31) == 0 && 8 * ((per_row + 1) / 2) <= 5 * per_row;
  const int64_t per = wide ? (per_row + 1) / 2 : per_row;
  auto kern = wide ? fp8_quant_kernel<2> : fp8_quant_kernel<1>;
  const int smem = kRowWarps * kRing;
  KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  KGE_CUDA_OK(launch_pdl(kern, dim3(148), dim3(kRowWarps * 32), (size_t)smem, (cudaStream_t)stream, (uint8_t*)codes, scales, (int64_t)scales_stride, (const bf16*)x, (int64_t)x_stride,
                         rows, (uint32_t)(T * per), K, (uint32_t)per));
  return 0;
}

extern "C" int KGE_API(kge_fp8_quant_weight)(void* codes, float* scales, const void* w, int E, int N, int K, void* stream) {
  KGE_REQUIRE(codes && scales && w, "kge_fp8_quant_weight: null pointer");
  KGE_REQUIRE(E > 0 && N > 0, "kge_fp8_quant_weight: %d matrices of %d rows", E, N);
  KGE_REQUIRE(K > 0 && K % 16 == 0, "kge_fp8_quant_weight: K=%d must be a positive multiple of 16", K);
  KGE_REQUIRE(aligned16(codes) && aligned16(w) && ((uintptr_t)scales & 3) == 0, "kge_fp8_quant_weight: codes and w must be 16-byte aligned");
  const int64_t most = (1ll << 31) - 4 * 148, steps_k = ((int64_t)K + 255) / 256, steps_n = fp8::blocks(N), steps = steps_k * steps_n < most ? steps_k * steps_n * E : most;
  KGE_REQUIRE(steps < most, "kge_fp8_quant_weight: %d matrices of %d x %d in one call", E, N, K);
  const int smem = kWStages * kWStage;
  KGE_CUDA_OK(cudaFuncSetAttribute(fp8_quant_weight_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  KGE_CUDA_OK(launch_pdl(fp8_quant_weight_kernel, dim3((unsigned)(steps < 148 ? steps : 148)), dim3(kWThreads), (size_t)smem, (cudaStream_t)stream, (uint8_t*)codes, scales,
                         (const bf16*)w, N, K, (uint32_t)steps, (uint32_t)steps_k, (uint32_t)steps_n));
  pdl_weights_written((cudaStream_t)stream);        // a product that is launched early reads weights before it waits for the kernel before it
  return 0;
}
