// Rows of the 4-bit key-value cache (layout: kv4.cuh): written behind rotary positions, and read back in 16 bits.
#include "common.cuh"
#include "kge.h"
#include "kv4.cuh"

namespace kge {
inline namespace KGE_ELT_NS {

#ifdef KGE_HALF
__device__ __forceinline__ bf16 f2bf_up(float v) { return __float2half_ru(v); }
__device__ __forceinline__ uint32_t bits16(bf16 v) { return __half_as_ushort(v); }
#else
__device__ __forceinline__ bf16 f2bf_up(float v) { return __float2bfloat16_ru(v); }
__device__ __forceinline__ uint32_t bits16(bf16 v) { return __bfloat16_as_ushort(v); }
#endif

// A thread has 8 dimensions of the first half of a row and the 8 that they turn with, HD / 16 neighbouring lanes a row; the rows of a token are its q
// heads, key heads and value heads.  x cos and y sin are exact in fp32 (16-bit factors), so a turned number is rounded twice in all, to fp32 and
// to 16 bits, and fused or not gives the same bits.
// Codes: c = rint(d (1 / s)), d = x - low, is the nearest code but where the quotient lies within rounding of a half; there the remainder d - c s,
// which one fma gives exactly, reaches s / 2 and says what is nearer, or that it is a tie.
// Its bytes are the qkv rows in, q rows and HD + 8 a token and kv head out, but instructions and the blocks' lives bound it: 8192 tokens of 32 / 8
// heads of 128 (179 MB, 27.7 us at the copy's rate) take 60 us with a division for every code, 57 without, 43 with both halves of a pair in one
// thread (no exchange of lanes, cosines read once for both); two or three tokens a thread 48 and 52, blocks of 64 or 384 threads 55 and 64.
// Few heads: a block of 128 threads takes several tokens (threadIdx.y); 8192 tokens of 8 / 1 heads of 64 10.3 -> 7.5 us, 4 / 2 of 128 11.8 -> 9.0.
template <int HD, bool TOKENS>
__global__ void __launch_bounds__(256)
rope_kv4write_kernel(bf16* q_out, int q_stride, uint8_t* cache, const bf16* qkv, const bf16* __restrict__ cos_sin, const int32_t* __restrict__ positions,
                     const int64_t* __restrict__ slots, int T, int H, int KV, int bs_shift) {
  constexpr int L = HD / 16;
  pdl_launch_dependents();
  pdl_wait();
  const int t = TOKENS ? blockIdx.x * blockDim.y + threadIdx.y : blockIdx.x;
  if (TOKENS && t >= T) return;                            // (the same for the warp)
  const int rows = H + 2 * KV, lane_at = blockIdx.y * blockDim.x + threadIdx.x;
  const int at = min(lane_at, rows * L - 1), head = at / L, c = threadIdx.x % L;      // (a last warp's surplus lanes go along with its last row)
  const bf16* src = qkv + ((int64_t)t * rows + head) * HD + c * 8;
  uint4 v[2] = {*reinterpret_cast<const uint4*>(src), *reinterpret_cast<const uint4*>(src + HD / 2)};
  const bool some_kv = !__all_sync(0xffffffffu, head < H);
  const int64_t slot = some_kv ? slots[t] : -1;
  uint32_t *xu = &v[0].x, *yu = &v[1].x;
  if (cos_sin && head < H + KV) {
    const bf16* cs = cos_sin + (int64_t)positions[t] * HD + c * 8;
    const uint4 cv = *reinterpret_cast<const uint4*>(cs), sv = *reinterpret_cast<const uint4*>(cs + HD / 2);
    const uint32_t *cu = &cv.x, *su = &sv.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x0 = bf_lo(xu[k]), x1 = bf_hi(xu[k]), y0 = bf_lo(yu[k]), y1 = bf_hi(yu[k]);
      const float c0 = bf_lo(cu[k]), c1 = bf_hi(cu[k]), s0 = bf_lo(su[k]), s1 = bf_hi(su[k]);
      xu[k] = pack_bf2(fmaf(x0, c0, -(y0 * s0)), fmaf(x1, c1, -(y1 * s1)));
      yu[k] = pack_bf2(fmaf(y0, c0, x0 * s0), fmaf(y1, c1, x1 * s1));
    }
  }
  if (head < H && lane_at < rows * L) {
    uint4* dst = reinterpret_cast<uint4*>(q_out + (int64_t)t * q_stride + head * HD + c * 8);
    dst[0] = v[0];
    dst[HD / 16] = v[1];
  }
  if (slot < 0) return;                                    // (the same for the warp)
  float x[16];
#pragma unroll
  for (int k = 0; k < 4; ++k) { x[2 * k] = bf_lo(xu[k]); x[2 * k + 1] = bf_hi(xu[k]); x[8 + 2 * k] = bf_lo(yu[k]); x[9 + 2 * k] = bf_hi(yu[k]); }
  float lo = x[0], hi = x[0], sum = x[0];
#pragma unroll
  for (int k = 1; k < 16; ++k) { lo = fminf(lo, x[k]); hi = fmaxf(hi, x[k]); sum += x[k]; }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  lo += 0.f;                                               // which zero a minimum gives is open: the positive one
  // A NaN makes the sum one; an infinity the range.  (A sum of finite numbers is NaN where it passed both infinities, and the range has then too.)
  const uint32_t row_lanes = ((1u << L) - 1) << (threadIdx.x & 31 & ~(L - 1));
  const bool fine = (__ballot_sync(0xffffffffu, sum == sum) & row_lanes) == row_lanes && hi - lo <= 3.402823466e38f;
  if (head < H || lane_at >= rows * L) return;
  uint32_t s16 = bits16(f2bf_up(__fdiv_rn(hi - lo, 15.f)));
  if (!(fabsf(bf2f(f2bf(fmaf(15.f, bf_lo(s16), lo)))) <= 3.402823466e38f)) --s16;      // low + 15 s would be an infinity
  const float s = bf_lo(s16), inv = __fdiv_rn(1.f, s), half = 0.5f * s;
  // n = 1.5 2^23 + rint(d / s) has the code in its last bits; what the constants of eight of them sum up to is taken off at the end
  constexpr uint32_t kAbove = 0x4b400000u;
  uint32_t word[2] = {0, 0};
  float far = 0.f;
#pragma unroll
  for (int k = 0; k < 16; ++k) {
    const float d = x[k] - lo, n = __fadd_rn(__fmul_rn(d, inv), 12582912.f);
    far = fmaxf(far, fabsf(fmaf(-__fsub_rn(n, 12582912.f), s, d)));
    word[k >> 3] += __float_as_uint(n) << (4 * ((k & 7) >> 1) + 16 * (k & 1));
  }
#pragma unroll
  for (int w = 0; w < 2; ++w) word[w] -= kAbove * 0x1111u + (kAbove << 16) * 0x1111u;
  if (!(far < half)) {                                     // a half, or a step beyond: to the nearest, to the even one of two
#pragma unroll
    for (int k = 0; k < 16; ++k) {
      const int bit = 4 * ((k & 7) >> 1) + 16 * (k & 1);
      const float d = x[k] - lo, n = __fsub_rn(__fadd_rn(__fmul_rn(d, inv), 12582912.f), 12582912.f), r = fmaf(-n, s, d);
      const bool odd = (word[k >> 3] >> bit) & 1u;
      if (r > half || (r == half && odd)) word[k >> 3] += 1u << bit;
      if (r < -half || (r == -half && odd)) word[k >> 3] -= 1u << bit;
    }
  }
  if (!fine || !(inv <= 3.402823466e38f)) {                // no number, no range, or an s so small that 1 / s is infinite
    word[0] = word[1] = 0;
    if (fine && s > 0.f)
#pragma unroll
      for (int k = 0; k < 16; ++k) word[k >> 3] |= (uint32_t)min(__float2int_rn(__fdiv_rn(x[k] - lo, s)), 15) << (4 * ((k & 7) >> 1) + 16 * (k & 1));
  }
  const bool key = head < H + KV;
  const int kh = head - H - (key ? 0 : KV), token = (int)(slot & 15);
  const int64_t blk = slot >> bs_shift;
  const int grp = (int)(slot & ((1 << bs_shift) - 1)) >> 4;
  uint32_t* g = reinterpret_cast<uint32_t*>(cache + (((blk * KV + kh) << (bs_shift - 4)) + grp) * kv4::group_bytes(HD));
  uint32_t* row = g + (key ? kv4::key_row(token) : 16 + token) * (2 * L);
  row[key ? c : kv4::value_word(HD, token, c)] = word[0];
  row[key ? c + L : kv4::value_word(HD, token, c + L)] = word[1];
  if (c == 0) g[64 * L + (key ? 0 : 16) + token] = fine ? s16 | bits16(f2bf(lo)) << 16 : 0x7fff7fffu;
}

// A thread has 8 dimensions of the key and of the value of one (token, kv head); rows whose slot is negative are zeros.  8192 tokens of 8 heads of 128:
// 10.7 us for 6.6 of bytes, most of them stores; with 16 dimensions a thread 9.8, but 64 tokens 1.9 in place of 1.6.
template <int HD>
__global__ void __launch_bounds__(256)
kv4_read_kernel(bf16* __restrict__ k_out, bf16* __restrict__ v_out, const uint8_t* __restrict__ cache, const int64_t* __restrict__ slots, uint32_t lanes, int KV,
                int bs_shift) {
  constexpr int L = HD / 8;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x;
  if (gid >= lanes) return;
  const uint32_t c = gid % L, row = gid / L, t = row / (uint32_t)KV, kh = row % (uint32_t)KV;
  const int64_t slot = slots[t];
  uint4 out[2] = {make_uint4(0, 0, 0, 0), make_uint4(0, 0, 0, 0)};
  if (slot >= 0) {
    const int token = (int)(slot & 15), grp = (int)(slot & ((1 << bs_shift) - 1)) >> 4;
    const uint32_t* g = reinterpret_cast<const uint32_t*>(cache + ((((slot >> bs_shift) * KV + kh) << (bs_shift - 4)) + grp) * kv4::group_bytes(HD));
    const uint32_t w[2] = {g[kv4::key_row(token) * L + c], g[16 * L + token * L + kv4::value_word(HD, token, (int)c)]};
    const uint32_t p[2] = {g[32 * L + token], g[32 * L + 16 + token]};
#pragma unroll
    for (int n = 0; n < 2; ++n) {
      const float s = bf_lo(p[n]), low = bf_hi(p[n]);
      uint32_t* o = &out[n].x;
#pragma unroll
      for (int k = 0; k < 4; ++k) o[k] = pack_bf2(fmaf(s, (float)((w[n] >> (4 * k)) & 15u), low), fmaf(s, (float)((w[n] >> (4 * k + 16)) & 15u), low));
    }
  }
  const int64_t at = (int64_t)gid * 8;
  *reinterpret_cast<uint4*>(k_out + at) = out[0];
  *reinterpret_cast<uint4*>(v_out + at) = out[1];
}

static bool aligned(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

}  // namespace KGE_ELT_NS
}  // namespace kge

using namespace kge;

#ifndef KGE_HALF
extern "C" int64_t kge_kv4_cache_bytes(int64_t num_blocks, int KV, int hd, int block_size) {
  if (num_blocks < 0 || KV <= 0 || (hd != 64 && hd != 128) || block_size < 16 || (block_size & (block_size - 1))) {
    kge::set_error("kge_kv4_cache_bytes: %lld blocks of %d tokens, %d kv heads of %d (heads of 64 or 128, a power of two of tokens from 16)", (long long)num_blocks, block_size,
                   KV, hd);
    return -1;
  }
  const int64_t block = (int64_t)block_size * (hd + 8);
  int64_t bytes;
  if (__builtin_mul_overflow((int64_t)KV, block, &bytes) || __builtin_mul_overflow(num_blocks, bytes, &bytes)) {
    kge::set_error("kge_kv4_cache_bytes: %lld blocks of %d tokens and %d kv heads are more bytes than 64 bits count", (long long)num_blocks, block_size, KV);
    return -1;
  }
  return bytes;
}
#endif

extern "C" int KGE_API(kge_rope_kv4write)(void* q_out, int q_out_stride, void* kv_cache, const void* qkv, const void* cos_sin, const int32_t* positions,
                                          const int64_t* slot_mapping, int T, int H, int KV, int hd, int block_size, void* stream) {
  KGE_REQUIRE(q_out && kv_cache && qkv && slot_mapping, "kge_rope_kv4write: null pointer");
  KGE_REQUIRE(!cos_sin || positions, "kge_rope_kv4write: cos_sin given without positions");
  KGE_REQUIRE(H > 0 && KV > 0, "kge_rope_kv4write: H=%d KV=%d", H, KV);
  KGE_REQUIRE(hd == 64 || hd == 128, "kge_rope_kv4write: head_dim=%d unsupported (64, 128)", hd);
  KGE_REQUIRE(block_size >= 16 && (block_size & (block_size - 1)) == 0, "kge_rope_kv4write: block_size=%d must be a power of two from 16", block_size);
  KGE_REQUIRE(((int64_t)H + 2ll * KV) * hd < (1ll << 24), "kge_rope_kv4write: %lld heads of %d", (long long)H + 2ll * KV, hd);
  KGE_REQUIRE(q_out_stride >= H * hd && q_out_stride % 8 == 0, "kge_rope_kv4write: rows of q_out %d apart (a multiple of 8, at least H * hd = %d)", q_out_stride, H * hd);
  KGE_REQUIRE(aligned(q_out, 16) && aligned(kv_cache, 16) && aligned(qkv, 16) && aligned(cos_sin, 16), "kge_rope_kv4write: pointers must be 16-byte aligned");
  if (T <= 0) return 0;
  int shift = 4;
  while ((1 << shift) < block_size) ++shift;
  const int lanes = (H + 2 * KV) * (hd / 16), th = lanes <= 256 ? (lanes + 31) & ~31 : 128, tokens = th <= 64 ? 128 / th : 1;      // (of a block)
  auto kern = hd == 128 ? (tokens > 1 ? rope_kv4write_kernel<128, true> : rope_kv4write_kernel<128, false>)
                        : (tokens > 1 ? rope_kv4write_kernel<64, true> : rope_kv4write_kernel<64, false>);
  KGE_CUDA_OK(launch_pdl(kern, dim3((T + tokens - 1) / tokens, (lanes + th - 1) / th), dim3(th, tokens), 0, (cudaStream_t)stream, (bf16*)q_out,
                         q_out_stride, (uint8_t*)kv_cache, (const bf16*)qkv, (const bf16*)cos_sin, positions, slot_mapping, T, H, KV, shift));
  return 0;
}

extern "C" int KGE_API(kge_kv4_read)(void* k_out, void* v_out, const void* kv_cache, const int64_t* slot_mapping, int T, int KV, int hd, int block_size, void* stream) {
  KGE_REQUIRE(k_out && v_out && kv_cache && slot_mapping, "kge_kv4_read: null pointer");
  KGE_REQUIRE(KV > 0, "kge_kv4_read: KV=%d", KV);
  KGE_REQUIRE(hd == 64 || hd == 128, "kge_kv4_read: head_dim=%d unsupported (64, 128)", hd);
  KGE_REQUIRE(block_size >= 16 && (block_size & (block_size - 1)) == 0, "kge_kv4_read: block_size=%d must be a power of two from 16", block_size);
  KGE_REQUIRE(aligned(k_out, 16) && aligned(v_out, 16) && aligned(kv_cache, 16), "kge_kv4_read: pointers must be 16-byte aligned");
  if (T <= 0) return 0;
  const int64_t lanes = (int64_t)T * (hd / 8) * (KV < (1 << 24) ? KV : 1 << 24);
  KGE_REQUIRE(KV < (1 << 24) && lanes < (1ll << 32) - 256, "kge_kv4_read: %d tokens of %d heads in one call", T, KV);
  int shift = 4;
  while ((1 << shift) < block_size) ++shift;
  auto kern = hd == 128 ? kv4_read_kernel<128> : kv4_read_kernel<64>;
  KGE_CUDA_OK(launch_pdl(kern, dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, (cudaStream_t)stream, (bf16*)k_out, (bf16*)v_out, (const uint8_t*)kv_cache, slot_mapping,
                         (uint32_t)lanes, KV, shift));
  return 0;
}
