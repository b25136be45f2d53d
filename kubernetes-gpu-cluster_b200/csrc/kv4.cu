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

// A thread has 16 bytes (8 dimensions) of a row, HD / 8 neighbouring lanes a row; rows of the launch: (token, head) with the q heads, the key
// heads and the value heads of a token in turn.  Rotation: the pair (i, i + HD / 2) lies HD / 16 lanes apart.  x cos and y sin are exact in
// fp32 (16-bit factors), so a turned number is rounded twice in all, to fp32 and to 16 bits, and fused or not gives the same bits.
// Bound by its bytes: the qkv rows in, q rows and HD + 8 bytes per token and kv head out.
template <int HD>
__global__ void __launch_bounds__(256)
rope_kv4write_kernel(bf16* q_out, int q_stride, uint8_t* cache, const bf16* qkv, const bf16* __restrict__ cos_sin, const int32_t* __restrict__ positions,
                     const int64_t* __restrict__ slots, uint32_t lanes, int H, int KV, int bs_shift) {
  constexpr int L = HD / 8;
  pdl_launch_dependents();
  pdl_wait();
  const uint32_t gid = blockIdx.x * 256u + threadIdx.x;
  if ((gid & ~31u) >= lanes) return;                       // (a warp's last lanes stay for its shuffles)
  const bool on = gid < lanes;
  const uint32_t per = (uint32_t)(H + 2 * KV) * L, t = (on ? gid : lanes - 1) / per, c = gid % L;
  const int head = (int)((on ? gid : lanes - 1) % per / L);
  const int64_t at = (int64_t)t * per * 8 + head * HD + (int)c * 8;
  uint4 v = *reinterpret_cast<const uint4*>(qkv + at);
  if (cos_sin) {                                           // (the same for all lanes)
    uint4 o;
    uint32_t *vu = &v.x, *ou = &o.x;
#pragma unroll
    for (int k = 0; k < 4; ++k) ou[k] = __shfl_xor_sync(0xffffffffu, vu[k], L / 2);
    if (head < H + KV) {
      const bf16* cs = cos_sin + (int64_t)positions[t] * HD + (c & (L / 2 - 1)) * 8;
      const uint4 cv = *reinterpret_cast<const uint4*>(cs), sv = *reinterpret_cast<const uint4*>(cs + HD / 2);
      const uint32_t *cu = &cv.x, *su = &sv.x;
      const float sign = c < L / 2 ? -1.f : 1.f;           // first half x cos - y sin, second half y cos + x sin
#pragma unroll
      for (int k = 0; k < 4; ++k)
        vu[k] = pack_bf2(fmaf(bf_lo(vu[k]), bf_lo(cu[k]), sign * (bf_lo(ou[k]) * bf_lo(su[k]))), fmaf(bf_hi(vu[k]), bf_hi(cu[k]), sign * (bf_hi(ou[k]) * bf_hi(su[k]))));
    }
  }
  if (head < H && on) *reinterpret_cast<uint4*>(q_out + (int64_t)t * q_stride + head * HD + c * 8) = v;
  if (__all_sync(0xffffffffu, head < H)) return;
  const uint32_t* u = &v.x;
  float x[8];
#pragma unroll
  for (int k = 0; k < 4; ++k) { x[2 * k] = bf_lo(u[k]); x[2 * k + 1] = bf_hi(u[k]); }
  float lo = x[0], hi = x[0];
  bool fine = true;
#pragma unroll
  for (int k = 0; k < 8; ++k) { lo = fminf(lo, x[k]); hi = fmaxf(hi, x[k]); fine = fine && fabsf(x[k]) <= 3.402823466e38f; }
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) {
    lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  }
  lo += 0.f;                                               // which zero a minimum gives is open: the positive one
  const uint32_t row_lanes = (L == 32 ? 0xffffffffu : (1u << L) - 1) << (threadIdx.x & 31 & ~(L - 1));
  fine = (__ballot_sync(0xffffffffu, fine) & row_lanes) == row_lanes && hi - lo <= 3.402823466e38f;
  const int64_t slot = on ? slots[t] : -1;
  if (head < H || slot < 0) return;
  uint32_t s16 = bits16(f2bf_up(__fdiv_rn(hi - lo, 15.f)));
  if (!(fabsf(bf2f(f2bf(fmaf(15.f, bf_lo(s16), lo)))) <= 3.402823466e38f)) --s16;      // low + 15 s would be an infinity
  const float s = bf_lo(s16);
  uint32_t word = 0;
  if (fine && s > 0.f)
#pragma unroll
    for (int k = 0; k < 8; ++k) word |= (uint32_t)min(__float2int_rn(__fdiv_rn(x[k] - lo, s)), 15) << (4 * (k / 2) + 16 * (k & 1));
  const int kh = head - H < KV ? head - H : head - H - KV, token = (int)(slot & 15);
  const bool key = head - H < KV;
  const int64_t blk = slot >> bs_shift;
  const int grp = (int)(slot & ((1 << bs_shift) - 1)) >> 4;
  uint8_t* g = cache + (((blk * KV + kh) << (bs_shift - 4)) + grp) * kv4::group_bytes(HD);
  const int place = key ? kv4::key_row(token) * L + (int)c : 16 * L + token * L + kv4::value_word(HD, token, (int)c);
  reinterpret_cast<uint32_t*>(g)[place] = word;
  if (c == 0) reinterpret_cast<uint32_t*>(g)[32 * L + (key ? 0 : 16) + token] = fine ? s16 | bits16(f2bf(lo)) << 16 : 0x7fff7fffu;
}

// A thread has 8 dimensions of the key and of the value of one (token, kv head); rows whose slot is negative are zeros.
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
  return num_blocks * KV * block_size * (hd + 8);
}
#endif

extern "C" int KGE_API(kge_rope_kv4write)(void* q_out, int q_out_stride, void* kv_cache, const void* qkv, const void* cos_sin, const int32_t* positions,
                                          const int64_t* slot_mapping, int T, int H, int KV, int hd, int block_size, void* stream) {
  KGE_REQUIRE(q_out && kv_cache && qkv && slot_mapping, "kge_rope_kv4write: null pointer");
  KGE_REQUIRE(!cos_sin || positions, "kge_rope_kv4write: cos_sin given without positions");
  KGE_REQUIRE(H > 0 && KV > 0, "kge_rope_kv4write: H=%d KV=%d", H, KV);
  KGE_REQUIRE(hd == 64 || hd == 128, "kge_rope_kv4write: head_dim=%d unsupported (64, 128)", hd);
  KGE_REQUIRE(block_size >= 16 && (block_size & (block_size - 1)) == 0, "kge_rope_kv4write: block_size=%d must be a power of two from 16", block_size);
  KGE_REQUIRE(q_out_stride >= H * hd && q_out_stride % 8 == 0, "kge_rope_kv4write: rows of q_out %d apart (a multiple of 8, at least H * hd = %d)", q_out_stride, H * hd);
  KGE_REQUIRE(aligned(q_out, 16) && aligned(kv_cache, 16) && aligned(qkv, 16) && aligned(cos_sin, 16), "kge_rope_kv4write: pointers must be 16-byte aligned");
  if (T <= 0) return 0;
  const int64_t lanes = (int64_t)T * (H + 2 * KV) * (hd / 8);
  KGE_REQUIRE(lanes < (1ll << 32) - 256, "kge_rope_kv4write: %d tokens of %d heads in one call", T, H + 2 * KV);
  int shift = 4;
  while ((1 << shift) < block_size) ++shift;
  auto kern = hd == 128 ? rope_kv4write_kernel<128> : rope_kv4write_kernel<64>;
  KGE_CUDA_OK(launch_pdl(kern, dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, (cudaStream_t)stream, (bf16*)q_out, q_out_stride, (uint8_t*)kv_cache, (const bf16*)qkv,
                         (const bf16*)cos_sin, positions, slot_mapping, (uint32_t)lanes, H, KV, shift));
  return 0;
}

extern "C" int KGE_API(kge_kv4_read)(void* k_out, void* v_out, const void* kv_cache, const int64_t* slot_mapping, int T, int KV, int hd, int block_size, void* stream) {
  KGE_REQUIRE(k_out && v_out && kv_cache && slot_mapping, "kge_kv4_read: null pointer");
  KGE_REQUIRE(KV > 0, "kge_kv4_read: KV=%d", KV);
  KGE_REQUIRE(hd == 64 || hd == 128, "kge_kv4_read: head_dim=%d unsupported (64, 128)", hd);
  KGE_REQUIRE(block_size >= 16 && (block_size & (block_size - 1)) == 0, "kge_kv4_read: block_size=%d must be a power of two from 16", block_size);
  KGE_REQUIRE(aligned(k_out, 16) && aligned(v_out, 16) && aligned(kv_cache, 16), "kge_kv4_read: pointers must be 16-byte aligned");
  if (T <= 0) return 0;
  const int64_t lanes = (int64_t)T * KV * (hd / 8);
  KGE_REQUIRE(lanes < (1ll << 32) - 256, "kge_kv4_read: %d tokens of %d heads in one call", T, KV);
  int shift = 4;
  while ((1 << shift) < block_size) ++shift;
  auto kern = hd == 128 ? kv4_read_kernel<128> : kv4_read_kernel<64>;
  KGE_CUDA_OK(launch_pdl(kern, dim3((unsigned)((lanes + 255) / 256)), dim3(256), 0, (cudaStream_t)stream, (bf16*)k_out, (bf16*)v_out, (const uint8_t*)kv_cache, slot_mapping,
                         (uint32_t)lanes, KV, shift));
  return 0;
}
