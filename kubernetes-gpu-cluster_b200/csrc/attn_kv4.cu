// Attention over the 4-bit key-value cache (layout: kv4.cuh), single-token requests; prompts: attn_kv4_tc.cuh.
//
// With key k = low_k + s_k n_k and value v = low_v + s_v n_v (n: codes 0..15), z = low + 8 s,
//   score = scale (s_k (q . n_k) + low_k sum(q))           out = (sum_j (p_j s_v,j) (n_v,j - 8) + sum_j p_j z_v,j) / sum_j p_j
// so the products run on codes, which 16 bits hold exactly, and the two numbers of a row are applied to scores and weights in fp32.
//
// Four warps take 32 keys each of tiles of 128, which a fifth brings by bulk copies (one per block of a tile), and multiply with mma.m16n8k16
// whose M side is the keys (scores) or the dimensions (outputs) and whose N side is the query heads of one kv head: 8 columns of which a group
// of 4 or 8 heads leaves few empty, half the products that heads as the M side cost.  Both operands are float16 in either build.
//   Codes: the bits n in the low half-byte of a float16 are the number n 2^-24 (its denormals), in the next one n 2^-20, so a code costs half an
//   AND and no arithmetic; powers of two are put right in q (scores) and in the outputs.  (As 1024 + n less 1032: 2.6 instructions a pair.)
//   q: a power of two moves the largest number of the group's heads to 2^14; exact but for what lies 2^-24 below that.
//   Weights: w = e s_v with e = 2^(x - R), rounded to float16; R is a reference per head, such that the largest w of a warp lies between 1 and
//   2^14.  It moves only when a weight would pass that, so most tiles rescale nothing and need no shuffles.  What is taken off for centring, 8
//   times the sum of the weights, is the sum of the ROUNDED ones (a product with ones), so a rounding's error meets |n - 8| and not n.
//   scores come out as (key, head) fragments; movmatrix turns a packed 8 x 8 of weights into the B operand of the second product
#include <algorithm>

#include "common.cuh"
#include "kge.h"
#include "kv4.cuh"

namespace kge {
inline namespace KGE_ELT_NS {

namespace ak4 {

constexpr int NW = 4, TK = 128, WK = TK / NW, GROUPS = TK / 16;      // computing warps, keys of a tile, of a warp; groups of a tile
constexpr int kThreads = NW * 32 + 32;
__host__ __device__ constexpr int stages(int nt) { return nt == 1 ? 3 : 4; }      // tiles on their way; CTAs of an SM
__host__ __device__ constexpr int ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }
constexpr int kMaxCtas = 148 * 3;
constexpr float kLog2e = 1.4426950408889634f, kNoRef = -1e30f;
constexpr float kExpRoom = 40.f;
constexpr uint32_t kWeightMost = 0x7400;       // 2^14 in float16

struct Args {
  bf16* out;
  const bf16* q;
  const uint8_t* cache;
  const int32_t *table, *lens, *qsl;
  float* part;                                 // partial outputs of the pieces: [2 per CTA][G][HD], then [2 per CTA][G] (R, l)
  int4* desc;                                  // per CTA: the group that starts in its share and ends in a later one's (merge kernel)
  int q_stride, max_blocks, B, H, KV, bs_shift, window, first;
  float scale_log2;
  __device__ __forceinline__ int len(int b) const { return min(max(lens[b], 0), max_blocks << bs_shift); }      // (no page beyond the table is read)
};

__device__ __forceinline__ uint32_t s_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void mma_f16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float lg2(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// nibbles 0 and 4, or 1 and 5, of w as two float16 numbers: n 2^-24 and n 2^-20
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) { return w & 0x00f000f0u; }
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The keys that a single-token request of `len` keys sees, in tiles of TK: the first ones that stay visible, then the window.
struct Span {
  int len, lo, npre, win0, n;
  __device__ __forceinline__ Span(int kv_len, int window, int first) {
    len = kv_len;
    lo = window > 0 ? max(kv_len - window, 0) : 0;
    win0 = lo / TK;
    npre = min((min(first, lo) + TK - 1) / TK, win0);
    n = kv_len > 0 ? npre + (kv_len + TK - 1) / TK - win0 : 1;        // (one empty tile writes the zeros of a request without keys)
  }
  __device__ __forceinline__ int key0(int tile) const { return (tile < npre ? tile : win0 + tile - npre) * TK; }
};
__device__ __forceinline__ void bar_compute() { asm volatile("bar.sync 1, 128;" ::: "memory"); }      // the computing warps

// A share of the launch's tiles, piece by piece: request-major, then kv head, then tile.
struct Walk {
  uint32_t u, u1;
  int b, kvh, t0, t1, n;                       // the current piece: tiles t0 .. t1 of a group of n
  __device__ __forceinline__ bool next(const uint32_t* pre, uint32_t KV) {
    if (u >= u1) return false;
    while (pre[b + 1] * KV <= u) ++b;
    const uint32_t groups = pre[b + 1] - pre[b], rel = u - pre[b] * KV;
    n = (int)groups;
    kvh = (int)(rel / groups);
    t0 = (int)(rel - kvh * groups);
    t1 = (int)min(groups, t0 + (u1 - u));
    u += t1 - t0;
    return true;
  }
};

template <int HD> __host__ __device__ constexpr int red_floats() { return NW * 4 * (HD + 4); }
template <int HD, int NT> __host__ __device__ constexpr int ring_bytes() { return stages(NT) * GROUPS * kv4::group_bytes(HD); }

// SPLIT: the tiles of all (request, kv head) groups are one sequence, every CTA takes an equal share of it, and a group that is cut is merged
// by the kernel behind.  Otherwise a CTA has a whole group.
template <int HD, int NT, bool SPLIT>
__global__ void __launch_bounds__(kThreads, ctas_per_sm(NT)) attn_kv4_kernel(const Args a, int min_chunk) {
  constexpr int GB = kv4::group_bytes(HD), W = HD / 32, NM = HD / 16, RS = HD + 4, ST = stages(NT);      // W: words of a thread's share of a key row
  extern __shared__ __align__(128) uint8_t smem[];
  float* red = reinterpret_cast<float*>(smem + ring_bytes<HD, NT>());
  uint64_t* bars = reinterpret_cast<uint64_t*>(red + red_floats<HD>());
  uint32_t* pre = reinterpret_cast<uint32_t*>(bars + 2 * ST);
  const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31, g = lane >> 2, t = lane & 3;
  const int G = a.H / a.KV;
  const uint32_t bar0 = s_addr(bars);
  // full(s): the producer's arrival and its copies' bytes; empty(s): the computing warps.  A wait for either comes before what the next
  // phase of it needs: a warp arrives on empty(s) only behind its wait for full(s), and the producer refills s only behind empty(s).
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (ST + s); };
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) {
      asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(full(s)));
      asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(empty(s)), "n"(NW));
    }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  pdl_launch_dependents();
  pdl_wait();

  Walk cons;
  uint32_t u0 = 0;
  if (SPLIT) {
    for (int b = tid; b < a.B; b += kThreads) pre[b + 1] = a.qsl[b + 1] - a.qsl[b] == 1 ? Span(a.len(b), a.window, a.first).n : 0;
    if (tid == 0) pre[0] = 0;
    __syncthreads();
    if (warp == 0) {
      const int per = (a.B + 31) / 32, lo = 1 + lane * per, hi = min(a.B + 1, lo + per);
      uint32_t sum = 0;
      for (int i = lo; i < hi; ++i) sum += pre[i];
      uint32_t incl = sum;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) { const uint32_t v = __shfl_up_sync(0xffffffffu, incl, d); if (lane >= d) incl += v; }
      uint32_t run = incl - sum;
      for (int i = lo; i < hi; ++i) { run += pre[i]; pre[i] = run; }
    }
    __syncthreads();
    const uint32_t KV = a.KV, U = pre[a.B] * KV, chunk = max((U + gridDim.x - 1) / gridDim.x, (uint32_t)min_chunk);
    auto request_of = [&](uint32_t unit) {
      int lo = 0, hi = a.B - 1;
      while (lo < hi) { const int mid = (lo + hi) >> 1; if (pre[mid + 1] * KV <= unit) lo = mid + 1; else hi = mid; }
      return lo;
    };
    u0 = min(U, blockIdx.x * chunk);
    cons.u = u0; cons.u1 = min(U, u0 + chunk); cons.b = u0 < cons.u1 ? request_of(u0) : 0;
    if (tid == 0) {
      // the group that begins in this share and ends beyond it
      int4 d = make_int4(-1, 0, 0, 0);
      if (u0 < cons.u1 && cons.u1 < U) {
        const int b = request_of(cons.u1 - 1);
        const uint32_t n = pre[b + 1] - pre[b], base = pre[b] * KV, kvh = (cons.u1 - 1 - base) / n, g0 = base + kvh * n, g1 = g0 + n;
        if (g0 >= u0 && g1 > cons.u1) d = make_int4(a.qsl[b], (int)kvh, (int)((g1 - 1) / chunk), g0 > u0);
      }
      a.desc[blockIdx.x] = d;
    }
  } else {
    cons.b = blockIdx.y;
    if (a.qsl[cons.b + 1] - a.qsl[cons.b] != 1) return;
    __syncthreads();                           // the barriers are there
  }
  auto piece = [&](bool again) {
    if (SPLIT) return cons.next(pre, a.KV);
    cons.kvh = blockIdx.x; cons.t0 = 0;
    cons.t1 = cons.n = Span(a.len(cons.b), a.window, a.first).n;
    return !again;
  };
  int stage = 0;
  uint32_t parity = 0;
  auto advance = [&]() { if (++stage == ST) { stage = 0; parity ^= 1; } };

  if (warp == NW) {
    // ---- the producer: a lane per block of a tile; the ids of the next tile are read while this one's stage is waited for
    const int bs = 1 << a.bs_shift, box = min(bs, TK);
    const uint32_t ring = s_addr(smem);
    bool refill = false;
    for (bool more = piece(false); more; more = piece(true)) {
      const Span sp(a.len(cons.b), a.window, a.first);
      const int32_t* btab = a.table + (int64_t)cons.b * a.max_blocks;
      // of this lane's block: the keys from `lo` to `hi` that somebody may see (all in one copy), and the block's id
      int lo = 0, hi = 0, blk = 0;
      auto look = [&](int tile) {
        const int k0 = sp.key0(tile) + lane * box;
        lo = a.first > k0 ? k0 : max(k0, sp.lo & ~15);
        hi = min(k0 + box, sp.len);
        if (sp.lo >= hi) hi = min(hi, a.first);
        if (tile >= cons.t1 || lane * box >= TK) hi = lo;
        if (lo < hi) blk = btab[lo >> a.bs_shift];
      };
      look(cons.t0);
      for (int tile = cons.t0; tile < cons.t1; ++tile) {
        const int first = lo & ~15, groups = lo < hi ? (hi - first + 15) >> 4 : 0, id = blk;
        const uint32_t bytes = __reduce_add_sync(0xffffffffu, (uint32_t)groups) * GB, place = (uint32_t)(first - sp.key0(tile)) >> 4;
        look(tile + 1);
        if (refill) mbar_wait(empty(stage), parity ^ 1);
        if (lane == 0) asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full(stage)), "r"(bytes) : "memory");
        __syncwarp();
        if (groups > 0)
          bulk_load(ring + (stage * GROUPS + place) * GB, a.cache + ((((int64_t)id * a.KV + cons.kvh) << (a.bs_shift - 4)) + ((first & (bs - 1)) >> 4)) * GB, groups * GB, full(stage));
        advance();
        if (stage == 0) refill = true;
      }
    }
    return;
  }

  for (bool more = piece(false); more; more = piece(true)) {
    const Span sp(a.len(cons.b), a.window, a.first);
    const int qrow = a.qsl[cons.b];
    // ---- the group's query heads: column n of block nt is head 8 nt + n
    uint32_t qb[NT][NM][2];
    float qs[NT][2], fs;                       // scale log2(e) sum(q) of this thread's two columns; what scores are multiplied with
    {
      uint4 raw[NT][W];
      float mx = 0.f;
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        const int head = nt * 8 + g;
        const uint4* src = reinterpret_cast<const uint4*>(a.q + (int64_t)qrow * a.q_stride + (cons.kvh * G + min(head, G - 1)) * HD + t * (HD / 4));
        float sum = 0.f;
#pragma unroll
        for (int i = 0; i < W; ++i) {
          raw[nt][i] = head < G ? src[i] : make_uint4(0, 0, 0, 0);
          const uint32_t* u = &raw[nt][i].x;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const float x = bf_lo(u[k]), y = bf_hi(u[k]);
            sum += x + y;
            mx = fmaxf(mx, fmaxf(fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.f, fabsf(y) <= 3.402823466e38f ? fabsf(y) : 0.f));
          }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qs[nt][0] = a.scale_log2 * __shfl_sync(0xffffffffu, sum, 8 * t);
        qs[nt][1] = a.scale_log2 * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
      }
      // 2^e brings the largest finite number to 2^14 (e from -100 to 100); high nibbles count 16 times, so what they meet is q 2^(e - 4)
      const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(mx));
      const int e = top ? min(max(141 - (int)(top >> 23), -100), 100) : 0;
      const float up = __uint_as_float((uint32_t)(127 + e) << 23), up4 = __uint_as_float((uint32_t)(123 + e) << 23);
      fs = a.scale_log2 * __uint_as_float((uint32_t)(151 - e) << 23);
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < W; ++i) {
          const uint32_t* u = &raw[nt][i].x;
#pragma unroll
          for (int k = 0; k < 4; ++k) qb[nt][2 * i + (k >> 1)][k & 1] = pack_h2(bf_lo(u[k]) * (k & 1 ? up4 : up), bf_hi(u[k]) * (k & 1 ? up4 : up));
        }
    }
    float o[NM][NT][4], ws[NT][4], ref[NT][2], l[NT][2], zs[NT][2];      // ws: sums of the rounded weights, from a product with ones
#pragma unroll
    for (int i = 0; i < NM; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) { ref[nt][h] = l[nt][h] = zs[nt][h] = ws[nt][h] = ws[nt][2 + h] = 0.f; }

    bool fresh = true;                         // the first tile sets the references
    for (int tile = cons.t0; tile < cons.t1; ++tile) {
      const int key0 = sp.key0(tile) + warp * WK;
      mbar_wait(full(stage), parity);
      if (key0 >= sp.len || (key0 + WK <= sp.lo && key0 >= a.first)) {        // nobody sees these keys
        if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty(stage)) : "memory");
        advance();
        continue;
      }
      const uint8_t* base = smem + (stage * GROUPS + warp * 2) * GB;
      // ---- scores in units of log 2, less the reference: rows g and g + 8 of group i are keys key0 + 16 i + key_token(g) and 8 further
      float x[2][NT][4], zv[2][2], sv[2][2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* grp = base + i * GB;
        uint32_t ka[W], kb[W];
        if (HD == 128) {
          const uint4 u = *reinterpret_cast<const uint4*>(grp + g * 64 + t * 16), v = *reinterpret_cast<const uint4*>(grp + 512 + g * 64 + t * 16);
          ka[0] = u.x; ka[1] = u.y; ka[W - 2] = u.z; ka[W - 1] = u.w;
          kb[0] = v.x; kb[1] = v.y; kb[W - 2] = v.z; kb[W - 1] = v.w;
        } else {
          const uint2 u = *reinterpret_cast<const uint2*>(grp + g * 32 + t * 8), v = *reinterpret_cast<const uint2*>(grp + 256 + g * 32 + t * 8);
          ka[0] = u.x; ka[1] = u.y;
          kb[0] = v.x; kb[1] = v.y;
        }
        float c[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) c[nt][0] = c[nt][1] = c[nt][2] = c[nt][3] = 0.f;
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const uint32_t a0 = ka[j], b0 = kb[j], a1 = a0 >> 8, b1 = b0 >> 8;
          const uint32_t f0[4] = {codes_lo(a0), codes_lo(b0), codes_hi(a0), codes_hi(b0)}, f1[4] = {codes_lo(a1), codes_lo(b1), codes_hi(a1), codes_hi(b1)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            mma_f16(c[nt], f0, qb[nt][2 * j][0], qb[nt][2 * j][1]);
            mma_f16(c[nt], f1, qb[nt][2 * j + 1][0], qb[nt][2 * j + 1][1]);
          }
        }
        const uint32_t* par = reinterpret_cast<const uint32_t*>(grp + 16 * HD) + kv4::key_token(g);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t pk = par[8 * r], pv = par[16 + 8 * r];
          const float lk = bf_hi(pk), f = fs * bf_lo(pk);
          sv[i][r] = bf_lo(pv);
          zv[i][r] = fmaf(8.f, sv[i][r], bf_hi(pv));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) x[i][nt][2 * r + h] = fmaf(c[nt][2 * r + h], f, fmaf(qs[nt][h], lk, -ref[nt][h]));
        }
      }
      if (key0 + WK > sp.len || (key0 < sp.lo && key0 + WK > a.first)) {      // the same for the warp
        const int mine = key0 + kv4::key_token(g);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int key = mine + 16 * i + 8 * r;
            if (!(key < sp.len && (key >= sp.lo || key < a.first))) {         // its numbers may be anything
              sv[i][r] = zv[i][r] = 0.f;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) x[i][nt][2 * r] = x[i][nt][2 * r + 1] = -INFINITY;
            }
          }
      }
      // ---- weights
      uint32_t w[2][NT][2];
      float e[2][NT][4];
      auto weigh = [&]() {                     // false: a weight has passed its bound (or is NaN)
        uint32_t most = 0;
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              e[i][nt][2 * r] = ex2(x[i][nt][2 * r]);
              e[i][nt][2 * r + 1] = ex2(x[i][nt][2 * r + 1]);
              w[i][nt][r] = pack_h2(e[i][nt][2 * r] * sv[i][r], e[i][nt][2 * r + 1] * sv[i][r]);
              most = max_u16x2(most, w[i][nt][r]);
            }
        return most < (kWeightMost << 16) && (most & 0xffffu) < kWeightMost;
      };
      const bool fits = weigh();
      if (fresh || !__all_sync(0xffffffffu, fits)) {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float top = fresh ? -INFINITY : 0.f;                              // how far the reference goes up (the first: or down)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int r = 0; r < 2; ++r) top = fmaxf(top, fmaxf(x[i][nt][2 * r + h] + lg2(sv[i][r]), x[i][nt][2 * r + h] - kExpRoom));
#pragma unroll
            for (int m = 4; m < 32; m <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
            if (top == -INFINITY) top = 0.f;                                  // (only NaN rows)
            const float f = ex2(-top);
            ref[nt][h] += top;
            l[nt][h] *= f;
            zs[nt][h] *= f;
            ws[nt][h] *= f;
#pragma unroll
            for (int i = 0; i < NM; ++i) { o[i][nt][h] *= f; o[i][nt][2 + h] *= f; }
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int r = 0; r < 2; ++r) x[i][nt][2 * r + h] -= top;
          }
        weigh();
        fresh = false;
      }
      uint32_t pb[2][NT][2];
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
#pragma unroll
            for (int h = 0; h < 2; ++h) { l[nt][h] += e[i][nt][2 * r + h]; zs[nt][h] = fmaf(e[i][nt][2 * r + h], zv[i][r], zs[nt][h]); }
            pb[i][nt][r] = turn8x8(w[i][nt][r]);
          }
          const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
          mma_f16(ws[nt], ones, pb[i][nt][0], pb[i][nt][1]);
        }
      // ---- outputs: rows g and g + 8 of fragment 4 j + p are dimensions d = (HD / 8) g + 8 j + 2 p and d + 1; the keys of thread t are
      // t, t + 4, t + 8, t + 12 of the group
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint8_t* val = base + i * GB + 8 * HD;
        constexpr int VW = HD / 64;                      // words of a thread's share of a value row
        uint32_t v[4][VW];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const int tok = t + 4 * k;
          if (HD == 128) {
            const uint2 u = *reinterpret_cast<const uint2*>(val + tok * 64 + ((g ^ ((t & 2) << 1)) << 3));      // value_word(): halves exchanged
            v[k][0] = u.x; v[k][VW - 1] = u.y;
          } else {
            v[k][0] = *reinterpret_cast<const uint32_t*>(val + tok * 32 + g * 4);
          }
        }
#pragma unroll
        for (int j = 0; j < VW; ++j) {
          const uint32_t xa = __byte_perm(v[0][j], v[1][j], 0x5410), ya = __byte_perm(v[0][j], v[1][j], 0x7632);
          const uint32_t xb = __byte_perm(v[2][j], v[3][j], 0x5410), yb = __byte_perm(v[2][j], v[3][j], 0x7632);
          const uint32_t xa8 = xa >> 8, ya8 = ya >> 8, xb8 = xb >> 8, yb8 = yb >> 8;
          const uint32_t f[4][4] = {{codes_lo(xa), codes_lo(ya), codes_lo(xb), codes_lo(yb)}, {codes_hi(xa), codes_hi(ya), codes_hi(xb), codes_hi(yb)},
                                    {codes_lo(xa8), codes_lo(ya8), codes_lo(xb8), codes_lo(yb8)}, {codes_hi(xa8), codes_hi(ya8), codes_hi(xb8), codes_hi(yb8)}};
#pragma unroll
          for (int p = 0; p < 4; ++p)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) mma_f16(o[4 * j + p][nt], f[p], pb[i][nt][0], pb[i][nt][1]);
        }
      }
      __syncwarp();                                      // the stage is read
      if (lane == 0) asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(empty(stage)) : "memory");
      advance();
    }

    // ---- the warps' (ref, l, out) of the piece, four heads at a time
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 4; m < 32; m <<= 1) {
          l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], m);
          zs[nt][h] += __shfl_xor_sync(0xffffffffu, zs[nt][h], m);
        }
    const bool whole = !SPLIT || (cons.t0 == 0 && cons.t1 == cons.n);
    const int slot = SPLIT ? 2 * (int)blockIdx.x + (cons.u - (cons.t1 - cons.t0) == u0 ? 0 : 1) : 0;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int half = 0; half < 2; ++half) {             // heads 8 nt + 4 half .. + 3: threads t = 2 half and 2 half + 1 of a quad
        const int r0 = 8 * nt + 4 * half;
        if (r0 >= G) continue;
        bar_compute();                                   // the pass before is read
        if ((t >> 1) == half)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            float* dst = red + (warp * 4 + 2 * (t & 1) + h) * RS;
            const float rest = fmaf(-8.f, ws[nt][h], zs[nt][h]);
#pragma unroll
            for (int i = 0; i < NM; i += 2)              // fragments of low nibbles (even) and of high ones
              *reinterpret_cast<float4*>(dst + g * (HD / 8) + 2 * i) = make_float4(fmaf(o[i][nt][h], 16777216.f, rest), fmaf(o[i][nt][2 + h], 16777216.f, rest),
                                                                                   fmaf(o[i + 1][nt][h], 1048576.f, rest), fmaf(o[i + 1][nt][2 + h], 1048576.f, rest));
            if (g == 0) { dst[HD] = fresh ? kNoRef : ref[nt][h]; dst[HD + 1] = l[nt][h]; }      // (a warp without a tile)
          }
        bar_compute();
        for (int it = tid; it < HD; it += NW * 32) {     // (row, 4 dimensions)
          const int r = it / (HD / 4), c = it % (HD / 4);
          if (r0 + r >= G) break;
          float mm = kNoRef;
#pragma unroll
          for (int w2 = 0; w2 < NW; ++w2) mm = fmaxf(mm, red[(w2 * 4 + r) * RS + HD]);
          float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
          float ll = 0.f;
#pragma unroll
          for (int w2 = 0; w2 < NW; ++w2) {
            const float* src = red + (w2 * 4 + r) * RS;
            const float f = ex2(src[HD] - mm);
            const float4 v = *reinterpret_cast<const float4*>(src + 4 * c);
            acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
            ll = fmaf(f, src[HD + 1], ll);
          }
          if (whole) {
            const float inv = ll != 0.f ? 1.f / ll : 0.f;
            *reinterpret_cast<uint2*>(a.out + ((int64_t)qrow * a.H + cons.kvh * G + r0 + r) * HD + 4 * c) = make_uint2(pack_bf2(acc.x * inv, acc.y * inv), pack_bf2(acc.z * inv, acc.w * inv));
          } else {
            const int64_t row = (int64_t)slot * G + r0 + r;
            *reinterpret_cast<float4*>(a.part + row * HD + 4 * c) = acc;
            if (c == 0) *reinterpret_cast<float2*>(a.part + (int64_t)2 * kMaxCtas * G * HD + row * 2) = make_float2(mm, ll);
          }
        }
      }
  }
}

// The groups that were cut: block (c, head) merges the pieces of the group that begins in the share of CTA c, in the order of the shares.
template <int HD>
__global__ void __launch_bounds__(HD) attn_kv4_merge_kernel(bf16* __restrict__ out, const float* __restrict__ part, const int4* __restrict__ desc, int H, int G) {
  pdl_launch_dependents();
  pdl_wait();
  __shared__ float4 sh[4][HD / 4];
  __shared__ float sl[4];
  const int4 d = desc[blockIdx.x];
  if (d.x < 0) return;
  const int c = blockIdx.x, r = blockIdx.y, n = d.z - c + 1, lane = threadIdx.x % (HD / 4), q = threadIdx.x / (HD / 4);      // four streams of pieces
  const float* ml = part + (int64_t)2 * kMaxCtas * G * HD;
  auto row = [&](int i) { return (int64_t)(2 * (c + i) + (i == 0 ? d.w : 0)) * G + r; };
  float mm = kNoRef;
  for (int i = 0; i < n; ++i) mm = fmaxf(mm, ml[row(i) * 2]);
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  float ll = 0.f;
#pragma unroll 4
  for (int i = q; i < n; i += 4) {
    const float2 p = *reinterpret_cast<const float2*>(ml + row(i) * 2);
    const float4 v = *reinterpret_cast<const float4*>(part + row(i) * HD + 4 * lane);
    const float f = ex2(p.x - mm);
    acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
    ll = fmaf(f, p.y, ll);
  }
  sh[q][lane] = acc;
  if (lane == 0) sl[q] = ll;
  __syncthreads();
  if (q == 0) {
    for (int k = 1; k < 4; ++k) {
      const float4 v = sh[k][lane];
      acc.x += v.x; acc.y += v.y; acc.z += v.z; acc.w += v.w;
      ll += sl[k];
    }
    const float inv = ll != 0.f ? 1.f / ll : 0.f;
    *reinterpret_cast<uint2*>(out + ((int64_t)d.x * H + d.y * G + r) * HD + 4 * lane) = make_uint2(pack_bf2(acc.x * inv, acc.y * inv), pack_bf2(acc.z * inv, acc.w * inv));
  }
}

constexpr int64_t workspace_bytes(int G, int hd) { return (int64_t)kMaxCtas * 16 + (int64_t)2 * kMaxCtas * G * (hd + 2) * 4; }
constexpr int kMaxRequests = 1024;             // requests of one launch (their tile counts lie in shared memory)

template <int HD, int NT>
static int launch(const Args& a, int max_seq_len, cudaStream_t st) {
  const int max_tiles = (max_seq_len + TK - 1) / TK;
  const int fixed = ring_bytes<HD, NT>() + red_floats<HD>() * 4 + 2 * stages(NT) * 8, ctas = 148 * ctas_per_sm(NT);
  if (max_tiles <= 4) {
    auto kern = attn_kv4_kernel<HD, NT, false>;
    KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, fixed));
    KGE_CUDA_OK(launch_pdl(kern, dim3(a.KV, a.B), dim3(kThreads), fixed, st, a, 0));
    return 0;
  }
  auto kern = attn_kv4_kernel<HD, NT, true>;
  const int smem = fixed + (a.B + 1) * 4;
  KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, fixed + (kMaxRequests + 1) * 4));
  KGE_CUDA_OK(launch_pdl(kern, dim3(ctas), dim3(kThreads), smem, st, a, 1));
  KGE_CUDA_OK(launch_pdl(attn_kv4_merge_kernel<HD>, dim3(ctas, a.H / a.KV), dim3(HD), 0, st, a.out, (const float*)a.part, (const int4*)a.desc, a.H, a.H / a.KV));
  return 0;
}

}  // namespace ak4

static int decode(ak4::Args a, int hd, int max_seq_len, cudaStream_t st) {
  const int B = a.B, G = a.H / a.KV;
  // requests of a launch: what shared memory has room for, and tiles that 32 bits count (a table's row bounds a request's)
  const int64_t tiles = ((((int64_t)a.max_blocks << a.bs_shift) + ak4::TK - 1) / ak4::TK + 1) * a.KV;
  const int most = (int)std::max<int64_t>(1, std::min<int64_t>(ak4::kMaxRequests, ((1ll << 31) - 1) / tiles));
  for (int b0 = 0; b0 < B; b0 += most) {
    ak4::Args p = a;
    p.B = std::min(B - b0, most);
    p.table += (int64_t)b0 * a.max_blocks; p.lens += b0; p.qsl += b0;
    int rc;
    if (hd == 128) rc = G <= 8 ? ak4::launch<128, 1>(p, max_seq_len, st) : ak4::launch<128, 2>(p, max_seq_len, st);
    else rc = G <= 8 ? ak4::launch<64, 1>(p, max_seq_len, st) : ak4::launch<64, 2>(p, max_seq_len, st);
    if (rc) return rc;
  }
  return 0;
}

int paged_attn_kv4_tc(bf16* out, const bf16* q, int q_stride, const uint8_t* cache, const int32_t* bt, int max_blocks, const int32_t* sl, const int32_t* qsl, int B, int T,
                      int max_q_len, int max_seq_len, int H, int KV, int hd, int bs, float scale, int window, int first, bool skip_single, cudaStream_t st);      // attn_tc.cu

}  // namespace KGE_ELT_NS
}  // namespace kge

using namespace kge;

#ifndef KGE_HALF
extern "C" int64_t kge_attn_kv4_workspace_bytes(int H, int KV, int hd) {
  if (H <= 0 || KV <= 0 || H % KV || (hd != 64 && hd != 128)) {
    kge::set_error("kge_attn_kv4_workspace_bytes: H=%d KV=%d head_dim=%d", H, KV, hd);
    return -1;
  }
  return H / KV <= 16 ? ak4::workspace_bytes(H / KV, hd) : 0;
}
#endif

extern "C" int KGE_API(kge_paged_attn_kv4)(void* out, const void* q, int q_stride, const void* kv_cache, const int32_t* block_table, int max_blocks_per_seq,
                                           const int32_t* seq_lens, const int32_t* query_start_loc, int B, int T, int max_q_len, int max_seq_len, int H, int KV, int hd,
                                           int block_size, float scale, int window, int first, void* workspace, int64_t workspace_bytes, void* stream) {
  KGE_REQUIRE(out && q && kv_cache && block_table && seq_lens && query_start_loc, "kge_paged_attn_kv4: null pointer");
  KGE_REQUIRE(H > 0 && KV > 0 && H % KV == 0 && H / KV <= 128, "kge_paged_attn_kv4: H=%d must be a multiple of KV=%d, at most 128 times it", H, KV);
  KGE_REQUIRE(hd == 64 || hd == 128, "kge_paged_attn_kv4: head_dim=%d unsupported (64, 128)", hd);
  KGE_REQUIRE(block_size >= 16 && block_size <= 4096 && (block_size & (block_size - 1)) == 0, "kge_paged_attn_kv4: block_size=%d must be a power of two, 16 to 4096", block_size);
  KGE_REQUIRE(q_stride % 8 == 0 && q_stride >= H * hd, "kge_paged_attn_kv4: q_stride=%d must be a multiple of 8, at least H * hd", q_stride);
  KGE_REQUIRE((((uintptr_t)out | (uintptr_t)q | (uintptr_t)kv_cache | (uintptr_t)workspace) & 15) == 0, "kge_paged_attn_kv4: pointers must be 16-byte aligned");
  KGE_REQUIRE(window >= 0 && first >= 0, "kge_paged_attn_kv4: window=%d first=%d", window, first);
  KGE_REQUIRE(scale > 0.f && scale < 3e38f, "kge_paged_attn_kv4: scale=%g must be positive", (double)scale);
  if (B <= 0 || T <= 0) return 0;
  KGE_REQUIRE(B <= 65535, "kge_paged_attn_kv4: %d requests (at most 65535)", B);
  KGE_REQUIRE(max_q_len >= 1 && max_seq_len >= 1 && max_blocks_per_seq >= 1, "kge_paged_attn_kv4: max_q_len / max_seq_len / max_blocks_per_seq must be >= 1");
  KGE_REQUIRE((int64_t)max_blocks_per_seq * block_size < (1ll << 31), "kge_paged_attn_kv4: %d blocks of %d tokens a request", max_blocks_per_seq, block_size);
  cudaStream_t st = (cudaStream_t)stream;
  const int G = H / KV;
  const bool single = G <= 16;                 // a kernel of their own for single-token requests
  if (!single || max_q_len > 1)
    if (int rc = paged_attn_kv4_tc((bf16*)out, (const bf16*)q, q_stride, (const uint8_t*)kv_cache, block_table, max_blocks_per_seq, seq_lens, query_start_loc, B, T, max_q_len,
                                   max_seq_len, H, KV, hd, block_size, scale, window, first, single, st))
      return rc;
  if (!single) return 0;
  const int64_t need = ak4::workspace_bytes(G, hd);
  KGE_REQUIRE(workspace && workspace_bytes >= need, "kge_paged_attn_kv4: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
  ak4::Args a;
  a.out = (bf16*)out; a.q = (const bf16*)q; a.cache = (const uint8_t*)kv_cache;
  a.table = block_table; a.lens = seq_lens; a.qsl = query_start_loc;
  a.desc = (int4*)workspace; a.part = (float*)((uint8_t*)workspace + (int64_t)ak4::kMaxCtas * 16);
  a.q_stride = q_stride; a.max_blocks = max_blocks_per_seq; a.B = B; a.H = H; a.KV = KV;
  a.bs_shift = 4;
  while ((1 << a.bs_shift) < block_size) ++a.bs_shift;
  a.window = window; a.first = first; a.scale_log2 = scale * ak4::kLog2e;
  return decode(a, hd, max_seq_len, st);
}
