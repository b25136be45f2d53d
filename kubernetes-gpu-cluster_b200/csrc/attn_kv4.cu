// Attention over the 4-bit key-value cache (layout: kv4.cuh), single-token requests; prompts: attn_kv4_tc.cuh.
//
// With key k = low_k + s_k n_k and value v = low_v + s_v n_v (n: codes 0..15), z = low + 8 s,
//   score = scale (s_k (q . n_k) + low_k sum(q))           out = (sum_j (p_j s_v,j) (n_v,j - 8) + sum_j p_j z_v,j) / sum_j p_j
// so the products run on codes, which 16 bits hold exactly, and the two numbers of a row are applied to scores and weights in fp32.
//
// A warp takes 32 keys at a time (a unit) from a ring of its own, which its lane 0 fills by bulk copies, and multiplies with mma.m16n8k16 whose M
// side is the keys (scores) or the dimensions (outputs) and whose N side is the query heads of one kv head: 8 columns of which a group of 4 or
// 8 heads leaves few empty, half the products that heads as the M side cost.  Both operands are float16 in either build.
//   Codes: the bits n in the low half-byte of a float16 are the number n 2^-24 (its denormals), in the next one n 2^-20, so a code costs half an
//   AND and no arithmetic; powers of two are put right in q (scores) and in the outputs.  (As 1024 + n less 1032: 2.6 instructions a pair.)
//   q: a power of two moves the largest number of the group's heads to 2^14, or of each head where they lie 2^10 apart; exact but for what lies
//   2^-24 below that.
//   Weights: w = e s_v with e = 2^(x - R), rounded to float16; R is a reference per head, such that the largest w of a warp lies between 1 and
//   2^14.  It moves only when a weight would pass that, so most tiles rescale nothing and need no shuffles.  What is taken off for centring, 8
//   times the sum of the weights, is the sum of the ROUNDED ones (a product with ones), so a rounding's error meets |n - 8| and not n.
//   Weights say nothing of e where a row's values are one constant (s_v = 0) or nearly, e ends before it counts for nothing where s_v is 2^80 and
//   more, and a score of 2^20 and more leaves a sum with log2(s_v) little of that.  Such units and heads take a path of their own (Core::hard), which
//   looks at the sums of e and e z_v too, keeps R in two parts and lets e become denormal.
//   scores come out as (key, head) fragments; movmatrix turns a packed 8 x 8 of weights into the B operand of the second product
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kge.h"
#include "kv4.cuh"

namespace kge {
inline namespace KGE_ELT_NS {

namespace ak4 {

constexpr int WK = 32, NW = 4, GROUPS = NW * WK / 16;       // keys of a unit, which a warp takes at a time; computing warps of a CTA; groups of a stage
__host__ __device__ constexpr int ctas_per_sm(int nt) { return nt == 1 ? 3 : 2; }
__host__ __device__ constexpr int stages(int nt) { return nt == 1 ? 3 : 4; }
__host__ __device__ constexpr int shares_of(int nt) { return 148 * ctas_per_sm(nt); }
constexpr int kMaxShares = 148 * 3;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRoom = 90.f, kRoomDown = 0x1p-90f;      // log2 of what e and e z_v may be when a reference is set; the least s_v that keeps them there
constexpr float kSumMost = 0x1p100f;           // what a unit's sums of e and e z_v may be
constexpr float kDeep = 80.f, kDeepMost = 0x1p80f, kSteep = 0x1p20f;      // a reference this far above its largest score, or this large, is for the hard path
constexpr uint32_t kWeightMost = 0x7400;       // 2^14 in float16

struct Args {
  bf16* out;
  const bf16* q;
  const uint8_t* cache;
  const int32_t *table, *lens, *qsl;
  float* part;                                 // outputs of the pieces of cut groups: [2 per share][G][HD], then [2 per share][G] Parts of 16 bytes
  int4* desc;                                  // per share: the group that begins in it and ends in a later one's: (row of q, kv head, last share, slot)
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
// the same into fresh accumulators
__device__ __forceinline__ void mma_f16_first(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
               : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.f));
}
__device__ __forceinline__ uint32_t lds32(uint32_t at) { uint32_t v; asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at)); return v; }
__device__ __forceinline__ uint2 lds64(uint32_t at) { uint2 v; asm volatile("ld.shared.v2.b32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(at)); return v; }
__device__ __forceinline__ uint4 lds128(uint32_t at) {
  uint4 v;
  asm volatile("ld.shared.v4.b32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at));
  return v;
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {
  uint32_t r;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
  return r;
}
__device__ __forceinline__ float ex2(float x) { float y; asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ float ex2_all(float x) { float y; asm("ex2.approx.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }      // (denormal results too)
__device__ __forceinline__ float lg2(float x) { float y; asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x)); return y; }
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
// nibbles 0 and 4, or 1 and 5, of w as two float16 numbers: n 2^-24 and n 2^-20
__device__ __forceinline__ uint32_t codes_lo(uint32_t w) { return w & 0x000f000fu; }
__device__ __forceinline__ uint32_t codes_hi(uint32_t w) { return w & 0x00f000f0u; }
__device__ __forceinline__ void ldsm_x4_trans(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at));
}
__device__ __forceinline__ uint32_t max_u16x2(uint32_t a, uint32_t b) {
  uint32_t r;
  asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  return r;
}

// The keys that a single-token request of `len` keys sees, in units of WK: the first ones that stay visible, then the window.
struct Span {
  int len, lo, npre, win0, n;
  Span() = default;
  __device__ __forceinline__ Span(int kv_len, int window, int first) {
    len = kv_len;
    lo = window > 0 ? max(kv_len - window, 0) : 0;
    win0 = lo / WK;
    npre = min((min(first, lo) + WK - 1) / WK, win0);
    n = kv_len > 0 ? npre + (kv_len + WK - 1) / WK - win0 : 1;        // (one empty unit writes the zeros of a request without keys)
  }
  __device__ __forceinline__ int key0(int unit) const { return (unit < npre ? unit : win0 + unit - npre) * WK; }
};
// One warp's work on one (request, kv head): the query heads as B operands, and what has been summed so far.  Column n of block nt is head
// 8 nt + n; of the accumulators, thread (g, t) = (lane / 4, lane % 4) has columns 2 t and 2 t + 1.
template <int HD, int NT>
struct Core {
  static constexpr int GB = kv4::group_bytes(HD), W = HD / 32, NM = HD / 16;      // W: words of a thread's share of a key row
  uint32_t qb[NT][NM][2];
  float qs[NT][2], fs;                         // scale log2(e) sum(q) of the two columns; what scores are multiplied with
  float o[NM][NT][4], ws[NT][4];               // outputs; sums of the rounded weights, from a product with ones
  float ref[NT][2], l[NT][2], zs[NT][2];
  bool fresh, hard, uneven;                    // the first unit sets the references; they have two parts, or e may be denormal; heads have an fs each

  __device__ __forceinline__ void start(const bf16* q, int G, float scale_log2, int lane, float* lows) {
    const int g = lane >> 2, t = lane & 3;
    uint4 raw[NT][W];
    float mx[NT], most = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int head = nt * 8 + g;
      const uint4* src = reinterpret_cast<const uint4*>(q + min(head, G - 1) * HD + t * (HD / 4));
      float sum = 0.f;
      mx[nt] = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        raw[nt][i] = head < G ? src[i] : make_uint4(0, 0, 0, 0);
        const uint32_t* u = &raw[nt][i].x;
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float x = bf_lo(u[k]), y = bf_hi(u[k]);
          sum += x + y;
          mx[nt] = fmaxf(mx[nt], fmaxf(fabsf(x) <= 3.402823466e38f ? fabsf(x) : 0.f, fabsf(y) <= 3.402823466e38f ? fabsf(y) : 0.f));
        }
      }
      most = fmaxf(most, mx[nt]);
      sum += __shfl_xor_sync(0xffffffffu, sum, 1);
      sum += __shfl_xor_sync(0xffffffffu, sum, 2);
      qs[nt][0] = scale_log2 * __shfl_sync(0xffffffffu, sum, 8 * t);
      qs[nt][1] = scale_log2 * __shfl_sync(0xffffffffu, sum, 8 * t + 4);
    }
    // 2^e brings the largest finite number to 2^14 (e from -100 to 100), of all heads or, where these lie 2^10 apart, of each; high nibbles count 16
    // times, so what they meet is q 2^(e - 4)
    auto exponent = [](uint32_t top) { return top ? min(max(141 - (int)(top >> 23), -100), 100) : 0; };
    auto factor = [&](int e) { return scale_log2 * __uint_as_float((uint32_t)(151 - e) << 23); };
    const uint32_t top = __reduce_max_sync(0xffffffffu, __float_as_uint(most));
    int es[NT];
    uneven = false;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      es[nt] = exponent(top);
      auto heads = [](uint32_t lanes) { return (lanes | lanes >> 1 | lanes >> 2 | lanes >> 3) & 0x11111111u; };
      uneven |= (heads(__ballot_sync(0xffffffffu, mx[nt] > 0.f)) & ~heads(__ballot_sync(0xffffffffu, mx[nt] >= __uint_as_float(top) * 0x1p-10f))) != 0;
    }
    fs = factor(es[0]);
    if (uneven) {                              // the same for the warp
#pragma unroll
      for (int nt = 0; nt < NT; ++nt) {
        mx[nt] = fmaxf(mx[nt], __shfl_xor_sync(0xffffffffu, mx[nt], 1));
        mx[nt] = fmaxf(mx[nt], __shfl_xor_sync(0xffffffffu, mx[nt], 2));
        es[nt] = exponent(__float_as_uint(mx[nt]));
        if (t == 0) lows[8 * (NT + nt) + g] = factor(es[nt]);
      }
      __syncwarp();
    }
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const float up = __uint_as_float((uint32_t)(127 + es[nt]) << 23), up4 = __uint_as_float((uint32_t)(123 + es[nt]) << 23);
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const uint32_t* u = &raw[nt][i].x;
#pragma unroll
        for (int k = 0; k < 4; ++k) qb[nt][2 * i + (k >> 1)][k & 1] = pack_h2(bf_lo(u[k]) * (k & 1 ? up4 : up), bf_hi(u[k]) * (k & 1 ? up4 : up));
      }
#pragma unroll
      for (int i = 0; i < NM; ++i) o[i][nt][0] = o[i][nt][1] = o[i][nt][2] = o[i][nt][3] = 0.f;
#pragma unroll
      for (int h = 0; h < 2; ++h) ref[nt][h] = l[nt][h] = zs[nt][h] = ws[nt][h] = ws[nt][2 + h] = 0.f;
    }
    fresh = true;
    hard = false;
  }

  // The hard path: weights and exponentials of any finite rows, references in two parts.
  __device__ __forceinline__ void reweigh(float (&x)[2][NT][4], const float (&sv)[2][2], const float (&zv)[2][2], float (&e)[2][NT][4], uint32_t (&wt)[2][NT][2], int t, int lane,
                                          float* lows) {
    bool harder = hard;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        float* low_at = lows + 8 * nt + 2 * t + h;
        float low = hard ? *low_at : 0.f;
#pragma unroll
        for (int i = 0; i < 2; ++i) { x[i][nt][h] -= low; x[i][nt][2 + h] -= low; }
        auto weigh = [&]() {                   // true: does not fit
          float sum_e = 0.f, sum_z = 0.f, w_most = 0.f;
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
              const float v = ex2_all(x[i][nt][2 * r + h]);
              e[i][nt][2 * r + h] = v;
              sum_e += v;
              sum_z = fmaf(v, zv[i][r], sum_z);
              w_most = fmaxf(w_most, v * sv[i][r]);
            }
          return !(fmaxf(sum_e, fabsf(sum_z)) < kSumMost && w_most < 16384.f);
        };
        // only a column that has passed a bound moves
        const bool over = __ballot_sync(0xffffffffu, weigh()) & (0x11111111u << t);
        float high = -INFINITY, top = -INFINITY;                  // of the column's scores; of what they are with their rows' numbers, less that
#pragma unroll
        for (int i = 0; i < 2; ++i) high = fmaxf(high, fmaxf(x[i][nt][h], x[i][nt][2 + h]));
#pragma unroll
        for (int m = 4; m < 32; m <<= 1) high = fmaxf(high, __shfl_xor_sync(0xffffffffu, high, m));
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
          for (int r = 0; r < 2; ++r)
            top = fmaxf(top, x[i][nt][2 * r + h] - high + fmaxf(lg2(sv[i][r]), fmaxf(lg2(fabsf(zv[i][r])) - kRoom, -kRoom)));
#pragma unroll
        for (int m = 4; m < 32; m <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
        const float up = high + top;                              // how far the reference goes up (the first: or down)
        if (fabsf(up) < INFINITY && (fresh || (over && up > 0.f))) {       // (not: only NaN rows)
          const bool steep = hard || fabsf(ref[nt][h]) + fabsf(up) > kSteep;
          ref[nt][h] += steep ? high : up;
          low += steep ? top : 0.f;
          harder |= steep || top > kDeep;
          const float f = fresh ? 1.f : ex2(-0.5f * up);          // twice the half: the sums may be as large as the change
          l[nt][h] = l[nt][h] * f * f;
          zs[nt][h] = zs[nt][h] * f * f;
          ws[nt][h] = ws[nt][h] * f * f;
#pragma unroll
          for (int i = 0; i < NM; ++i) { o[i][nt][h] = o[i][nt][h] * f * f; o[i][nt][2 + h] = o[i][nt][2 + h] * f * f; }
#pragma unroll
          for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 2; ++r) x[i][nt][2 * r + h] = x[i][nt][2 * r + h] - high - top;
          weigh();
        }
        __syncwarp();
        if ((lane >> 2) == 0) *low_at = low;
      }
    fresh = false;
    hard = __any_sync(0xffffffffu, harder);
    __syncwarp();                                                 // (`lows`)
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 2; ++r) wt[i][nt][r] = pack_h2(e[i][nt][2 * r] * sv[i][r], e[i][nt][2 * r + 1] * sv[i][r]);
  }

  // A unit whose two groups lie at shared address `at`.  edge: some of its keys are not visible - those from `len` on, and those below `lo` but
  // the first `first` ones.
  // lows: numbers of the warp's own in shared memory, 8 NT for the references' other parts, R = ref + low, and an fs for each of 8 NT heads.
  __device__ __forceinline__ void unit(uint32_t at, int lane, bool edge, int key0, int len, int lo, int first, float* lows) {
    const int g = lane >> 2, t = lane & 3;
    const uint32_t k_at = at + g * (HD / 2) + t * (HD / 8), n_at = at + 16 * HD + kv4::key_token(g) * 4;
    // ---- scores in units of log 2, less the reference: rows g and g + 8 of group i are keys key0 + 16 i + key_token(g) and 8 further
    float x[2][NT][4], zv[2][2], sv[2][2];
    auto scores = [&](auto each) {             // each: heads have an fs of their own (a path of its own: 2 % of long batches' time in the other)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        uint32_t ka[W], kb[W];
        if (HD == 128) {
          const uint4 u = lds128(k_at + i * GB), v = lds128(k_at + i * GB + 512);
          ka[0] = u.x; ka[1] = u.y; ka[W - 2] = u.z; ka[W - 1] = u.w;
          kb[0] = v.x; kb[1] = v.y; kb[W - 2] = v.z; kb[W - 1] = v.w;
        } else {
          const uint2 u = lds64(k_at + i * GB), v = lds64(k_at + i * GB + 256);
          ka[0] = u.x; ka[1] = u.y;
          kb[0] = v.x; kb[1] = v.y;
        }
        float c[NT][4];
#pragma unroll
        for (int j = 0; j < W; ++j) {
          const uint32_t a0 = ka[j], b0 = kb[j], a1 = a0 >> 8, b1 = b0 >> 8;
          const uint32_t f0[4] = {codes_lo(a0), codes_lo(b0), codes_hi(a0), codes_hi(b0)}, f1[4] = {codes_lo(a1), codes_lo(b1), codes_hi(a1), codes_hi(b1)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            if (j == 0) mma_f16_first(c[nt], f0, qb[nt][0][0], qb[nt][0][1]);
            else mma_f16(c[nt], f0, qb[nt][2 * j][0], qb[nt][2 * j][1]);
            mma_f16(c[nt], f1, qb[nt][2 * j + 1][0], qb[nt][2 * j + 1][1]);
          }
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const uint32_t pk = lds32(n_at + i * GB + 32 * r), pv = lds32(n_at + i * GB + 64 + 32 * r);
          const float lk = bf_hi(pk), f = fs * bf_lo(pk);
          sv[i][r] = bf_lo(pv);
          zv[i][r] = fmaf(8.f, sv[i][r], bf_hi(pv));
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int h = 0; h < 2; ++h) x[i][nt][2 * r + h] = fmaf(c[nt][2 * r + h], decltype(each)::value ? lows[8 * (NT + nt) + 2 * t + h] * bf_lo(pk) : f, fmaf(qs[nt][h], lk, -ref[nt][h]));
        }
      }
    };
    if (uneven) scores(std::true_type());      // the same for the warp
    else scores(std::false_type());
    if (edge) {                                // the same for the warp
      const int mine = key0 + kv4::key_token(g);
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = mine + 16 * i + 8 * r;
          if (!(key < len && (key >= lo || key < first))) {       // its numbers may be anything
            sv[i][r] = 1.f;                      // (which makes nothing of a weight of zero)
            zv[i][r] = 0.f;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) x[i][nt][2 * r] = x[i][nt][2 * r + 1] = -INFINITY;
          }
        }
    }
    // ---- weights
    uint32_t wt[2][NT][2];
    float e[2][NT][4];
    auto weigh = [&]() {                       // false: a weight has passed its bound (or is NaN)
      uint32_t most = 0;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            e[i][nt][2 * r] = ex2(x[i][nt][2 * r]);
            e[i][nt][2 * r + 1] = ex2(x[i][nt][2 * r + 1]);
            wt[i][nt][r] = pack_h2(e[i][nt][2 * r] * sv[i][r], e[i][nt][2 * r + 1] * sv[i][r]);
            most = max_u16x2(most, wt[i][nt][r]);
          }
      return most < (kWeightMost << 16) && (most & 0xffffu) < kWeightMost;
    };
    const bool fits = weigh();
    // Small weights say that e and e z_v are small where no s_v is zero (it is 2^-16 |z_v| then, or more) or next to it.
    const bool plain = fminf(fminf(sv[0][0], sv[0][1]), fminf(sv[1][0], sv[1][1])) >= kRoomDown;
    if (!__all_sync(0xffffffffu, fits & plain & !fresh & !hard)) {
      bool wide = hard || !plain || fmaxf(fmaxf(sv[0][0], sv[0][1]), fmaxf(sv[1][0], sv[1][1])) > kDeepMost;      // for the hard path
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const float high = fmaxf(fmaxf(x[0][nt][h], x[0][nt][2 + h]), fmaxf(x[1][nt][h], x[1][nt][2 + h]));
          wide |= fabsf(ref[nt][h]) > kSteep || (fabsf(high) > kSteep && fabsf(high) < INFINITY);
        }
      if (__any_sync(0xffffffffu, wide)) {
        reweigh(x, sv, zv, e, wt, t, lane, lows);
      } else {
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            // only a column that has passed the bound moves: what a head gets does not hang on its neighbours
            uint32_t most = 0;
#pragma unroll
            for (int i = 0; i < 2; ++i) most = max_u16x2(most, max_u16x2(wt[i][nt][0], wt[i][nt][1]));
            const bool over = __ballot_sync(0xffffffffu, (h ? most >> 16 : most & 0xffffu) >= kWeightMost) & (0x11111111u << t);
            float top = fresh ? -INFINITY : 0.f;                    // how far the reference goes up (the first: or down)
#pragma unroll
            for (int i = 0; i < 2; ++i)
#pragma unroll
              for (int r = 0; r < 2; ++r) top = fmaxf(top, x[i][nt][2 * r + h] + lg2(sv[i][r]));
#pragma unroll
            for (int m = 4; m < 32; m <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, m));
            if (top == -INFINITY || !(fresh || over)) top = 0.f;    // (the first: only NaN rows)
            const float f = fresh ? 1.f : ex2(-top);                // (2^-top may be infinite where the first one goes down, and the sums are zeros)
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
          pb[i][nt][r] = turn8x8(wt[i][nt][r]);
        }
        const uint32_t ones[4] = {0x3c003c00u, 0x3c003c00u, 0x3c003c00u, 0x3c003c00u};
        mma_f16(ws[nt], ones, pb[i][nt][0], pb[i][nt][1]);
      }
    // ---- outputs: a transposing ldmatrix of 16-bit pieces (four codes each) hands a thread the pieces g of two keys, rows 2 t and 2 t + 1 of
    // eight; rows are keys in the order of the scores' rows.  Matrices: pieces 8 q .. 8 q + 7 of the first and second eight keys, q = 2 m and
    // 2 m + 1; kv4::value_word exchanges halves of rows.  Row g of fragment 4 m + p is dimension 64 m + 8 (g / 2) + 2 p + g % 2, row g + 8 is 32
    // further.
    const int tok = ((lane >> 4) << 3) | kv4::key_token(lane & 7), q0 = (lane >> 3) & 1;
    const uint32_t v_at = at + 8 * HD + tok * (HD / 2) + (HD == 128 ? (q0 ^ (tok & 2)) * 16 : q0 * 16);
#pragma unroll
    for (int i = 0; i < 2; ++i)
#pragma unroll
      for (int m = 0; m < HD / 64; ++m) {
        uint32_t v[4];
        ldsm_x4_trans(v, (v_at + i * GB) ^ (m * 32));
        const uint32_t u[4] = {v[0] >> 8, v[1] >> 8, v[2] >> 8, v[3] >> 8};
        const uint32_t f[4][4] = {{codes_lo(v[0]), codes_lo(v[1]), codes_lo(v[2]), codes_lo(v[3])}, {codes_hi(v[0]), codes_hi(v[1]), codes_hi(v[2]), codes_hi(v[3])},
                                  {codes_lo(u[0]), codes_lo(u[1]), codes_lo(u[2]), codes_lo(u[3])}, {codes_hi(u[0]), codes_hi(u[1]), codes_hi(u[2]), codes_hi(u[3])}};
#pragma unroll
        for (int p = 0; p < 4; ++p)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) mma_f16(o[4 * m + p][nt], f[p], pb[i][nt][0], pb[i][nt][1]);
      }
  }

  __device__ __forceinline__ void sums() {     // over the lanes of a column
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int m = 4; m < 32; m <<= 1) {
          l[nt][h] += __shfl_xor_sync(0xffffffffu, l[nt][h], m);
          zs[nt][h] += __shfl_xor_sync(0xffffffffu, zs[nt][h], m);
        }
  }
  // Eight dimensions from dim(m) on of this thread's column h of block nt; the lanes of g and g ^ 1 exchange what the other's eight have.  Low
  // nibbles (p even) count 2^24, high ones 2^20.
  static __device__ __forceinline__ int dim(int m, int lane) { return 64 * m + 32 * ((lane >> 2) & 1) + 8 * (lane >> 3); }
  __device__ __forceinline__ void rows(int nt, int h, int m, int lane, float (&v)[8]) const {
    const float rest = fmaf(-8.f, ws[nt][h], zs[nt][h]);
    const bool odd = lane & 4;
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      const float up = p & 1 ? 1048576.f : 16777216.f, near = fmaf(o[4 * m + p][nt][h], up, rest), far = fmaf(o[4 * m + p][nt][2 + h], up, rest);
      const float got = __shfl_xor_sync(0xffffffffu, odd ? near : far, 4);
      v[2 * p] = odd ? got : near;
      v[2 * p + 1] = odd ? far : got;
    }
  }
};

__device__ __forceinline__ void bar_compute() { asm volatile("bar.sync 1, 128;" ::: "memory"); }      // the computing warps
template <int HD> __host__ __device__ constexpr int red_floats() { return NW * 4 * (HD + 4); }

// Part of a head's keys: R = x + m (m -inf: no keys) and the sum of e.  Parts are joined in units of the largest R.
struct Part { float x, m, l; };
__device__ __forceinline__ Part no_part() { return {0.f, -INFINITY, 0.f}; }
__device__ __forceinline__ bool above(const Part& a, const Part& b) { return a.m > -INFINITY && (b.m == -INFINITY || (a.x - b.x) + (a.m - b.m) > 0.f); }
// 2^((a - b) / 2) of their R: a sum of e may be as large as the difference is, so it is multiplied twice
__device__ __forceinline__ float half_of(const Part& a, const Part& b) { return a.m == -INFINITY ? 0.f : ex2(0.5f * ((a.x - b.x) + (a.m - b.m))); }

// The four warps' sums of one (request, kv head) in shared memory, four heads at a time: write(row, first of four dimensions, part, values)
template <int HD, int NT, typename F>
__device__ __forceinline__ void combine(Core<HD, NT>& core, const float* lows, float* red, int warp, int lane, int G, F write) {
  constexpr int RS = HD + 4, NV = HD / 64;
  const int t = lane & 3;
  core.sums();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt) {
    if (8 * nt >= G) break;
    float v[2][NV][8];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int m = 0; m < NV; ++m) core.rows(nt, h, m, lane, v[h][m]);
    // (not unrolled: what a CTA runs once costs it the way of its code from the L2; 16 requests of 2048 keys, 16 heads to a kv head, 26.7 us against 23.0)
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {               // heads 8 nt + 4 half .. + 3: threads t = 2 half and 2 half + 1 of a quad
      const int r0 = 8 * nt + 4 * half;
      if (r0 >= G) break;
      bar_compute();                                     // what was there is read
      if ((t >> 1) == half)
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          float* dst = red + (warp * 4 + 2 * (t & 1) + h) * RS;
#pragma unroll
          for (int m = 0; m < NV; ++m) {
            float4* at = reinterpret_cast<float4*>(dst + core.dim(m, lane));
            at[0] = make_float4(v[h][m][0], v[h][m][1], v[h][m][2], v[h][m][3]);
            at[1] = make_float4(v[h][m][4], v[h][m][5], v[h][m][6], v[h][m][7]);
          }
          if (lane < 4) {
            dst[HD] = core.ref[nt][h];
            dst[HD + 1] = core.fresh ? -INFINITY : core.hard ? lows[8 * nt + 2 * t + h] : 0.f;      // (fresh: a warp without a unit)
            dst[HD + 2] = core.l[nt][h];
          }
        }
      bar_compute();
      for (int it = warp * 32 + lane; it < HD; it += NW * 32) {       // (row, 4 dimensions)
        const int r = it / (HD / 4), c = it % (HD / 4);
        if (r0 + r >= G) break;
        auto part_of = [&](int w) { const float* src = red + (w * 4 + r) * RS + HD; return Part{src[0], src[1], src[2]}; };
        Part all = no_part();
#pragma unroll
        for (int w = 0; w < NW; ++w)
          if (above(part_of(w), all)) all = part_of(w);
        all.l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < NW; ++w) {
          const Part p = part_of(w);
          const float half = half_of(p, all), f = half * half;
          const float4 u = *reinterpret_cast<const float4*>(red + (w * 4 + r) * RS + 4 * c);
          acc.x = fmaf(f, u.x, acc.x); acc.y = fmaf(f, u.y, acc.y); acc.z = fmaf(f, u.z, acc.z); acc.w = fmaf(f, u.w, acc.w);
          all.l = fmaf(half, half * p.l, all.l);
        }
        write(r0 + r, 4 * c, all, acc);
      }
    }
  }
}
__device__ __forceinline__ uint2 divided(float4 v, float l) {
  const float inv = l != 0.f ? 1.f / l : 0.f;
  return make_uint2(pack_bf2(v.x * inv, v.y * inv), pack_bf2(v.z * inv, v.w * inv));
}

__device__ __forceinline__ void mbar_init(uint32_t bar, int count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void mbar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void mbar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// `groups` groups of one block from `key` on
template <int HD>
__device__ __forceinline__ void copy_groups(const Args& a, uint32_t dst, int blk, int kvh, int key, int groups, uint32_t bar) {
  bulk_load(dst, a.cache + ((((int64_t)blk * a.KV + kvh) << (a.bs_shift - 4)) + ((key & ((1 << a.bs_shift) - 1)) >> 4)) * kv4::group_bytes(HD), groups * kv4::group_bytes(HD), bar);
}

// ---- short contexts: a CTA per (request, kv head), its warps take every fourth unit.  A warp fills a ring of its own: lane 0 (and lane 1, where a
// unit lies in two blocks) asks for a unit, and asks again in a stage that the warp itself has read, so there is nothing else to wait for.
template <int HD, int NT>
__global__ void __launch_bounds__(NW * 32, NT == 1 ? 4 : 3) attn_kv4_kernel(const Args a) {
  constexpr int ST = 3, GB = kv4::group_bytes(HD);
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float all_lows[NW][2 * 8 * NT];
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  float* lows = all_lows[warp];
  const uint32_t ring = s_addr(smem) + warp * ST * 2 * GB, bars = s_addr(smem) + NW * ST * 2 * GB + warp * ST * 8;
  if (lane == 0)
    for (int s = 0; s < ST; ++s) mbar_init(bars + 8 * s, 1);
  asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  __syncwarp();
  pdl_launch_dependents();
  pdl_wait();
  const int b = blockIdx.y, kvh = blockIdx.x, G = a.H / a.KV;
  // the first units' block ids without a window come at the same time as the length that says which of them count
  int blk[ST];
#pragma unroll
  for (int s = 0; s < ST; ++s) {
    const int64_t at = ((int64_t)(warp + s * NW) * WK + lane * 16) >> a.bs_shift;
    blk[s] = lane < 2 && at < a.max_blocks && a.window == 0 ? a.table[(int64_t)b * a.max_blocks + at] : 0;
  }
  const int qrow = a.qsl[b];
  if (a.qsl[b + 1] - qrow != 1) return;
  const Span sp(a.len(b), a.window, a.first);
  const bool two = a.bs_shift == 4;
  auto block_of = [&](int u) {
    const int key = sp.key0(u) + lane * 16;
    return u < sp.n && lane < 2 && key < sp.len ? a.table[(int64_t)b * a.max_blocks + (key >> a.bs_shift)] : 0;
  };
  auto ask = [&](int u, int stage, int blk) {
    if (u >= sp.n) return;
    const int key0 = sp.key0(u), groups = min(2, (sp.len - key0 + 15) >> 4);
    if (lane == 0) mbar_expect(bars + 8 * stage, (uint32_t)(groups * GB));
    __syncwarp();
    if (lane < (two ? groups : min(groups, 1))) copy_groups<HD>(a, ring + (stage * 2 + lane) * GB, blk, kvh, key0 + lane * 16, two ? 1 : groups, bars + 8 * stage);
  };
  if (a.window)
#pragma unroll
    for (int s = 0; s < ST; ++s) blk[s] = block_of(warp + s * NW);
#pragma unroll
  for (int s = 0; s < ST; ++s) ask(warp + s * NW, s, blk[s]);
  Core<HD, NT> core;
  core.start(a.q + (int64_t)qrow * a.q_stride + kvh * G * HD, G, a.scale_log2, lane, lows);
  int stage = 0;
  uint32_t parity = 0;
  for (int u = warp; u < sp.n; u += NW) {
    const int key0 = sp.key0(u), next = block_of(u + ST * NW);
    mbar_wait(bars + 8 * stage, parity);
    if (sp.len > 0) core.unit(ring + stage * 2 * GB, lane, key0 + WK > sp.len || (key0 < sp.lo && key0 + WK > a.first), key0, sp.len, sp.lo, a.first, lows);
    __syncwarp();
    ask(u + ST * NW, stage, next);
    if (++stage == ST) { stage = 0; parity ^= 1; }
  }
  combine<HD, NT>(core, lows, reinterpret_cast<float*>(smem), warp, lane, G, [&](int r, int d, const Part& p, float4 v) {      // over the rings, which are read
    *reinterpret_cast<uint2*>(a.out + ((int64_t)qrow * a.H + kvh * G + r) * HD + d) = divided(v, p.l);
  });
}

// ---- long contexts: the units of all (request, kv head) groups, request-major, are one sequence, of which every CTA takes an equal share in a
// row.  A share covers the end of one group, whole groups and the start of another; whole groups go to the output, pieces to the workspace, and
// the kernel behind merges them.  A producer warp finds the share's pieces and runs ahead of the computing warps, into the next piece while
// they combine the last one's; what they need to know of a piece lies beside its query heads in shared memory.
template <int HD, int NT> __host__ __device__ constexpr int q_bytes() { return 2 * NT * 8 * HD * 2; }
template <int HD, int NT> __host__ __device__ constexpr int share_smem() {
  return stages(NT) * GROUPS * kv4::group_bytes(HD) + q_bytes<HD, NT>() + red_floats<HD>() * 4 + 2 * 48 + (2 * stages(NT) + 4) * 8;
}
struct __align__(16) Piece { int t0, t1, row, kvh; Span span; int slot; int pad[2]; };      // t0 == t1: no more; slot: of the workspace, -1: a whole group

template <int HD, int NT>
__global__ void __launch_bounds__(NW * 32 + 32, ctas_per_sm(NT)) attn_kv4_share_kernel(const Args a) {
  constexpr int GB = kv4::group_bytes(HD), ST = stages(NT), STAGE = GROUPS * GB;
  static_assert(sizeof(Piece) == 48, "as the launch counts");
  extern __shared__ __align__(128) uint8_t smem[];
  uint8_t* sq = smem + ST * STAGE;                       // query heads of a piece, two buffers
  float* red = reinterpret_cast<float*>(sq + q_bytes<HD, NT>());
  Piece* pieces = reinterpret_cast<Piece*>(red + red_floats<HD>());
  __shared__ float all_lows[NW][2 * 8 * NT];
  const int tid = threadIdx.x, warp = uniform_warp(), lane = tid & 31, G = a.H / a.KV;
  const uint32_t ring = s_addr(smem), bar0 = s_addr(pieces + 2);
  // full(s), p_full(i): the producer's arrival and its copies' bytes; empty(s), p_empty(i): the computing warps.  A wait for one comes before
  // what its next phase needs: a warp arrives on empty(s) only behind its wait for full(s), and the producer refills s only behind empty(s).
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (ST + s); };
  auto p_full = [&](int i) { return bar0 + 8u * (2 * ST + i); };
  auto p_empty = [&](int i) { return bar0 + 8u * (2 * ST + 2 + i); };
  if (tid == 0) {
    for (int s = 0; s < ST; ++s) { mbar_init(full(s), 1); mbar_init(empty(s), NW); }
    for (int i = 0; i < 2; ++i) { mbar_init(p_full(i), 1); mbar_init(p_empty(i), NW); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncthreads();
  pdl_launch_dependents();
  pdl_wait();
  int stage = 0, pi = 0;
  uint32_t parity = 0, p_parity = 0;

  if (warp == NW) {
    // ---- the producer: all units, then the request that holds this share's first
    auto units_of = [&](int b) { return a.qsl[b + 1] - a.qsl[b] == 1 ? (uint32_t)Span(a.len(b), a.window, a.first).n : 0u; };
    uint32_t sum = 0;
    for (int b = lane; b < a.B; b += 32) sum += units_of(b);
    const uint32_t U = __reduce_add_sync(0xffffffffu, sum) * a.KV, chunk = max((U + gridDim.x - 1) / gridDim.x, (uint32_t)NW), u0 = min(U, blockIdx.x * chunk);
    const uint32_t all = min(U, u0 + chunk) - u0;
    uint32_t left = all, before = 0;
    int b = 0, n = 0, kvh = 0, t0 = 0;                   // the current piece begins at unit t0 of the n of (b, kvh)
    for (int b0 = 0; left; b0 += 32) {
      const uint32_t mine = b0 + lane < a.B ? units_of(b0 + lane) : 0;
      uint32_t incl = mine * a.KV;
#pragma unroll
      for (int d = 1; d < 32; d <<= 1) { const uint32_t v = __shfl_up_sync(0xffffffffu, incl, d); if (lane >= d) incl += v; }
      const uint32_t past = __ballot_sync(0xffffffffu, before + incl > u0);
      if (past) {
        const int l = __ffs(past) - 1;
        b = b0 + l;
        n = (int)__shfl_sync(0xffffffffu, mine, l);
        before += __shfl_sync(0xffffffffu, incl, l) - n * a.KV;
        kvh = (int)((u0 - before) / n);
        t0 = (int)(u0 - before) - kvh * n;
        break;
      }
      before += __shfl_sync(0xffffffffu, incl, 31);
    }
    int4 desc = make_int4(-1, 0, 0, 0);
    // a lane per unit of a stage (two lanes where blocks have 16 tokens); the block ids of the next stage are read while this one is waited for
    const int unit = a.bs_shift == 4 ? lane >> 1 : lane, sub = a.bs_shift == 4 ? (lane & 1) * 16 : 0, box = a.bs_shift == 4 ? 16 : WK;
    bool refill = false, refill_p = false;
    while (left) {
      const int t1 = (int)min((uint32_t)n, t0 + left), row = a.qsl[b];
      const Span sp(a.len(b), a.window, a.first);
      int key = 0, groups = 0, blk = 0;                  // this lane's copy of the next stage
      auto look = [&](int u) {
        key = sp.key0(u + unit) + sub;
        groups = unit < NW && u + unit < t1 ? max(min(box, sp.len - key + 15), 0) >> 4 : 0;
        if (groups) blk = a.table[(int64_t)b * a.max_blocks + (key >> a.bs_shift)];
      };
      look(t0);
      if (refill_p) mbar_wait_idle(p_empty(pi), p_parity ^ 1);
      if (lane == 0) {
        Piece p;
        p.t0 = t0; p.t1 = t1; p.row = row; p.kvh = kvh; p.span = sp;
        p.slot = t0 == 0 && t1 == n ? -1 : 2 * (int)blockIdx.x + (t0 == 0);      // slot 0: the end or the middle of a group, slot 1: its start
        pieces[pi] = p;
        mbar_expect(p_full(pi), (uint32_t)(G * HD * 2));
        bulk_load(s_addr(sq) + pi * (q_bytes<HD, NT>() / 2), a.q + (int64_t)row * a.q_stride + kvh * G * HD, (uint32_t)(G * HD * 2), p_full(pi));
      }
      pi ^= 1;
      if (pi == 0) { p_parity ^= 1; refill_p = true; }
      if (t0 == 0 && t1 < n) desc = make_int4(row, kvh, (int)((u0 + all - 1 + n - t1) / chunk), 0);      // (the share's last piece)
      for (int u = t0; u < t1; u += NW) {
        const int now = groups, id = blk, at = key;
        const uint32_t bytes = __reduce_add_sync(0xffffffffu, (uint32_t)now) * GB;
        look(u + NW);
        if (refill) mbar_wait_idle(empty(stage), parity ^ 1);
        if (lane == 0) mbar_expect(full(stage), bytes);
        __syncwarp();
        if (now) copy_groups<HD>(a, ring + stage * STAGE + (unit * 2 + (sub >> 4)) * GB, id, kvh, at, now, full(stage));
        if (++stage == ST) { stage = 0; parity ^= 1; refill = true; }
      }
      left -= t1 - t0;
      t0 = 0;
      if (left && ++kvh == a.KV) {
        kvh = 0;
        do ++b; while ((n = (int)units_of(b)) == 0);
      }
    }
    if (refill_p) mbar_wait_idle(p_empty(pi), p_parity ^ 1);
    if (lane == 0) {
      pieces[pi].t0 = pieces[pi].t1 = 0;
      mbar_arrive(p_full(pi));
      a.desc[blockIdx.x] = desc;
    }
    return;
  }

  const uint32_t own = ring + warp * 2 * GB;
  float* lows = all_lows[warp];
  while (true) {
    mbar_wait(p_full(pi), p_parity);
    const Piece p = pieces[pi];
    if (p.t0 == p.t1) break;
    Core<HD, NT> core;
    core.start(reinterpret_cast<const bf16*>(sq + pi * (q_bytes<HD, NT>() / 2)), G, a.scale_log2, lane, lows);
    __syncwarp();
    if (lane == 0) mbar_arrive(p_empty(pi));
    pi ^= 1;
    if (pi == 0) p_parity ^= 1;
    for (int u = p.t0; u < p.t1; u += NW) {
      mbar_wait(full(stage), parity);
      if (u + warp < p.t1 && p.span.len > 0) {
        const int key0 = p.span.key0(u + warp);
        core.unit(own + stage * STAGE, lane, key0 + WK > p.span.len || (key0 < p.span.lo && key0 + WK > a.first), key0, p.span.len, p.span.lo, a.first, lows);
      }
      __syncwarp();                                      // the stage is read
      if (lane == 0) mbar_arrive(empty(stage));
      if (++stage == ST) { stage = 0; parity ^= 1; }
    }
    if (p.slot < 0) {
      combine<HD, NT>(core, lows, red, warp, lane, G, [&](int r, int d, const Part& all, float4 v) {
        *reinterpret_cast<uint2*>(a.out + ((int64_t)p.row * a.H + p.kvh * G + r) * HD + d) = divided(v, all.l);
      });
    } else {
      combine<HD, NT>(core, lows, red, warp, lane, G, [&](int r, int d, const Part& all, float4 v) {
        const int64_t at = (int64_t)p.slot * G + r;
        *reinterpret_cast<float4*>(a.part + at * HD + d) = v;
        if (d == 0) *reinterpret_cast<float4*>(a.part + (int64_t)2 * kMaxShares * G * HD + at * 4) = make_float4(all.x, all.m, all.l, 0.f);
      });
    }
  }
}

// Groups that were cut: warp (share, row) merges the pieces of the group that begins in the share, in the order of the shares; where there are
// many, the whole block does, piece i by warp i mod 8.
constexpr int MW = 8, kFewPieces = 12;
template <int HD>
__global__ void __launch_bounds__(MW * 32) attn_kv4_merge_kernel(bf16* __restrict__ out, const float* __restrict__ part, const int4* __restrict__ desc, int H, int G, int shares) {
  constexpr int C = HD / 4;                    // lanes of a row (the others of a warp idle along)
  __shared__ float4 sh[MW][C];
  __shared__ Part sp[MW];
  __shared__ int4 sd[MW];
  pdl_launch_dependents();
  pdl_wait();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, r = blockIdx.y, c = lane % C;
  const float4* ml = reinterpret_cast<const float4*>(part + (int64_t)2 * kMaxShares * G * HD);
  const int4 mine = blockIdx.x * MW + warp < shares ? desc[blockIdx.x * MW + warp] : make_int4(-1, 0, 0, 0);
  // pieces first .. n - 1 of the group of d that begins in share s, by steps
  auto merge = [&](int s, const int4& d, int first, int step, Part& all, float4& acc) {
    const int n = d.z - s + 1;
    constexpr int AT_ONCE = 8;
    for (int i0 = first; i0 < n; i0 += AT_ONCE * step) {
      Part p[AT_ONCE];
      float4 v[AT_ONCE];
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k) {
        const int i = min(i0 + k * step, n - 1);
        const int64_t row = (int64_t)(2 * (s + i) + (i == 0)) * G + r;      // slot 1 of the first share, slot 0 of the others
        const float4 u = ml[row];
        p[k] = {u.x, i0 + k * step < n ? u.y : -INFINITY, u.z};
        v[k] = *reinterpret_cast<const float4*>(part + row * HD + 4 * c);
      }
      const Part was = all;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (above(p[k], all)) all = p[k];
      const float old_half = half_of(was, all), old = old_half * old_half;
      acc.x *= old; acc.y *= old; acc.z *= old; acc.w *= old;
      all.l = was.l * old_half * old_half;
#pragma unroll
      for (int k = 0; k < AT_ONCE; ++k)
        if (i0 + k * step < n) {
          const float half = half_of(p[k], all), f = half * half;
          acc.x = fmaf(f, v[k].x, acc.x); acc.y = fmaf(f, v[k].y, acc.y); acc.z = fmaf(f, v[k].z, acc.z); acc.w = fmaf(f, v[k].w, acc.w);
          all.l = fmaf(half, half * p[k].l, all.l);
        }
    }
  };
  auto write = [&](const int4& d, float l, const float4& acc) {
    *reinterpret_cast<uint2*>(out + ((int64_t)d.x * H + d.y * G + r) * HD + 4 * c) = divided(acc, l);
  };
  const bool many = mine.x >= 0 && mine.z - (int)(blockIdx.x * MW + warp) >= kFewPieces;
  if (mine.x >= 0 && !many) {
    Part all = no_part();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    merge(blockIdx.x * MW + warp, mine, 0, 1, all, acc);
    if (lane < C) write(mine, all.l, acc);
  }
  if (!__syncthreads_or(many)) return;
  if (lane == 0) sd[warp] = many ? mine : make_int4(-1, 0, 0, 0);
  __syncthreads();
  for (int w = 0; w < MW; ++w) {
    const int4 d = sd[w];
    if (d.x < 0) continue;                     // (the same for the block)
    Part all = no_part();
    float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
    merge(blockIdx.x * MW + w, d, warp, MW, all, acc);
    if (lane < C) sh[warp][c] = acc;
    if (lane == 0) sp[warp] = all;
    __syncthreads();
    if (warp == 0) {
      all = no_part();
#pragma unroll
      for (int k = 0; k < MW; ++k)
        if (above(sp[k], all)) all = sp[k];
      acc = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll
      for (int k = 0; k < MW; ++k) {
        const float half = half_of(sp[k], all), f = half * half;
        const float4 v = sh[k][c];
        acc.x = fmaf(f, v.x, acc.x); acc.y = fmaf(f, v.y, acc.y); acc.z = fmaf(f, v.z, acc.z); acc.w = fmaf(f, v.w, acc.w);
        l = fmaf(half, half * sp[k].l, l);
      }
      if (lane < C) write(d, l, acc);
    }
    __syncthreads();
  }
}

constexpr int kDescBytes = kMaxShares * 16;    // the workspace's start
constexpr int64_t workspace_bytes(int G, int hd) { return kDescBytes + (int64_t)2 * kMaxShares * G * (hd + 4) * 4; }
constexpr int kMaxRequests = 1024;             // requests of one launch (every warp reads their lengths)

// Which kernel.  A CTA per (request, kv head) has four CTAs an SM (three for groups of 9 to 16), which cover each other's starts and ends, and the
// hardware's queue; shares have three (two), a producer and a merge behind them (4 us), but every SM has work whatever the lengths are.  us with a
// CTA each / with shares, 32 / 8 heads of 128:
//                             1024 keys     1500         2048         2900         4096         6000
//      8 requests (64 groups)  8.9 / 11.3  12.0 / 12.3  15.0 / 12.7  20.7 / 14.2  29.2 / 17.3  41.1 / 19.4
//     48 (384)                19.5 / 20.9  25.5 / 25.4  31.9 / 29.2  42.6 / 36.4  56.9 / 45.5  80.5 / 60.3
//     72 (576)                20.8 / 27.7  26.7 / 33.6  33.3 / 39.2  44.2 / 50.2  59.0 / 64.2  83.0 / 88.1
//    100 (800)                28.2 / 32.6  37.3 / 41.2  47.3 / 49.1  63.5 / 63.6  85.2 / 83.0   122 / 117
//    150 (1200)               38.8 / 44.6  52.3 / 56.7  67.0 / 69.2  90.8 / 90.7   123 / 122    179 / 173
//                   32 / 8 heads of 64                      128 / 8 heads of 128
//                   1024 keys    2048         4096          1024         2048         4096
//      8 (64)        7.4 /  9.8  12.2 / 10.7  22.0 / 13.0   14.4 / 20.1  23.1 / 22.0  42.7 / 27.4
//     48 (384)      15.0 / 15.9  26.0 / 22.3  46.5 / 34.2   25.0 / 37.9  40.0 / 50.6  68.9 / 77.4
//    100 (800)      21.2 / 25.0  34.5 / 36.7  61.6 / 60.5   46.3 / 58.3  74.9 / 84.7   132 / 138
// so: up to 1024 keys, or six groups for every 32 keys; and up to 8192 keys, since one long context among many short ones is a single CTA's
// work (0.35 us for 128 keys).  How evenly the groups fall on the SMs is not looked at: that gives up 9 % at 384 groups of 2048 keys (17 % with
// heads of 64) and at 576 of 4096, 6 % at 576 of 6000, 12 % at 384 groups of 16 heads and 4096 keys, and up to 4 % in other cells.
static bool cta_each(int64_t groups, int keys) {
  const int units = (keys + WK - 1) / WK;
  return units <= 32 || (units <= 256 && groups >= 6 * units);
}

template <int HD, int NT>
static int launch(const Args& a, int max_seq_len, cudaStream_t st) {
  // a window leaves its own keys (from inside a unit on) and the first ones
  const int keys = a.window > 0 ? (int)std::min<int64_t>(max_seq_len, (int64_t)a.window + a.first + 2 * WK) : max_seq_len;
  if (cta_each((int64_t)a.B * a.KV, keys)) {
    constexpr int ring = NW * 3 * 2 * kv4::group_bytes(HD) + NW * 3 * 8, smem = ring > red_floats<HD>() * 4 ? ring : red_floats<HD>() * 4;
    auto kern = attn_kv4_kernel<HD, NT>;
    if (smem > (int)kPlainShared) KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    KGE_CUDA_OK(launch_pdl(kern, dim3(a.KV, a.B), dim3(NW * 32), smem, st, a));
    return 0;
  }
  auto kern = attn_kv4_share_kernel<HD, NT>;
  const int G = a.H / a.KV, shares = shares_of(NT);
  KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, share_smem<HD, NT>()));
  KGE_CUDA_OK(launch_pdl(kern, dim3(shares), dim3(NW * 32 + 32), share_smem<HD, NT>(), st, a));
  KGE_CUDA_OK(launch_pdl(attn_kv4_merge_kernel<HD>, dim3((shares + MW - 1) / MW, G), dim3(MW * 32), 0, st, a.out, (const float*)a.part, (const int4*)a.desc, a.H, G, shares));
  return 0;
}

}  // namespace ak4

static int decode(ak4::Args a, int hd, int max_seq_len, cudaStream_t st) {
  const int B = a.B, G = a.H / a.KV;
  // requests of a launch: few enough to be read by every warp, and units that 32 bits count (a table's row bounds a request's)
  const int64_t tiles = ((((int64_t)a.max_blocks << a.bs_shift) + ak4::WK - 1) / ak4::WK + 1) * a.KV;
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
  KGE_REQUIRE(q_stride % 8 == 0 && q_stride >= (int64_t)H * hd, "kge_paged_attn_kv4: q_stride=%d must be a multiple of 8, at least H * hd", q_stride);
  KGE_REQUIRE((((uintptr_t)out | (uintptr_t)q | (uintptr_t)kv_cache | (uintptr_t)workspace) & 15) == 0, "kge_paged_attn_kv4: pointers must be 16-byte aligned");
  KGE_REQUIRE(window >= 0 && first >= 0, "kge_paged_attn_kv4: window=%d first=%d", window, first);
  KGE_REQUIRE(scale > 0.f && scale < 1e38f, "kge_paged_attn_kv4: scale=%g must be positive", (double)scale);
  if (B <= 0 || T <= 0) return 0;
  KGE_REQUIRE(B <= 65535, "kge_paged_attn_kv4: %d requests (at most 65535)", B);
  KGE_REQUIRE(max_q_len >= 1 && max_seq_len >= 1 && max_blocks_per_seq >= 1, "kge_paged_attn_kv4: max_q_len / max_seq_len / max_blocks_per_seq must be >= 1");
  KGE_REQUIRE((int64_t)max_blocks_per_seq * block_size <= (1ll << 30), "kge_paged_attn_kv4: %d blocks of %d tokens a request (at most 2^30 tokens)", max_blocks_per_seq,
              block_size);
  const int most = max_blocks_per_seq * block_size;      // keys of a request: what is beyond makes no difference, and sums stay in range
  if (window >= most) window = 0;
  first = std::min(first, most);
  max_seq_len = std::min(max_seq_len, most);
  cudaStream_t st = (cudaStream_t)stream;
  const int G = H / KV;
  const bool single = G <= 16;                 // a kernel of their own for single-token requests
  const int64_t need = single ? ak4::workspace_bytes(G, hd) : 0;
  KGE_REQUIRE(!single || (workspace && workspace_bytes >= need), "kge_paged_attn_kv4: workspace %lld < %lld bytes", (long long)workspace_bytes, (long long)need);
  if (!single || max_q_len > 1)
    if (int rc = paged_attn_kv4_tc((bf16*)out, (const bf16*)q, q_stride, (const uint8_t*)kv_cache, block_table, max_blocks_per_seq, seq_lens, query_start_loc, B, T, max_q_len,
                                   max_seq_len, H, KV, hd, block_size, scale, window, first, single, st))
      return rc;
  if (!single) return 0;
  ak4::Args a;
  a.out = (bf16*)out; a.q = (const bf16*)q; a.cache = (const uint8_t*)kv_cache;
  a.table = block_table; a.lens = seq_lens; a.qsl = query_start_loc;
  a.desc = (int4*)workspace; a.part = (float*)((uint8_t*)workspace + ak4::kDescBytes);
  a.q_stride = q_stride; a.max_blocks = max_blocks_per_seq; a.B = B; a.H = H; a.KV = KV;
  a.bs_shift = 4;
  while ((1 << a.bs_shift) < block_size) ++a.bs_shift;
  a.window = window; a.first = first; a.scale_log2 = scale * ak4::kLog2e;
  return decode(a, hd, max_seq_len, st);
}
