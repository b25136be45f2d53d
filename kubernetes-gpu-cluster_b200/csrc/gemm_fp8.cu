// Products of 8-bit codes with a scale for each block of 128 (fp8.cuh), dense and grouped by expert:
//   y[t, n] = sum_b xs[b, t] ws[n / 128, b] sum_{k in block b} x[t, k] w[n, k]  (+ bias[n])
//   h[t, j] = silu(gate) * up of such a pair of products, quantised row by row in blocks of 128 in the same kernel.
//
// Orientation: the MMA's M rows are TOKENS and its N columns weight rows, so that what a thread reads back of tensor memory (one lane) belongs to one
// token and, within 128 columns, to one scale of the weights: a single factor for all of them.  tcgen05.mma sums a block of K (four instructions of
// 32) in fp32 in tensor memory, and eight warps add it, times its factor, to accumulators in registers: TM += factor * D, two numbers an
// instruction.  Tensor memory holds several blocks, so that the next ones are multiplied meanwhile.
//
// Two kernels.
//  fp8_stream_kernel: tiles of 128 tokens x NT weight rows by single CTAs, one an SM; the (tile, block of K) units of the whole problem are laid end
//    to end and cut into equal shares, so every SM reads the same number of weight bytes whatever the sizes are.  A tile that a share's end cuts is
//    summed by the last of its CTAs to arrive, from fp32 partial sums in the workspace and in the order of K: the same bits each time.
//  fp8_pair_kernel: tiles of 256 x 256 by pairs of CTAs (cta_group::2), for many tokens: a CTA has its own 128 tokens and half of the weight rows in
//    shared memory, 32 KB a block of K, where its MMA takes 512 cycles.
#include <cuda.h>

#include "f32x2.cuh"
#include "fp8.cuh"
#include "kge.h"

namespace kge {
inline namespace KGE_ELT_NS {

constexpr int kRows = 128;                        // tokens of a CTA's tile
constexpr int kSlab = 128 * 128;                  // bytes of 128 rows of a block of K
constexpr int kThreads = 384;                     // producer, MMA, tensor memory, table; eight warps that add up
constexpr int kCounters = 256;                    // arrival counters at the head of the workspace
constexpr int kMaxCtas = 160;
constexpr int kMaxGroups = 1024;
constexpr int kSmem = 226 * 1024;
constexpr int kPairStages = 6;
constexpr int kPairBand = 8;                      // 74 pairs at work: 8 x 9 tiles share 17 slabs a block of K, 32 x 2.3 would 34

struct Fp8Params {
  bf16* y;                                        // plain: [T, N]
  const bf16* bias;
  uint8_t* codes;                                 // gated: [T, N] codes, N = f
  float* out_scales;                              //        [N / 128][out_stride]
  int64_t out_stride;
  const float* xs;                                // [block of K][xs_stride]
  int64_t xs_stride;
  const float* ws;                                // [group][blocks of the weight rows][blocks of K]
  const int32_t* offsets;                         // grouped: rows of group e are offsets[e] .. offsets[e + 1]
  int E, T, N, KB, n_tiles, w_rows, w_blocks;     // w_rows, w_blocks: of one group's matrix (2 N when gated)
  float* part;                                    // stream: partial sums
  unsigned int* count;
  int quarters, stages, x_bytes, min_units;       // stream: 32-row quarters that a tile can have, stages, bytes of a stage's tokens, least units of a share
};

__device__ __forceinline__ uint32_t s_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) { asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void load_box2(uint32_t dst, const CUtensorMap* map, uint32_t bar_of_leader, int c0, int c1) {
  asm volatile("cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
               ::"r"(dst), "l"(map), "r"(bar_of_leader), "r"(c0), "r"(c1) : "memory");
}
__device__ __forceinline__ void fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void commit2(uint32_t bar, uint16_t mask) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"(mask) : "memory");
}
__device__ __forceinline__ void mma8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
__device__ __forceinline__ void mma8x2(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t add) {
  asm volatile("{\n.reg .pred p;\nsetp.ne.b32 p, %4, 0;\ntcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n}" ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(add) : "memory");
}
// 32 columns of this warp's 32 lanes; the caller waits (tmem_wait_ld)
__device__ __forceinline__ void tmem_ld32(uint32_t at, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                 "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                 "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
               : "r"(at));
}
// K-major tile of 128-byte rows with 128-byte swizzle, atoms of 8 rows 1024 bytes apart
__device__ __forceinline__ uint64_t tile_desc(uint32_t at) {
  return (uint64_t)((at & 0x3ffffu) >> 4) | (uint64_t)1 << 16 | (uint64_t)(1024 >> 4) << 32 | (uint64_t)1 << 46 | (uint64_t)2 << 61;
}
// kind::f8f6f4 with e4m3 operands and fp32 sums
__host__ __device__ constexpr uint32_t instr_desc(int m, int n) { return (1u << 4) | (uint32_t)(n >> 3) << 17 | (uint32_t)(m >> 4) << 24; }

template <int REGS> __device__ __forceinline__ void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS)); }
template <int REGS> __device__ __forceinline__ void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS)); }
__device__ __forceinline__ void sums_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Rows of group e, whatever the table holds.
__device__ __forceinline__ void group_rows(const Fp8Params& p, int e, int& r0, int& r1) {
  if (!p.offsets) { r0 = 0; r1 = p.T; return; }
  r0 = min(max(p.offsets[e], 0), p.T);
  r1 = max(r0, min(p.offsets[e + 1], p.T));
}
// One warp: starts[e] = tiles of the groups before e.
__device__ __forceinline__ void count_tiles(const Fp8Params& p, int tile_rows, int* starts, int lane) {
  int total = 0;
  for (int e0 = 0; e0 < p.E; e0 += 32) {
    int n = 0;
    if (e0 + lane < p.E) {
      int r0, r1;
      group_rows(p, e0 + lane, r0, r1);
      n = (r1 - r0 + tile_rows - 1) / tile_rows * p.n_tiles;
    }
    int s = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, s, o); if (lane >= o) s += v; }
    if (e0 + lane < p.E) starts[e0 + lane] = total + s - n;
    total += __shfl_sync(0xffffffffu, s, 31);
  }
  if (lane == 0) starts[p.E] = total;
}

// A tile: rows [row, row + rows) of the tokens and column tile n of group e.
struct Tile { int e, n, row, rows; };
// From a tile's number; the group is looked for from `e` on (numbers come in rising order).  Tiles of a group run over BAND token tiles (0: all), then
// the next column tile: neighbours share weights, and a band's tokens stay in the L2 meanwhile.
template <int TILE_ROWS, int BAND>
__device__ __forceinline__ Tile find_tile(const Fp8Params& p, const int* starts, int tile, int& e) {
  while (e + 1 < p.E && tile >= starts[e + 1]) ++e;
  int r0, r1;
  group_rows(p, e, r0, r1);
  const int m_tiles = (r1 - r0 + TILE_ROWS - 1) / TILE_ROWS, local = tile - starts[e], band = BAND ? BAND : m_tiles;
  const int g = local / (band * p.n_tiles), first = g * band, width = min(band, m_tiles - first), in = local - g * band * p.n_tiles;
  Tile t;
  t.e = e;
  t.n = in / width;
  t.row = r0 + (first + in - t.n * width) * TILE_ROWS;
  t.rows = min(TILE_ROWS, r1 - t.row);
  return t;
}
__device__ __forceinline__ int first_group(const Fp8Params& p, const int* starts, int tile) {
  int lo = 0, hi = p.E - 1;
  while (lo < hi) { const int mid = (lo + hi + 1) / 2; if (starts[mid] <= tile) lo = mid; else hi = mid - 1; }
  return lo;
}

// The running sums of a thread: one token, C columns.
template <int C>
struct Sums {
  f2 v[C / 2];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < C / 2; ++i) v[i] = 0ull;
  }
  // += factor * D of 32 columns at c
  __device__ __forceinline__ void add(int c, const uint32_t (&r)[32], float factor) {
    const f2 s = pk(factor, factor);
#pragma unroll
    for (int i = 0; i < 16; ++i) v[c / 2 + i] = fma2(pk(__uint_as_float(r[2 * i]), __uint_as_float(r[2 * i + 1])), s, v[c / 2 + i]);
  }
  __device__ __forceinline__ void at(int c, float& a, float& b) const { upk(v[c / 2], a, b); }
};

// A block of K, at tensor memory address `at`: columns below C / 2 times f0, the others times f1 (the same but for gate and up).
template <int C>
__device__ __forceinline__ void add_block(Sums<C>& s, uint32_t at, float f0, float f1) {
  uint32_t r[2][32];
  tmem_ld32(at, r[0]);
#pragma unroll
  for (int c = 0; c < C; c += 32) {
    tmem_wait_ld(r[(c / 32) & 1]);
    if (c + 32 < C) tmem_ld32(at + c + 32, r[(c / 32 + 1) & 1]);
    s.add(c, r[(c / 32) & 1], c < C / 2 ? f0 : f1);
  }
}

// Factors of the blocks of K for a thread's token and its columns, asked for three blocks ahead.
template <bool GATED>
struct Factors {
  const float *xs, *w0, *w1;
  int64_t stride;
  int kb, end;
  float x[3], a[3], b[3];
  __device__ __forceinline__ void ask(int i) {
    const bool in = kb < end;
    x[i] = xs && in ? __ldg(xs) : 0.f;
    a[i] = in ? __ldg(w0 + kb) : 0.f;
    if (GATED) b[i] = in ? __ldg(w1 + kb) : 0.f;
    if (xs) xs += stride;
    ++kb;
  }
  __device__ __forceinline__ void start(const Fp8Params& p, int row, bool there, int64_t block0, int64_t block1, int kb0, int kb1) {
    stride = p.xs_stride;
    xs = there ? p.xs + kb0 * stride + row : nullptr;
    w0 = p.ws + block0 * p.KB;
    w1 = p.ws + block1 * p.KB;
    kb = kb0; end = kb1;
#pragma unroll
    for (int i = 0; i < 3; ++i) ask(i);
  }
  __device__ __forceinline__ void next(float& f0, float& f1) {
    f0 = x[0] * a[0];
    f1 = GATED ? x[0] * b[0] : f0;
    x[0] = x[1]; x[1] = x[2]; a[0] = a[1]; a[1] = a[2];
    if (GATED) { b[0] = b[1]; b[1] = b[2]; }
    ask(2);
  }
};

// One row's C columns from n0 on, rounded once.
template <int C>
__device__ __forceinline__ void store_row(const Fp8Params& p, const Sums<C>& s, int row, int n0) {
  bf16* dst = p.y + (int64_t)row * p.N + n0;
  if (n0 + C <= p.N && (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0) {
#pragma unroll
    for (int c = 0; c < C; c += 8) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b;
        s.at(c + 2 * i, a, b);
        if (p.bias) { a += bf2f(p.bias[n0 + c + 2 * i]); b += bf2f(p.bias[n0 + c + 2 * i + 1]); }
        u[i] = pack_bf2(a, b);
      }
      *reinterpret_cast<uint4*>(dst + c) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < C; c += 2) {
      float a, b;
      s.at(c, a, b);
      if (n0 + c < p.N) dst[c] = f2bf(p.bias ? a + bf2f(p.bias[n0 + c]) : a);
      if (n0 + c + 1 < p.N) dst[c + 1] = f2bf(p.bias ? b + bf2f(p.bias[n0 + c + 1]) : b);
    }
  }
}

// Gated: a thread has 64 columns of the gate and the same 64 of up, its counterpart in the other warpgroup the block's other 64.  The block's largest
// magnitude goes through shared memory (two rows of 128 words).  Called by all 256 threads.
__device__ __forceinline__ void store_gated(const Fp8Params& p, const Sums<128>& s, int row, bool there, int n, uint32_t* both, int half, int lane128) {
  float h[64];
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < 64; c += 2) {
    float g[2], u[2];
    s.at(c, g[0], g[1]);
    s.at(64 + c, u[0], u[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      h[c + i] = __fdividef(g[i], 1.f + __expf(-g[i])) * u[i];
      m = max(m, __float_as_uint(h[c + i]) & 0x7fffffffu);       // (NaN above all)
    }
  }
  both[half * 128 + lane128] = m;
  sums_sync();
  m = max(m, both[(half ^ 1) * 128 + lane128]);
  sums_sync();                                                   // (the next tile writes there)
  if (!there) return;
  float scale, factor;
  fp8::scale_of(__uint_as_float(m), scale, factor);
  uint8_t* dst = p.codes + (int64_t)row * p.N + n * 128 + half * 64;
#pragma unroll
  for (int c = 0; c < 64; c += 16) {
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q[i] = factor > 0.f ? fp8::pack4(h[c + 4 * i] * factor, h[c + 4 * i + 1] * factor, h[c + 4 * i + 2] * factor, h[c + 4 * i + 3] * factor) : 0u;
    *reinterpret_cast<uint4*>(dst + c) = make_uint4(q[0], q[1], q[2], q[3]);
  }
  if (half == 0) p.out_scales[n * p.out_stride + row] = scale;
}

// ----------------------------------------------------------------------------------------------------- equal shares of all units

// A share as pieces of tiles: blocks of K [kb0, kb1) of tile `tile`.
struct Pieces {
  int64_t cur, end;
  int KB;
  __device__ __forceinline__ bool next(int& tile, int& kb0, int& kb1) {
    if (cur >= end) return false;
    tile = (int)(cur / KB);
    kb0 = (int)(cur - (int64_t)tile * KB);
    const int64_t left = end - cur;
    kb1 = left < KB - kb0 ? kb0 + (int)left : KB;
    cur += kb1 - kb0;
    return true;
  }
};

template <int NT, bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
fp8_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Fp8Params p) {
  constexpr int C = NT / 2, BUFS = 512 / NT;
  static_assert(!GATED || NT == 256, "a gated tile holds 128 columns of each");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * 32 + 2 * BUFS];
  __shared__ uint32_t tmem_slot;
  __shared__ int last_flag;
  __shared__ uint32_t both[256];
  __shared__ int starts[kMaxGroups + 1];
  const int stages = p.stages;
  const uint32_t stage_bytes = (uint32_t)p.x_bytes + NT * 128;
  const uint32_t base = s_addr(smem), bar0 = s_addr(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (32 + s); };
  auto tfull = [&](int b) { return bar0 + 8u * (64 + b); };
  auto tempty = [&](int b) { return bar0 + 8u * (64 + BUFS + b); };
  const int warp = uniform_warp(), lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < stages; ++s) { bar_init(full(s), 1); bar_init(empty(s), 1); }
    for (int b = 0; b < BUFS; ++b) { bar_init(tfull(b), 1); bar_init(tempty(b), 8); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (warp == 3 && !p.offsets) count_tiles(p, kRows, starts, lane);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_launch_dependents();
  if (p.offsets) {                                  // which tiles there are is the kernel before's output
    pdl_wait();
    if (warp == 3) count_tiles(p, kRows, starts, lane);
    __syncthreads();
  }
  const int KB = p.KB;
  const int64_t U = (int64_t)starts[p.E] * KB;
  const int64_t G = max((int64_t)1, min((int64_t)gridDim.x, U / p.min_units)), me = blockIdx.x;
  const int64_t u0 = me < G ? U * me / G : U, u1 = me < G ? U * (me + 1) / G : U;
  const int e_first = u0 < u1 ? first_group(p, starts, (int)(u0 / KB)) : 0;

  if (warp == 0) {
    regs_down<72>();
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      auto load_w = [&](int s, const Tile& t, int kb) {
        const uint32_t dst = base + s * stage_bytes + p.x_bytes;
        const int row = t.e * p.w_rows;
        if (GATED) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            load_box(dst + h * kSlab, &map_w, full(s), kb * 128, row + t.n * 128 + h * 64);
            load_box(dst + h * kSlab + kSlab / 2, &map_w, full(s), kb * 128, row + p.N + t.n * 128 + h * 64);
          }
        } else {
#pragma unroll
          for (int h = 0; h < NT / 128; ++h) load_box(dst + h * kSlab, &map_w, full(s), kb * 128, row + t.n * NT + h * 128);
        }
      };
      auto load_x = [&](int s, const Tile& t, int kb) {
        for (int r = 0; r < t.rows; r += 32) load_box(base + s * stage_bytes + r * 128, &map_x, full(s), kb * 128, t.row + r);
      };
      auto bytes_of = [&](const Tile& t) { return (uint32_t)(NT * 128 + (t.rows + 31) / 32 * 4096); };
      // What the weights are is known before the kernel before has ended: its first tile's, as many as there are stages.
      int tile, kb0, kb1, ahead = 0, e = e_first;
      if (!p.offsets) {
        Pieces it{u0, u1, KB};
        if (it.next(tile, kb0, kb1)) {
          const Tile t = find_tile<kRows, 0>(p, starts, tile, e);
          ahead = min(stages, kb1 - kb0);
          for (int i = 0; i < ahead; ++i) { bar_expect(full(i), bytes_of(t)); load_w(i, t, kb0 + i); }
        }
        pdl_wait();
      }
      Pieces it{u0, u1, KB};
      while (it.next(tile, kb0, kb1)) {
        const Tile t = find_tile<kRows, 0>(p, starts, tile, e);
        for (int kb = kb0; kb < kb1; ++kb) {
          if (ahead > 0) {
            --ahead;
          } else {
            mbar_wait(empty(stage), phase ^ 1);
            bar_expect(full(stage), bytes_of(t));
            load_w(stage, t, kb);
          }
          load_x(stage, t, kb);
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    regs_down<72>();
    if (elect_one()) {
      constexpr uint32_t idesc = instr_desc(kRows, NT);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      const uint64_t a0 = tile_desc(base), b0 = tile_desc(base + p.x_bytes);
      uint64_t a = a0, b = b0;
      for (int64_t u = u0; u < u1; ++u) {
        mbar_wait(tempty(buf), buf_phase ^ 1);
        mbar_wait(full(stage), phase);
        fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k) mma8(tmem + buf * NT, a + 2 * k, b + 2 * k, idesc, k > 0);
        commit(empty(stage));
        commit(tfull(buf));
        a += stage_bytes >> 4; b += stage_bytes >> 4;
        if (++stage == stages) { stage = 0; phase ^= 1; a = a0; b = b0; }
        if (++buf == BUFS) { buf = 0; buf_phase ^= 1; }
      }
    }
  } else if (warp < 4) {
    regs_down<72>();
  } else {
    regs_up<216>();
    const int q = warp & 3, half = (warp - 4) >> 2, tid = threadIdx.x - 128, lane128 = q * 32 + lane;
    pdl_wait();
    int buf = 0, tile, kb0, kb1, e = e_first;
    uint32_t buf_phase = 0;
    Pieces it{u0, u1, KB};
    while (it.next(tile, kb0, kb1)) {
      const Tile t = find_tile<kRows, 0>(p, starts, tile, e);
      const bool some = q * 32 < t.rows, there = lane128 < t.rows;
      const int row = t.row + lane128, n0 = t.n * NT + half * C;
      const int64_t wb = (int64_t)t.e * p.w_blocks;
      Sums<C> s;
      s.clear();
      Factors<GATED> f;
      f.start(p, row, there, wb + (GATED ? t.n : min(n0 / 128, p.w_blocks - 1)), wb + (GATED ? p.N / 128 + t.n : 0), kb0, kb1);
      const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + half * C;
      for (int kb = kb0; kb < kb1; ++kb) {
        float f0, f1;
        f.next(f0, f1);
        mbar_wait(tfull(buf), buf_phase);
        if (some) {
          fence_after();
          add_block<C>(s, at + buf * NT, f0, f1);
          fence_before();
        }
        __syncwarp();
        if (lane == 0) bar_arrive(tempty(buf));
        if (++buf == BUFS) { buf = 0; buf_phase ^= 1; }
      }
      if (kb1 - kb0 != KB) {
        // A part of the tile's sum: to the workspace, [slot][quarter][half][column / 4][lane] of 16 bytes.  A share has at most two such pieces: slot 0
        // the one that it begins with.
        constexpr int kPer = 2 * (C / 4) * 32;          // float4 of a quarter
        const int64_t x0 = (int64_t)tile * KB;
        auto slot_of = [&](int64_t cta, int slot) { return reinterpret_cast<float4*>(p.part) + ((cta * 2 + slot) * p.quarters + q) * kPer + half * (C / 4) * 32 + lane; };
        if (some) {
          float4* dst = slot_of(me, x0 + kb0 == u0 ? 0 : 1);
#pragma unroll
          for (int c = 0; c < C; c += 4) {
            float4 v;
            s.at(c, v.x, v.y);
            s.at(c + 2, v.z, v.w);
            __stcg(dst + c / 4 * 32, v);
          }
        }
        __threadfence();
        sums_sync();
        // its CTAs: from the one with its first unit to the one with its last; they count in the first one's counter
        const int64_t c0 = ((x0 + 1) * G + U - 1) / U - 1, c1 = ((x0 + KB) * G + U - 1) / U - 1;
        if (tid == 0) {
          const bool mine = atomicAdd(p.count + c0, 1u) == (unsigned)(c1 - c0);
          if (mine) p.count[c0] = 0;                    // ready for the next launch
          last_flag = mine;
        }
        sums_sync();
        const bool last = last_flag != 0;
        sums_sync();                                    // (the next piece writes there)
        if (!last) continue;
        __threadfence();
        s.clear();
        if (some)
          for (int64_t c = c0; c <= c1; ++c) {
            const float4* src = slot_of(c, U * c / G >= x0 ? 0 : 1);
#pragma unroll
            for (int i = 0; i < C / 4; ++i) {
              const float4 v = __ldcg(src + i * 32);
              s.v[2 * i] = add2(s.v[2 * i], pk(v.x, v.y));
              s.v[2 * i + 1] = add2(s.v[2 * i + 1], pk(v.z, v.w));
            }
          }
      }
      if constexpr (GATED) store_gated(p, s, row, there, t.n, both, half, lane128);
      else if (there) store_row<C>(p, s, row, n0);
    }
  }
  fence_before();
  __syncthreads();
  if (warp == 2) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
}

// -------------------------------------------------------------------------------------------------------------- pairs

template <bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Fp8Params p) {
  constexpr int C = 128, STAGES = kPairStages;
  constexpr uint32_t kStage = 2 * kSlab;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * STAGES + 4];
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t both[256];
  __shared__ int starts[kMaxGroups + 1];
  const uint32_t base = s_addr(smem), bar0 = s_addr(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tfull = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto tempty = [&](int b) { return bar0 + 8u * (2 * STAGES + 2 + b); };
  const int warp = uniform_warp(), lane = threadIdx.x & 31, rank = (int)cluster_ctarank();

  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) { bar_init(full(s), 1); bar_init(empty(s), 1); }
    for (int b = 0; b < 2; ++b) { bar_init(tfull(b), 1); bar_init(tempty(b), 16); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (warp == 3 && !p.offsets) count_tiles(p, 2 * kRows, starts, lane);
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_launch_dependents();
  cluster_arrive(); cluster_wait();                 // the peer's barriers are there
  pdl_wait();
  if (p.offsets) {
    if (warp == 3) count_tiles(p, 2 * kRows, starts, lane);
    __syncthreads();
  }
  const int KB = p.KB, total = starts[p.E], first = (int)blockIdx.x >> 1, step = (int)gridDim.x >> 1;
  const int e_first = first < total ? first_group(p, starts, first) : 0;

  if (warp == 0) {
    regs_down<72>();
    if (elect_one()) {
      int stage = 0, e = e_first;
      uint32_t phase = 0;
      const uint32_t lead0 = mapa_u32(full(0), 0);
      for (int w = first; w < total; w += step) {
        const Tile t = find_tile<2 * kRows, kPairBand>(p, starts, w, e);
        const int wr = t.e * p.w_rows + (GATED ? t.n * 128 + rank * 64 : t.n * 256 + rank * 128), xr = t.row + rank * kRows;
        for (int kb = 0; kb < KB; ++kb) {
          mbar_wait(empty(stage), phase ^ 1);
          if (rank == 0) bar_expect(full(stage), 2 * kStage);
          const uint32_t dst = base + stage * kStage, lead = lead0 + 8u * stage;
          load_box2(dst, &map_x, lead, kb * 128, xr);
          if (GATED) {
            load_box2(dst + kSlab, &map_w, lead, kb * 128, wr);
            load_box2(dst + kSlab + kSlab / 2, &map_w, lead, kb * 128, wr + p.N);
          } else {
            load_box2(dst + kSlab, &map_w, lead, kb * 128, wr);
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    regs_down<72>();
    if (rank == 0 && elect_one()) {                 // the leader issues for both
      constexpr uint32_t idesc = instr_desc(2 * kRows, 256);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      const uint64_t a0 = tile_desc(base), b0 = tile_desc(base + kSlab);
      uint64_t a = a0, b = b0;
      for (int w = first; w < total; w += step)
        for (int kb = 0; kb < KB; ++kb) {
          mbar_wait(tempty(buf), buf_phase ^ 1);
          mbar_wait(full(stage), phase);
          fence_after();
#pragma unroll
          for (int k = 0; k < 4; ++k) mma8x2(tmem + buf * 256, a + 2 * k, b + 2 * k, idesc, k > 0);
          commit2(empty(stage), 3);
          commit2(tfull(buf), 3);
          a += kStage >> 4; b += kStage >> 4;
          if (++stage == STAGES) { stage = 0; phase ^= 1; a = a0; b = b0; }
          if (++buf == 2) { buf = 0; buf_phase ^= 1; }
        }
    }
  } else if (warp < 4) {
    regs_down<72>();
  } else {
    regs_up<216>();
    const int q = warp & 3, half = (warp - 4) >> 2, lane128 = q * 32 + lane;
    const uint32_t lead_tempty = mapa_u32(tempty(0), 0);
    int buf = 0, e = e_first;
    uint32_t buf_phase = 0;
    for (int w = first; w < total; w += step) {
      const Tile t = find_tile<2 * kRows, kPairBand>(p, starts, w, e);
      const int mine = rank * kRows + lane128;
      const bool some = rank * kRows + q * 32 < t.rows, there = mine < t.rows;
      const int row = t.row + mine, n0 = t.n * 256 + half * C;
      const int64_t wb = (int64_t)t.e * p.w_blocks;
      Sums<C> s;
      s.clear();
      Factors<GATED> f;
      f.start(p, row, there, wb + (GATED ? t.n : min(n0 / 128, p.w_blocks - 1)), wb + (GATED ? p.N / 128 + t.n : 0), 0, KB);
      const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + half * C;
      for (int kb = 0; kb < KB; ++kb) {
        float f0, f1;
        f.next(f0, f1);
        mbar_wait(tfull(buf), buf_phase);
        if (some) {
          fence_after();
          add_block<C>(s, at + buf * 256, f0, f1);
          fence_before();
        }
        __syncwarp();
        if (lane == 0) bar_arrive_cluster(lead_tempty + 8u * buf);
        if (++buf == 2) { buf = 0; buf_phase ^= 1; }
      }
      if constexpr (GATED) store_gated(p, s, row, there, t.n, both, half, lane128);
      else if (there) store_row<C>(p, s, row, n0);
    }
  }
  fence_before();
  cluster_arrive(); cluster_wait();                 // the leader's MMAs and the peer's arrivals are done
  if (warp == 2) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
}

// --------------------------------------------------------------------------------------------------------------- host

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// [rows, cols] bytes, boxes of 128 columns x box_rows
static int encode_map(CUtensorMap* m, const void* ptr, int64_t rows, int64_t cols, int box_rows) {
  static const EncodeFn enc = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    const bool ok = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &found) == cudaSuccess && found == cudaDriverEntryPointSuccess;
    return ok ? reinterpret_cast<EncodeFn>(f) : nullptr;
  }();
  KGE_REQUIRE(enc, "cuTensorMapEncodeTiled unavailable (no CUDA driver?)");
  cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)cols};
  cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUresult r = enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  KGE_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (%d) rows=%lld cols=%lld", (int)r, (long long)rows, (long long)cols);
  return 0;
}

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n < kMaxCtas ? n : kMaxCtas;
}

template <int NT, bool GATED>
static int launch_stream(Fp8Params& p, const void* x, const void* w, int K, cudaStream_t st) {
  constexpr int box = GATED ? 64 : 128;
  const int widest = p.T < kRows ? p.T : kRows;
  p.quarters = (widest + 31) / 32;
  p.x_bytes = p.quarters * 4096;
  p.n_tiles = (p.N + (GATED ? 128 : NT) - 1) / (GATED ? 128 : NT);
  constexpr int own = 8 * 1024;                            // the kernel's own shared memory, and rounding up to 1024
  p.stages = (kSmem - own) / (p.x_bytes + NT * 128);
  if (p.stages > 16) p.stages = 16;
  p.min_units = 2;
  // an MMA reads 128 rows of tokens from where they begin, and finds others' bytes behind the last: never beyond the stage's weights
  static_assert(NT * 128 >= kRows * 128, "");
  const int smem = p.stages * (p.x_bytes + NT * 128) + 1024;
  CUtensorMap mw, mx;
  if (int rc = encode_map(&mw, w, (int64_t)p.E * p.w_rows, K, box)) return rc;
  if (int rc = encode_map(&mx, x, p.T, K, 32)) return rc;
  auto kern = fp8_stream_kernel<NT, GATED>;
  KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int sms = sm_count();
  KGE_REQUIRE(sms > 0, "kge_gemm_fp8: no CUDA device");
  int64_t ctas = sms;
  if (!p.offsets) {
    const int64_t units = (int64_t)((p.T + kRows - 1) / kRows) * p.n_tiles * p.KB / p.min_units;
    ctas = units < 1 ? 1 : units < ctas ? units : ctas;
  }
  KGE_CUDA_OK(launch_pdl(kern, dim3((unsigned)ctas), dim3(kThreads), (size_t)smem, st, mw, mx, p));
  return 0;
}

template <bool GATED>
static int launch_pairs(Fp8Params& p, const void* x, const void* w, int K, cudaStream_t st) {
  p.n_tiles = (p.N + (GATED ? 128 : 256) - 1) / (GATED ? 128 : 256);
  const int smem = kPairStages * 2 * kSlab + 1024;
  CUtensorMap mw, mx;
  if (int rc = encode_map(&mw, w, (int64_t)p.E * p.w_rows, K, GATED ? 64 : 128)) return rc;
  if (int rc = encode_map(&mx, x, p.T, K, 128)) return rc;
  auto kern = fp8_pair_kernel<GATED>;
  KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  prefer_max_shared(kern);
  const int sms = sm_count();
  KGE_REQUIRE(sms > 1, "kge_gemm_fp8: no CUDA device");
  int64_t pairs = sms / 2;
  if (!p.offsets) {
    const int64_t tiles = (int64_t)((p.T + 2 * kRows - 1) / (2 * kRows)) * p.n_tiles;
    if (tiles < pairs) pairs = tiles;
  }
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(2 * pairs)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr; cfg.numAttrs = pdl_for_this_launch() ? 2 : 1;
  KGE_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, mw, mx, p));
  return 0;
}

static int64_t workspace_bytes_of(int T) {
  if (T <= 0) return 0;
  const int64_t quarters = ((T < kRows ? T : kRows) + 31) / 32;
  return kCounters * 4 + (int64_t)kMaxCtas * 2 * quarters * 256 * 128;
}

static bool aligned_to(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

// What all four have in common; N: columns of the result.
static int gemm_fp8(const char* name, Fp8Params& p, bool gated, const void* x, int x_scales_stride, const void* w, int K, void* workspace, int64_t workspace_bytes, cudaStream_t st) {
  KGE_REQUIRE(x && p.xs && w && p.ws && (gated ? p.codes && p.out_scales : p.y != nullptr), "%s: null pointer", name);
  KGE_REQUIRE(p.T >= 0 && p.N > 0 && K > 0 && K % 16 == 0, "%s: K=%d must be a positive multiple of 16, N=%d and T=%d not negative", name, K, p.N, p.T);
  KGE_REQUIRE(!gated || p.N % 128 == 0, "%s: f=%d must be a multiple of 128", name, p.N);
  KGE_REQUIRE(p.E > 0 && p.E <= kMaxGroups, "%s: %d groups (1 to %d)", name, p.E, kMaxGroups);
  const int64_t rows = (int64_t)p.N * (gated ? 2 : 1);
  KGE_REQUIRE(rows * p.E < (1ll << 31) - 256 && (int64_t)p.T + 2 * kRows < (1ll << 31), "%s: %d groups of %lld weight rows, %d rows of x", name, p.E, (long long)rows, p.T);
  KGE_REQUIRE(x_scales_stride >= p.T && (!gated || p.out_stride >= p.T), "%s: scales less than %d apart", name, p.T);
  KGE_REQUIRE(aligned_to(x, 16) && aligned_to(w, 16) && (!gated || aligned_to(p.codes, 16)), "%s: x, w and codes must be 16-byte aligned", name);
  KGE_REQUIRE(aligned_to(p.xs, 4) && aligned_to(p.ws, 4) && aligned_to(p.out_scales, 4) && aligned_to(p.y, 2) && aligned_to(p.bias, 2) && aligned_to(p.offsets, 4),
              "%s: a pointer is not aligned to its type", name);
  if (p.T == 0) return 0;
  p.xs_stride = x_scales_stride;
  p.KB = (int)fp8::blocks(K);
  p.w_rows = (int)rows;
  p.w_blocks = (int)fp8::blocks(rows);
  const int64_t tiles = ((int64_t)p.T / kRows + p.E) * p.w_blocks;
  KGE_REQUIRE(tiles < (1ll << 31), "%s: %lld tiles in one call", name, (long long)tiles);
  KGE_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(p.T) && aligned_to(workspace, 16), "%s: needs a workspace of %lld bytes, 16-byte aligned", name,
              (long long)workspace_bytes_of(p.T));
  p.count = (unsigned int*)workspace;
  p.part = (float*)((uint8_t*)workspace + kCounters * 4);
  const bool pairs = p.T / p.E > 256;
#ifndef KGE_HALF
  if (gated) return pairs ? launch_pairs<true>(p, x, w, K, st) : launch_stream<256, true>(p, x, w, K, st);
#endif
  return pairs ? launch_pairs<false>(p, x, w, K, st) : launch_stream<128, false>(p, x, w, K, st);
}

}  // namespace KGE_ELT_NS
}  // namespace kge

using namespace kge;

extern "C" int KGE_API(kge_gemm_fp8)(void* y, const void* x, const float* x_scales, int x_scales_stride, const void* w, const float* w_scales, const void* bias, int T, int N, int K,
                                     void* workspace, int64_t workspace_bytes, void* stream) {
  Fp8Params p = {};
  p.y = (bf16*)y; p.bias = (const bf16*)bias; p.xs = x_scales; p.ws = w_scales; p.E = 1; p.T = T; p.N = N;
  return gemm_fp8("kge_gemm_fp8", p, false, x, x_scales_stride, w, K, workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" int KGE_API(kge_gemm_fp8_grouped)(void* y, const void* x, const float* x_scales, int x_scales_stride, const void* w, const float* w_scales, const int32_t* offsets, int E,
                                             int T, int N, int K, void* workspace, int64_t workspace_bytes, void* stream) {
  KGE_REQUIRE(offsets, "kge_gemm_fp8_grouped: null pointer");
  Fp8Params p = {};
  p.y = (bf16*)y; p.xs = x_scales; p.ws = w_scales; p.offsets = offsets; p.E = E; p.T = T; p.N = N;
  return gemm_fp8("kge_gemm_fp8_grouped", p, false, x, x_scales_stride, w, K, workspace, workspace_bytes, (cudaStream_t)stream);
}

#ifndef KGE_HALF      // codes come out of these: the same for both element types
extern "C" int64_t kge_gemm_fp8_workspace_bytes(int T) { return workspace_bytes_of(T); }

extern "C" int kge_gemm_fp8_silu_gate(void* codes, float* scales, int scales_stride, const void* x, const float* x_scales, int x_scales_stride, const void* w_gate_up,
                                      const float* w_scales, int T, int f, int K, void* workspace, int64_t workspace_bytes, void* stream) {
  Fp8Params p = {};
  p.codes = (uint8_t*)codes; p.out_scales = scales; p.out_stride = scales_stride; p.xs = x_scales; p.ws = w_scales; p.E = 1; p.T = T; p.N = f;
  return gemm_fp8("kge_gemm_fp8_silu_gate", p, true, x, x_scales_stride, w_gate_up, K, workspace, workspace_bytes, (cudaStream_t)stream);
}

extern "C" int kge_gemm_fp8_grouped_silu_gate(void* codes, float* scales, int scales_stride, const void* x, const float* x_scales, int x_scales_stride, const void* w_gate_up,
                                              const float* w_scales, const int32_t* offsets, int E, int T, int f, int K, void* workspace, int64_t workspace_bytes, void* stream) {
  KGE_REQUIRE(offsets, "kge_gemm_fp8_grouped_silu_gate: null pointer");
  Fp8Params p = {};
  p.codes = (uint8_t*)codes; p.out_scales = scales; p.out_stride = scales_stride; p.xs = x_scales; p.ws = w_scales; p.offsets = offsets; p.E = E; p.T = T; p.N = f;
  return gemm_fp8("kge_gemm_fp8_grouped_silu_gate", p, true, x, x_scales_stride, w_gate_up, K, workspace, workspace_bytes, (cudaStream_t)stream);
}
#endif
