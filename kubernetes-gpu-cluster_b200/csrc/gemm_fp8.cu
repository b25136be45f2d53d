// Products of 8-bit codes with a scale for each block of 128 (fp8.cuh), dense and grouped by expert:
//   y[t, n] = sum_b xs[b, t] ws[n / 128, b] sum_{k in block b} x[t, k] w[n, k]  (+ bias[n])
//   h[t, j] = silu(gate) * up of such a pair of products, quantised row by row in blocks of 128 in the same kernel.
//
// Orientation: the MMA's M rows are TOKENS and its N columns weight rows, so that what a thread reads back of tensor memory (one lane) belongs to one
// token and, within 128 columns, to one scale of the weights: a single factor for all of them.  tcgen05.mma sums a block of K (four instructions of
// 32) in fp32 in tensor memory, and eight warps add it, times its factor, to accumulators in registers.  Tensor memory holds several blocks, so that the next ones are multiplied meanwhile.
//
// Two kernels.
//  fp8_stream_kernel: tiles of 128 tokens x NT weight rows by single CTAs, one an SM; the (tile, block of K) units of the whole problem are laid end
//    to end and cut into equal shares, so every SM reads the same number of weight bytes whatever the sizes are.  A tile that a share's end cuts is
//    summed by the last of its CTAs to arrive, from fp32 partial sums in the workspace and in the order of K: the same bits each time.
//  fp8_pair_kernel: tiles of 256 x 256 by pairs of CTAs (cta_group::2), for many tokens: a CTA has its own 128 tokens and half of the weight rows in
//    shared memory, 32 KB a block of K, where its MMA takes 512 cycles.
#include <cuda.h>

#include "fp8.cuh"
#include "kge.h"

namespace kge {
inline namespace KGE_ELT_NS {

constexpr int kRows = 128;                        // tokens of a CTA's tile
constexpr int kSlab = 128 * 128;                  // bytes of 128 rows of a block of K
#ifndef FP8_CHUNK
#define FP8_CHUNK 32
#define FP8_UP 216
#define FP8_DOWN 72
#endif
constexpr int kSumWarps = 8;                      // warps that add up: a token of 128 and 64 columns of each 128 a thread
constexpr int kThreads = 128 + 32 * kSumWarps;    // producer, MMA, tensor memory, factors; those
constexpr int kChunk = FP8_CHUNK;                 // columns that a warp reads of tensor memory at a time
constexpr int kCounters = 256;                    // arrival counters at the head of the workspace
constexpr int kMaxCtas = 160;
constexpr int kMaxGroups = 1024;
constexpr int kSmem = 226 * 1024;
constexpr int kPairStages = 6;
constexpr int kPairSlots = kPairStages + 2;
constexpr int kPairBatch = 4, kBatch = 2;         // blocks that a warp prepares factors of at a time
static_assert(kPairStages > kPairBatch, "");
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
  int wide;                                       // pairs: y's rows are 16-byte aligned
  int quarters, stages, x_bytes, min_units;       // stream: 32-row quarters that a tile can have, stages, bytes of a stage's tokens, least units of a share
};

__device__ __forceinline__ uint32_t s_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory"); }
// On a barrier of the pair's leader.  What it tells is that tensor memory has been read (tcgen05.wait::ld, the fence before): nothing in memory is
// published, and a release for the whole cluster would wait for all of a thread's stores, every block of K (2048 x 9472 x 4096: 194 us with it).
__device__ __forceinline__ void bar_arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
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
// N columns of this warp's 32 lanes; the caller waits (tmem_wait_ld)
template <int N>
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[N]) {
  static_assert(N == 16 || N == 32, "");
  if constexpr (N == 32)
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
                   "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(at));
  else
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
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
// starts[e] = tiles of the groups before e.  By all threads of the CTA.
__device__ __forceinline__ void count_tiles(const Fp8Params& p, int tile_rows, int* starts) {
  for (int e = threadIdx.x; e < p.E; e += kThreads) {
    int r0, r1;
    group_rows(p, e, r0, r1);
    starts[e] = (r1 - r0 + tile_rows - 1) / tile_rows * p.n_tiles;
  }
  __syncthreads();
  if (threadIdx.x < 32) {
    int total = 0;
    for (int e0 = 0; e0 < p.E; e0 += 32) {
      const int e = e0 + threadIdx.x, n = e < p.E ? starts[e] : 0;
      int s = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, s, o); if ((int)threadIdx.x >= o) s += v; }
      if (e < p.E) starts[e] = total + s - n;
      total += __shfl_sync(0xffffffffu, s, 31);
    }
    if (threadIdx.x == 0) starts[p.E] = total;
  }
  __syncthreads();
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
  float v[C];
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < C; ++i) v[i] = 0.f;
  }
  // += factor * D of kChunk columns at c
  __device__ __forceinline__ void add(int c, const uint32_t (&r)[kChunk], float factor) {
#pragma unroll
    for (int i = 0; i < kChunk; ++i) asm volatile("fma.rn.f32 %0, %1, %2, %0;" : "+f"(v[c + i]) : "f"(__uint_as_float(r[i])), "f"(factor));
  }
  __device__ __forceinline__ void at(int c, float& a, float& b) const { a = v[c]; b = v[c + 1]; }
};

// Adds up `blocks` blocks of K.  wait(): the address of the next block's columns in tensor memory and its factors, when they are there; read(): they are
// in registers.  A thread's second 64 columns (if it has them) lie SKIP columns behind its first, with a factor of their own.  The next block is waited
// for, and its first columns asked for, before the last ones of this block are added, so that the way to tensor memory and back passes under arithmetic.
template <int C, int SKIP, typename W, typename R>
__device__ __forceinline__ void add_blocks(Sums<C>& s, int blocks, W wait, R read) {
  uint32_t r[2][kChunk], at;
  float f0, f1;
  wait(at, f0, f1);
  tmem_ld(at, r[0]);
#pragma unroll 1
  for (; blocks > 0; --blocks) {
    const float g0 = f0, g1 = f1;
#pragma unroll
    for (int c = 0; c < C; c += kChunk) {
      uint32_t (&now)[kChunk] = r[(c / kChunk) & 1], (&then)[kChunk] = r[(c / kChunk + 1) & 1];
      tmem_wait_ld(now);
      if (c + kChunk < C) {
        tmem_ld(at + c + kChunk + (c + kChunk >= 64 ? SKIP : 0), then);
      } else {
        read();
        if (blocks > 1) {
          wait(at, f0, f1);
          tmem_ld(at, then);
        }
      }
      s.add(c, now, c < 64 ? g0 : g1);
    }
  }
}

// The factors of a tile's rows, block of K by block of K: xs ws for the 128 rows and its first (gate) and second (up) 128 columns, by two warps for
// those that add up, in a ring in shared memory, BATCH blocks of one and BATCH of the other.  A warp sees every barrier of the stages' ring at least once a
// round, as a wait by parity needs it, where there are more stages than the other's blocks.  (A thread's own loads, two blocks ahead, came too late: with the copies at full rate a load takes
// more than 1000 cycles, and 190 to 230 cycles of every block went into waiting for it.)
template <int SETS, int BATCH>
struct Factors {
  float x[BATCH][4], w[BATCH][SETS];
  // asks for n <= BATCH blocks from kb on
  __device__ __forceinline__ void ask(const Fp8Params& p, int row, int rows, int64_t block0, int64_t block1, int kb, int n, int lane) {
#pragma unroll
    for (int i = 0; i < BATCH; ++i) {
#pragma unroll
      for (int q = 0; q < 4; ++q) x[i][q] = i < n && q * 32 + lane < rows ? __ldg(p.xs + (kb + i) * p.xs_stride + row + q * 32 + lane) : 0.f;
      w[i][0] = i < n ? __ldg(p.ws + block0 * p.KB + kb + i) : 0.f;
      if (SETS == 2) w[i][SETS - 1] = i < n ? __ldg(p.ws + block1 * p.KB + kb + i) : 0.f;
    }
  }
  __device__ __forceinline__ void put(float* slot, int i, int lane) const {
#pragma unroll
    for (int s = 0; s < SETS; ++s)
#pragma unroll
      for (int q = 0; q < 4; ++q) slot[s * 128 + q * 32 + lane] = x[i][q] * w[i][s];
  }
};

// 64 columns of a row from n0 on, rounded once; c0: where their sums begin.
template <int C>
__device__ __forceinline__ void store_row(const Fp8Params& p, const Sums<C>& s, int c0, int row, int n0) {
  bf16* dst = p.y + (int64_t)row * p.N + n0;
  if (n0 + 64 <= p.N && (p.N & 7) == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0) {
#pragma unroll
    for (int c = 0; c < 64; c += 8) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        float a, b;
        s.at(c0 + c + 2 * i, a, b);
        if (p.bias) { a += bf2f(p.bias[n0 + c + 2 * i]); b += bf2f(p.bias[n0 + c + 2 * i + 1]); }
        u[i] = pack_bf2(a, b);
      }
      *reinterpret_cast<uint4*>(dst + c) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  } else {
#pragma unroll
    for (int c = 0; c < 64; c += 2) {
      float a, b;
      s.at(c0 + c, a, b);
      if (n0 + c < p.N) dst[c] = f2bf(p.bias ? a + bf2f(p.bias[n0 + c]) : a);
      if (n0 + c + 1 < p.N) dst[c + 1] = f2bf(p.bias ? b + bf2f(p.bias[n0 + c + 1]) : b);
    }
  }
}

// A warp's 32 rows (from `row` on, `rows` of them there) of C columns, 32 at a time through 2 KB of its own in shared memory: rows of 64 bytes, whose
// 16-byte pieces are exchanged by two bits of the row, so that neither side meets in a bank.  A lane then stores 16 bytes beside its neighbour's.
template <int C>
__device__ __forceinline__ void store_rows(const Fp8Params& p, const Sums<C>& s, int row, int rows, int n0, uint32_t buffer, int lane) {
  const int j = lane & 3, r = lane >> 2;
  const uint32_t put = buffer + lane * 64, get = buffer + r * 64 + ((j ^ ((r >> 1) & 3)) << 4);
  bf16* dst = p.y + (int64_t)(row + r) * p.N + n0 + j * 8;
#pragma unroll
  for (int c0 = 0; c0 < C; c0 += 32) {
    if (n0 + c0 >= p.N) break;
    __syncwarp();
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      uint32_t u[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int c = c0 + k * 8 + 2 * i;
        float a, b;
        s.at(c, a, b);
        if (p.bias) {
          const int at = n0 + c;
          if (at < p.N) a += bf2f(p.bias[at]);
          if (at + 1 < p.N) b += bf2f(p.bias[at + 1]);
        }
        u[i] = pack_bf2(a, b);
      }
      asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(put + ((k ^ ((lane >> 1) & 3)) << 4)), "r"(u[0]), "r"(u[1]), "r"(u[2]), "r"(u[3]) : "memory");
    }
    __syncwarp();
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t u[4];
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]) : "r"(get + i * 512) : "memory");
      if (r + i * 8 < rows && n0 + c0 + j * 8 < p.N) *reinterpret_cast<uint4*>(dst + (int64_t)i * 8 * p.N + c0) = make_uint4(u[0], u[1], u[2], u[3]);
    }
  }
}

// Gated: a thread has 64 columns of the gate and the same of up, the block's other 64 are another warp's; its largest magnitude goes through shared
// memory (two rows of 128 words).  Called by all warps that add up.
__device__ __forceinline__ void store_gated(const Fp8Params& p, const Sums<128>& s, int row, bool there, int n, uint32_t* tops, int part, int lane128) {
  constexpr int H = 64;
  float h[H];
  uint32_t m = 0;
#pragma unroll
  for (int c = 0; c < H; c += 2) {
    float g[2], u[2];
    s.at(c, g[0], g[1]);
    s.at(H + c, u[0], u[1]);
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      h[c + i] = __fdividef(g[i], 1.f + __expf(-g[i])) * u[i];
      m = max(m, __float_as_uint(h[c + i]) & 0x7fffffffu);       // (NaN above all)
    }
  }
  tops[part * 128 + lane128] = m;
  sums_sync();
  m = max(m, tops[(part ^ 1) * 128 + lane128]);
  sums_sync();                                                   // (the next tile writes there)
  if (!there) return;
  float scale, factor;
  fp8::scale_of(__uint_as_float(m), scale, factor);
  uint8_t* dst = p.codes + (int64_t)row * p.N + n * 128 + part * H;
#pragma unroll
  for (int c = 0; c < H; c += 16) {
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
      q[i] = factor > 0.f ? fp8::pack4(h[c + 4 * i] * factor, h[c + 4 * i + 1] * factor, h[c + 4 * i + 2] * factor, h[c + 4 * i + 3] * factor) : 0u;
    *reinterpret_cast<uint4*>(dst + c) = make_uint4(q[0], q[1], q[2], q[3]);
  }
  if (part == 0) p.out_scales[n * p.out_stride + row] = scale;
}

// ----------------------------------------------------------------------------------------------------- equal shares of all units

// U units in G equal shares: share c begins at floor(U c / G) (one 32-bit quotient of small numbers).
struct Shares {
  uint32_t U, G, q, r;
  __device__ __forceinline__ Shares(uint32_t units, uint32_t shares) : U(units), G(shares), q(units / shares), r(units - units / shares * shares) {}
  __device__ __forceinline__ uint32_t begin(uint32_t c) const { return q * c + r * c / G; }
  // the share with unit x
  __device__ __forceinline__ uint32_t of(uint32_t x) const {
    uint32_t c = min(G - 1, (uint32_t)((float)x * ((float)G / (float)U)));
    while (begin(c) > x) --c;
    while (c + 1 < G && begin(c + 1) <= x) ++c;
    return c;
  }
};
// A share as pieces of tiles: blocks of K [kb0, kb1) of tile `tile`.
struct Pieces {
  int cur, end, KB, tile, kb;
  __device__ __forceinline__ Pieces(int u0, int u1, int KB_, int tile0) : cur(u0), end(u1), KB(KB_), tile(tile0), kb(u0 - tile0 * KB_) {}
  __device__ __forceinline__ bool next(int& t, int& kb0, int& kb1) {
    if (cur >= end) return false;
    t = tile; kb0 = kb;
    kb1 = min(KB, kb + end - cur);
    cur += kb1 - kb0;
    ++tile; kb = 0;
    return true;
  }
};

template <int NT, bool GATED>
__global__ void __launch_bounds__(kThreads, 1)
fp8_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Fp8Params p) {
  constexpr int C = NT / 2, BUFS = 512 / NT, SETS = NT / 128;
  static_assert(!GATED || NT == 256, "a gated tile holds 128 columns of each");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * 32 + 2 * BUFS];
  __shared__ uint32_t tmem_slot;
  __shared__ int last_flag;
  __shared__ uint32_t tops[256];
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
    for (int s = 0; s < stages; ++s) { bar_init(full(s), 2); bar_init(empty(s), 1); }
    for (int b = 0; b < BUFS; ++b) { bar_init(tfull(b), 1); bar_init(tempty(b), kSumWarps); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (!p.offsets && threadIdx.x == 0) { starts[0] = 0; starts[1] = (p.T + kRows - 1) / kRows * p.n_tiles; }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_launch_dependents();
  if (p.offsets) {                                  // which tiles there are is the kernel before's output
    pdl_wait();
    count_tiles(p, kRows, starts);
  }
  const int KB = p.KB;
  const uint32_t U = (uint32_t)starts[p.E] * KB;
  const Shares shares(U, max(1u, min(gridDim.x, U / p.min_units)));
  const uint32_t me = blockIdx.x, u0 = me < shares.G ? shares.begin(me) : U, u1 = me < shares.G ? shares.begin(me + 1) : U;
  const int tile0 = u0 < u1 ? (int)(u0 / (uint32_t)KB) : 0, e_first = u0 < u1 ? first_group(p, starts, tile0) : 0;
  // A slot of the ring is free again when its block is added up.  The block `stages` further is then at the earliest on its way (its stage was freed by an
  // MMA that began after the sums BUFS blocks before had been read).
  float* factors = reinterpret_cast<float*>(smem + stages * stage_bytes);
  const int slots = stages + BUFS;

  if (warp == 0) {
    regs_down<FP8_DOWN>();
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      auto load_w = [&](int s, const Tile& t, int kb) {
        const uint32_t dst = base + s * stage_bytes + p.x_bytes;
        const int row = t.e * p.w_rows;
#pragma unroll
        for (int h = 0; h < NT / 128; ++h) load_box(dst + h * kSlab, &map_w, full(s), kb * 128, row + (GATED ? t.n * 128 + h * p.N : t.n * NT + h * 128));
      };
      auto load_x = [&](int s, const Tile& t, int kb) {
        for (int r = 0; r < t.rows; r += 32) load_box(base + s * stage_bytes + r * 128, &map_x, full(s), kb * 128, t.row + r);
      };
      auto bytes_of = [&](const Tile& t) { return (uint32_t)(NT * 128 + (t.rows + 31) / 32 * 4096); };
      // What the weights are is known before the kernel before has ended: its first tile's, as many as there are stages.
      int tile, kb0, kb1, ahead = 0, e = e_first;
      if (!p.offsets) {
        Pieces it(u0, u1, KB, tile0);
        if (it.next(tile, kb0, kb1)) {
          const Tile t = find_tile<kRows, 0>(p, starts, tile, e);
          ahead = min(stages, kb1 - kb0);
          for (int i = 0; i < ahead; ++i) { bar_expect(full(i), bytes_of(t)); load_w(i, t, kb0 + i); }
        }
        pdl_wait();
      }
      Pieces it(u0, u1, KB, tile0);
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
    regs_down<FP8_DOWN>();
    if (elect_one()) {
      constexpr uint32_t idesc = instr_desc(kRows, NT);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      const uint64_t a0 = tile_desc(base), b0 = tile_desc(base + p.x_bytes);
      uint64_t a = a0, b = b0;
      for (uint32_t u = u0; u < u1; ++u) {
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
    regs_down<FP8_DOWN>();
    pdl_wait();
    int stage = 0, slot = 0, tile, kb0, kb1, e = e_first, turn = warp & 1;
    uint32_t phase = 0;
    Pieces it(u0, u1, KB, tile0);
    while (it.next(tile, kb0, kb1)) {
      const Tile t = find_tile<kRows, 0>(p, starts, tile, e);
      const int64_t wb = (int64_t)t.e * p.w_blocks + (GATED ? t.n : t.n * SETS);
      Factors<SETS, kBatch> f;
      for (int kb = kb0; kb < kb1; kb += kBatch) {
        turn ^= 1;
        if (turn) {                                  // the other warp's
          const int n = min(kBatch, kb1 - kb);
          for (stage += n; stage >= stages; stage -= stages) phase ^= 1;
          for (slot += n; slot >= slots; slot -= slots) {}
          continue;
        }
        f.ask(p, t.row, t.rows, wb, GATED ? wb + p.N / 128 : wb + (t.n * SETS + 1 < p.w_blocks), kb, min(kBatch, kb1 - kb), lane);
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
          if (kb + i >= kb1) break;
          mbar_wait(empty(stage), phase ^ 1);
          f.put(factors + slot * SETS * 128, i, lane);
          __syncwarp();
          if (lane == 0) bar_arrive(full(stage));
          if (++stage == stages) { stage = 0; phase ^= 1; }
          if (++slot == slots) slot = 0;
        }
      }
    }
  } else {
    regs_up<FP8_UP>();
    const int q = warp & 3, part = (warp - 4) >> 2, tid = threadIdx.x - 128, lane128 = q * 32 + lane;
    pdl_wait();
    int buf = 0, slot = 0, tile, kb0, kb1, e = e_first;
    uint32_t buf_phase = 0;
    Pieces it(u0, u1, KB, tile0);
    while (it.next(tile, kb0, kb1)) {
      const Tile t = find_tile<kRows, 0>(p, starts, tile, e);
      const bool some = q * 32 < t.rows, there = lane128 < t.rows;
      const int row = t.row + lane128, n0 = t.n * NT + part * 64;
      Sums<C> s;
      s.clear();
      const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + part * 64;
      auto read = [&] {
        fence_before();
        if (lane == 0) bar_arrive(tempty(buf));
        if (++buf == BUFS) { buf = 0; buf_phase ^= 1; }
        if (++slot == slots) slot = 0;
      };
      auto wait = [&](uint32_t& from, float& f0, float& f1) {
        mbar_wait(tfull(buf), buf_phase);
        fence_after();
        const float* f = factors + slot * SETS * 128 + lane128;
        f0 = f[0];
        f1 = f[SETS == 2 ? 128 : 0];
        from = at + buf * NT;
      };
      if (some) {
        add_blocks<C, 64>(s, kb1 - kb0, wait, read);
      } else {
        for (int kb = kb0; kb < kb1; ++kb) { mbar_wait(tfull(buf), buf_phase); read(); }
      }
      if (kb1 - kb0 != KB) {
        // A part of the tile's sum: to the workspace, [slot][quarter][part][column / 4][lane] of 16 bytes.  A share has at most two such pieces: slot 0
        // the one that it begins with.
        constexpr int kPer = (NT / 4) * 32;          // float4 of a quarter
        const uint32_t x0 = (uint32_t)tile * KB;
        auto slot_of = [&](uint32_t cta, int slot) { return reinterpret_cast<float4*>(p.part) + ((cta * 2 + slot) * p.quarters + q) * kPer + part * (C / 4) * 32 + lane; };
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
        sums_sync();
        // its CTAs: from the one with its first unit to the one with its last; they count in the first one's counter
        const uint32_t c0 = shares.of(x0), c1 = shares.of(x0 + KB - 1);
        if (tid == 0) {
          __threadfence();                              // (of what all threads of the barrier have stored)
          const bool mine = atomicAdd(p.count + c0, 1u) == c1 - c0;
          if (mine) p.count[c0] = 0;                    // ready for the next launch
          __threadfence();
          last_flag = mine;
        }
        sums_sync();
        const bool last = last_flag != 0;
        sums_sync();                                    // (the next piece writes there)
        if (!last) continue;
        s.clear();
        if (some)
#pragma unroll
          for (int h = 0; h < C; h += 64)
            for (uint32_t c = c0; c <= c1; ++c) {
              const float4* src = slot_of(c, shares.begin(c) >= x0 ? 0 : 1) + h / 4 * 32;
              float4 v[16];
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __ldcg(src + i * 32);
#pragma unroll
              for (int i = 0; i < 16; ++i) { s.v[h + 4 * i] += v[i].x; s.v[h + 4 * i + 1] += v[i].y; s.v[h + 4 * i + 2] += v[i].z; s.v[h + 4 * i + 3] += v[i].w; }
            }
      }
      if constexpr (GATED) {
        store_gated(p, s, row, there, t.n, tops, part, lane128);
      } else if (there) {
#pragma unroll
        for (int h = 0; h < C / 64; ++h) store_row<C>(p, s, h * 64, row, n0 + h * 128);
      }
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
  __shared__ uint64_t bars[2 * STAGES + 8];
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t tops[256];
  __shared__ int4 tiles[16];                        // n, row, rows of the tiles under way: at most one a block of K of the rings, and the last one
  __shared__ int starts[kMaxGroups + 1];
  const uint32_t base = s_addr(smem), bar0 = s_addr(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tfull = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto tempty = [&](int b) { return bar0 + 8u * (2 * STAGES + 4 + b); };
  const int warp = uniform_warp(), lane = threadIdx.x & 31, rank = (int)cluster_ctarank();

  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) { bar_init(full(s), 3); bar_init(empty(s), 2); }       // (full: the leader's copies, both CTAs' factors)
    for (int b = 0; b < 4; ++b) { bar_init(tfull(b), 1); bar_init(tempty(b), kSumWarps); }       // (of two blocks, the first and the second 128 columns)
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (!p.offsets && threadIdx.x == 0) { starts[0] = 0; starts[1] = (p.T + 2 * kRows - 1) / (2 * kRows) * p.n_tiles; }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_launch_dependents();
  cluster_arrive(); cluster_wait();                 // the peer's barriers are there
  pdl_wait();
  if (p.offsets) count_tiles(p, 2 * kRows, starts);
  const int KB = p.KB, total = starts[p.E], first = (int)blockIdx.x >> 1, step = (int)gridDim.x >> 1;
  const int e_first = first < total ? first_group(p, starts, first) : 0;
  float* factors = reinterpret_cast<float*>(smem + STAGES * kStage + (GATED ? 0 : kSumWarps * 2048));

  if (warp == 0 || warp == 3) {
    // the copies and factors of kPairBatch blocks of K by one of the two, of as many by the other
    regs_down<FP8_DOWN>();
    int stage = 0, slot = 0, tile = 0, e = e_first, turn = 1 - (warp & 1);
    uint32_t phase = 0;
    const uint32_t lead0 = mapa_u32(full(0), 0);
    for (int w = first; w < total; w += step) {
      const Tile t = find_tile<2 * kRows, kPairBand>(p, starts, w, e);
      const int64_t wb = (int64_t)t.e * p.w_blocks + (GATED ? t.n : t.n * 2);
      // 64 weight rows for the first 128 columns, 64 for the second: half of each block or, gated, the leader's of the gate and the other's of up
      const int wr = t.e * p.w_rows + (GATED ? t.n * 128 + rank * p.N : t.n * 256 + rank * 64), xr = t.row + rank * kRows;
      Factors<2, kPairBatch> f;
      if (turn && lane == 0) tiles[tile & 15] = make_int4(t.n, t.row, t.rows, 0);      // (the first batch is this warp's)
      ++tile;
      for (int kb = 0; kb < KB; kb += kPairBatch) {
        const int n = min(kPairBatch, KB - kb);
        turn ^= 1;
        if (turn) {                                  // the other warp's
          for (stage += n; stage >= STAGES; stage -= STAGES) phase ^= 1;
          slot = (slot + n) % kPairSlots;
          continue;
        }
        f.ask(p, xr, t.rows - rank * kRows, wb, GATED ? wb + p.N / 128 : wb + (t.n * 2 + 1 < p.w_blocks), kb, n, lane);
#pragma unroll
        for (int i = 0; i < kPairBatch; ++i) {
          if (i >= n) break;
          mbar_wait(empty(stage), phase ^ 1);
          const uint32_t lead = lead0 + 8u * stage;
          if (elect_one()) {
            if (rank == 0) bar_expect(full(stage), 2 * kStage);
            const uint32_t dst = base + stage * kStage;
            load_box2(dst, &map_x, lead, (kb + i) * 128, xr);
            load_box2(dst + kSlab, &map_w, lead, (kb + i) * 128, wr);
            load_box2(dst + kSlab + kSlab / 2, &map_w, lead, (kb + i) * 128, wr + (GATED ? 64 : 128));
          }
          __syncwarp();
          f.put(factors + slot * 256, i, lane);
          __syncwarp();
          if (lane == 0) bar_arrive_at(lead);
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
          if (++slot == kPairSlots) slot = 0;
        }
      }
    }
  } else if (warp < 4) {
    regs_down<FP8_DOWN>();
    if (rank == 0 && elect_one()) {                 // the leader issues for both, the first 128 columns by one thread and the second by another
      constexpr uint32_t idesc = instr_desc(2 * kRows, 128);
      const int h = warp - 1;
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      const uint64_t a0 = tile_desc(base), b0 = tile_desc(base + kSlab + h * (kSlab / 2));
      uint64_t a = a0, b = b0;
      const uint32_t d = tmem + h * 128;
      const int tiles = first < total ? (total - 1 - first) / step + 1 : 0;
      bool f_there = false, t_there = false;
      for (int64_t n = (int64_t)tiles * KB; n > 0; --n) {
        if (!f_there) mbar_wait(full(stage), phase);
        if (!t_there) mbar_wait(tempty(2 * buf + h), buf_phase ^ 1);
        const int s1 = stage + 1 == STAGES ? 0 : stage + 1, v1 = buf ^ 1;
        const uint32_t p1 = stage + 1 == STAGES ? phase ^ 1 : phase, w1 = buf_phase ^ buf;
        f_there = mbar_test(full(s1), p1);
        t_there = mbar_test(tempty(2 * v1 + h), w1 ^ 1);
        fence_after();
#pragma unroll
        for (int k = 0; k < 4; ++k) mma8x2(d + buf * 256, a + 2 * k, b + 2 * k, idesc, k > 0);
        commit2(tfull(2 * buf + h), 3);
        commit2(empty(stage), 3);
        a += kStage >> 4; b += kStage >> 4;
        if (s1 == 0) { a = a0; b = b0; }
        stage = s1; phase = p1; buf = v1; buf_phase = w1;
      }
    }
  } else {
    regs_up<FP8_UP>();
    const int q = warp & 3, part = (warp - 4) >> 2, lane128 = q * 32 + lane;
    const uint32_t lead_tempty = mapa_u32(tempty(part), 0);
    int buf = 0, slot = 0, tile = 0;
    uint32_t buf_phase = 0;
    for (int w = first; w < total; w += step) {
      mbar_wait(tfull(2 * buf + part), buf_phase);
      const int4 found = tiles[tile++ & 15];
      const Tile t = {0, found.x, found.y, found.z};
      const int mine = rank * kRows + lane128;
      const bool some = rank * kRows + q * 32 < t.rows, there = mine < t.rows;
      const int row = t.row + mine, n0 = t.n * 256 + part * 128;
      Sums<C> s;
      s.clear();
      const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + part * 128;
      auto read = [&] {
        fence_before();
        if (lane == 0) bar_arrive_at(lead_tempty + 16u * buf);
        if (++buf == 2) { buf = 0; buf_phase ^= 1; }
        if (++slot == kPairSlots) slot = 0;
      };
      auto wait = [&](uint32_t& from, float& f0, float& f1) {
        mbar_wait(tfull(2 * buf + part), buf_phase);
        fence_after();
        const float* f = factors + slot * 256 + lane128;
        f0 = f[GATED ? 0 : part * 128];
        f1 = GATED ? f[128] : f0;
        from = at + buf * 256;
      };
      if (some) {
        add_blocks<C, 0>(s, KB, wait, read);
      } else {
        for (int kb = 0; kb < KB; ++kb) { mbar_wait(tfull(2 * buf + part), buf_phase); read(); }
      }
      if constexpr (GATED) {
        store_gated(p, s, row, there, t.n, tops, part, lane128);
      } else if (p.wide) {
        if (some) store_rows<C>(p, s, row - lane, t.rows - (mine - lane), n0, base + STAGES * kStage + (warp - 4) * 2048, lane);
      } else if (there) {
#pragma unroll
        for (int h = 0; h < C / 64; ++h) store_row<C>(p, s, h * 64, row, n0 + h * 64);
      }
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

static bool aligned_to(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n < kMaxCtas ? n : kMaxCtas;
}

template <int NT, bool GATED>
static int launch_stream(Fp8Params& p, const void* x, const void* w, int K, cudaStream_t st) {
  const int widest = p.T < kRows ? p.T : kRows;
  p.quarters = (widest + 31) / 32;
  p.x_bytes = p.quarters * 4096;
  p.n_tiles = (p.N + (GATED ? 128 : NT) - 1) / (GATED ? 128 : NT);
  constexpr int own = 8 * 1024;                            // the kernel's own shared memory, and rounding up to 1024
  constexpr int slot_bytes = NT / 128 * 512, more = 512 / NT;
  p.stages = (kSmem - own - more * slot_bytes) / (p.x_bytes + NT * 128 + slot_bytes);
  if (p.stages > 16) p.stages = 16;
  static_assert((kSmem - own - more * slot_bytes) / (kRows * 128 + NT * 128 + slot_bytes) > kBatch, "");
  p.min_units = 2;
  // an MMA reads 128 rows of tokens from where they begin, and finds others' bytes behind the last: never beyond the stage's weights
  static_assert(NT * 128 >= kRows * 128, "");
  const int smem = p.stages * (p.x_bytes + NT * 128 + slot_bytes) + more * slot_bytes + 1024;
  CUtensorMap mw, mx;
  if (int rc = encode_map(&mw, w, (int64_t)p.E * p.w_rows, K, 128)) return rc;
  if (int rc = encode_map(&mx, x, p.T, K, 32)) return rc;
  auto kern = fp8_stream_kernel<NT, GATED>;
  KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  const int sms = sm_count();
  KGE_REQUIRE(sms > 0, "kge_gemm_fp8: no CUDA device");
  int64_t ctas = sms;
  if (!p.offsets) {
    // Whole numbers of CTAs a tile cost each of them one partial sum in place of two: worth up to a tenth of the SMs.
    const int64_t tiles = (int64_t)((p.T + kRows - 1) / kRows) * p.n_tiles, most = tiles * p.KB / p.min_units, even = tiles < sms ? sms / tiles * tiles : sms;
    if (even * 10 >= sms * 9) ctas = even;
    if (ctas > most) ctas = most < 1 ? 1 : most;
  }
  KGE_CUDA_OK(launch_pdl(kern, dim3((unsigned)ctas), dim3(kThreads), (size_t)smem, st, mw, mx, p));
  return 0;
}

template <bool GATED>
static int launch_pairs(Fp8Params& p, const void* x, const void* w, int K, cudaStream_t st) {
  p.n_tiles = (p.N + (GATED ? 128 : 256) - 1) / (GATED ? 128 : 256);
  const int smem = kPairStages * 2 * kSlab + kPairSlots * 1024 + (GATED ? 0 : kSumWarps * 2048) + 1024;
  CUtensorMap mw, mx;
  if (int rc = encode_map(&mw, w, (int64_t)p.E * p.w_rows, K, 64)) return rc;
  if (int rc = encode_map(&mx, x, p.T, K, 128)) return rc;
  p.wide = !GATED && p.N % 8 == 0 && aligned_to(p.y, 16);
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
  KGE_REQUIRE(tiles * p.KB < (1ll << 31), "%s: %lld tiles of %d blocks in one call", name, (long long)tiles, p.KB);
  KGE_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(p.T) && aligned_to(workspace, 16), "%s: needs a workspace of %lld bytes, 16-byte aligned", name,
              (long long)workspace_bytes_of(p.T));
  p.count = (unsigned int*)workspace;
  p.part = (float*)((uint8_t*)workspace + kCounters * 4);
  const bool pairs = p.T / p.E > 96;
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
