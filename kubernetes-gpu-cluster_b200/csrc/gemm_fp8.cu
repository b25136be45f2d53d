// Products of 8-bit codes with a scale for each block of 128 (fp8.cuh), dense and grouped by expert:
//   y[t, n] = sum_b xs[b, t] ws[n / 128, b] sum_{k in block b} x[t, k] w[n, k]  (+ bias[n])
//   h[t, j] = silu(gate) * up of such a pair of products, quantised row by row in blocks of 128 in the same kernel.
//
// Orientation: the MMA's M rows are TOKENS and its N columns weight rows, so that what a thread reads back of tensor memory (one lane) belongs to one
// token and, within 128 columns, to one scale of the weights: a single factor for all of them.  tcgen05.mma sums a block of K (four instructions of
// 32) in fp32 in tensor memory, and eight warps add it, times its factor, to accumulators in registers.  Tensor memory holds several blocks, so that the next ones are multiplied meanwhile.
//
// Two kernels.
//  fp8_stream_kernel: tiles of 128 tokens x 128 or 256 weight rows by single CTAs, one an SM, for calls that a pass over the weights bounds.  With at least
//    half as many tiles as SMs a CTA has whole tiles; fewer tiles are cut along K, over the CTAs of a cluster where the host knows their number, and
//    else (few rows in groups) over CTAs that meet in the workspace.  Shares are added in the order of K: the same bits each time.
//  fp8_pair_kernel: tiles of 256 x 256 by pairs of CTAs (cta_group::2), for many tokens: a CTA has its own 128 tokens and half of the weight rows in
//    shared memory, 32 KB a block of K, where its MMA takes 512 cycles.
#include <cuda.h>

#include <atomic>

#include "fp8.cuh"
#include "kge.h"

namespace kge {
inline namespace KGE_ELT_NS {

constexpr int kRows = 128;                        // tokens of a CTA's tile
constexpr int kSlab = 128 * 128;                  // bytes of 128 rows of a block of K
constexpr int kSumWarps = 8;                      // warps that add up: a token of 128 and 64 columns of each 128 a thread
constexpr int kThreads = 128 + 32 * kSumWarps;    // producer, MMA, tensor memory, factors; those
constexpr int kSumRegs = 216, kOtherRegs = 72;    // registers of those and of the others: 256 x 216 + 128 x 72 = 384 x 168, what the block is launched with
constexpr int kCounters = 256;                    // arrival counters at the head of the workspace
constexpr int kMaxCtas = 160;
constexpr int kMaxGroups = 1024, kNearGroups = 256;      // groups; those whose rows are kept in shared memory
constexpr int kMaxStages = 16;
constexpr int kSlotBytes = 136 * 4;               // factors of a block of K: of 128 rows, of up to two sets of columns
constexpr int kMaxSplits = 8;                     // CTAs of a cluster
constexpr int kSmem = 226 * 1024;
constexpr int kOwn = 14 * 1024;                   // of it, at most, a kernel's own
constexpr int kPairStages = 6;
constexpr int kPairSlots = kPairStages + 2;
constexpr int kPairBatch = 2;                     // blocks of K that a warp brings in at a time
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
  int wide;                                       // plain: y's rows are 16-byte aligned
  int quarters, stages, x_bytes, ahead;           // stream: 32-row quarters that a tile can have, stages, bytes of a stage's tokens, stages filled early
  int splits;                                     // stream, dense: shares of K that a tile is cut into
  int over;                                       // of a cluster: its sums are exchanged where the stages were
  int most;                                       // column groups that a CTA finishes at most,
  uint8_t first[kMaxSplits + 1], owner[16];       // the first of 16 that each finishes, which CTA finishes each
};

__device__ __forceinline__ uint32_t s_addr(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) { asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count)); }
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// On a barrier of the pair's leader.  What it tells is that tensor memory has been read (tcgen05.wait::ld, the fence before), or that factors are on their way (Told
// publishes them): nothing in memory is published, and a release for the whole cluster is a fence every block of K (2048 x 9472 x 4096: 194 us with it by those
// that add up, 85 with it by those that bring in, 66.5 without).
__device__ __forceinline__ void bar_arrive_at(uint32_t bar) { asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory"); }
// The same by lane 0 of a warp, without a branch that the other lanes would have to wait behind (2 % of a block of K).
__device__ __forceinline__ void bar_arrive_lane0(uint32_t bar, int lane) {
  asm volatile("{\n.reg .pred p;\nsetp.eq.s32 p, %1, 0;\n@p mbarrier.arrive.shared::cluster.b64 _, [%0];\n}" ::"r"(bar), "r"(lane) : "memory");
}
// A barrier for each slot of a ring: who fills a slot tells the readers, all in its own CTA.  (The pair's stages go to the leader's threads and back; what the other CTA
// stores would have to be released to the cluster on that way.)
struct Told {
  uint32_t bars;
  __device__ __forceinline__ void init(int slots) const { for (int s = 0; s < slots; ++s) bar_init(bars + 8u * s, 1); }
  __device__ __forceinline__ void tell(int slot) const { asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bars + 8u * slot) : "memory"); }
  __device__ __forceinline__ void wait(int slot, uint32_t phase) const { mbar_wait(bars + 8u * slot, phase); }
  __device__ __forceinline__ bool test(int slot, uint32_t phase) const { return mbar_test(bars + 8u * slot, phase); }
};
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
__device__ __forceinline__ void tmem_ld(uint32_t at, uint32_t (&r)[32]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]),
               "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]),
               "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
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

// Which rows and tiles the groups have, in shared memory: starts[e] = tiles of the groups before e, near[e] = {first row, behind the last}.
template <int GROUPS>
struct Groups {
  int starts[GROUPS + 1];
  int2 near[GROUPS < kNearGroups ? GROUPS : kNearGroups];
};
// Rows of group e, whatever the table of offsets holds.
__device__ __forceinline__ int2 rows_of(const Fp8Params& p, int e) {
  if (!p.offsets) return make_int2(0, p.T);
  const int r0 = min(max(p.offsets[e], 0), p.T);
  return make_int2(r0, max(r0, min(p.offsets[e + 1], p.T)));
}
// Fills them, by all threads of the CTA.
template <int GROUPS>
__device__ __forceinline__ void count_tiles(const Fp8Params& p, int tile_rows, Groups<GROUPS>& groups) {
  int* starts = groups.starts;
  for (int e = threadIdx.x; e < p.E; e += kThreads) {
    const int2 r = rows_of(p, e);
    starts[e] = (r.y - r.x + tile_rows - 1) / tile_rows * p.n_tiles;
    if (e < kNearGroups) groups.near[e] = r;
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
// A value that all lanes of a converged warp have, so that the compiler knows it: what comes out of shared memory it takes for different in each (gated 8192 x
// 28672 x 4096 802 us without, 796 with, both before what gated results cost now).
__device__ __forceinline__ int same(int v) { return __shfl_sync(0xffffffffu, v, 0); }
__device__ __forceinline__ Tile same(const Tile& t) { return Tile{same(t.e), same(t.n), same(t.row), same(t.rows)}; }
// From a tile's number; the group is looked for from `e` on (numbers come in rising order).  Tiles of a group run over BAND token tiles (0: all), then
// the next column tile: neighbours share weights, and a band's tokens stay in the L2 meanwhile.
template <int TILE_ROWS, int BAND, int GROUPS>
__device__ __forceinline__ Tile find_tile(const Fp8Params& p, const Groups<GROUPS>& groups, int tile, int& e) {
  while (e + 1 < p.E && tile >= groups.starts[e + 1]) ++e;
  const int2 r = e < (GROUPS < kNearGroups ? GROUPS : kNearGroups) ? groups.near[e] : rows_of(p, e);
  const int m_tiles = (r.y - r.x + TILE_ROWS - 1) / TILE_ROWS, local = tile - groups.starts[e];
  Tile t;
  t.e = e;
  int m = 0;
  if (m_tiles == 1) {
    t.n = local;
  } else {
    const int band = BAND ? BAND : m_tiles, g = BAND ? local / (band * p.n_tiles) : 0, first = g * band, width = min(band, m_tiles - first), in = local - g * band * p.n_tiles;
    t.n = in / width;
    m = first + in - t.n * width;
  }
  t.row = r.x + m * TILE_ROWS;
  t.rows = min(TILE_ROWS, r.y - t.row);
  return t;
}
template <int GROUPS>
__device__ __forceinline__ int first_group(const Fp8Params& p, const Groups<GROUPS>& groups, int tile) {
  int lo = 0, hi = p.E - 1;
  while (lo < hi) { const int mid = (lo + hi + 1) / 2; if (groups.starts[mid] <= tile) lo = mid; else hi = mid - 1; }
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
  // += factor * D of N columns at c, two an instruction (the pipe does as many without, but takes more power: 8192 x 4096 x 14336 over and over 453 and 441 us)
  template <int N>
  __device__ __forceinline__ void add(int c, const uint32_t (&r)[N], float factor) {
#pragma unroll
    for (int i = 0; i < N; i += 2)
      asm volatile("{\n.reg .b64 a, b, d;\nmov.b64 a, {%2, %3};\nmov.b64 b, {%4, %4};\nmov.b64 d, {%0, %1};\nfma.rn.f32x2 d, a, b, d;\nmov.b64 {%0, %1}, d;\n}"
                   : "+f"(v[c + i]), "+f"(v[c + i + 1]) : "f"(__uint_as_float(r[i])), "f"(__uint_as_float(r[i + 1])), "f"(factor));
  }
  __device__ __forceinline__ void at(int c, float& a, float& b) const { a = v[c]; b = v[c + 1]; }
};

// Adds up `blocks` blocks of K.  wait(): the address of the next block's columns in tensor memory and its factors, when they are there; read(): they are
// in registers.  A thread's second 64 columns (if it has them) lie SKIP columns behind its first, with a factor of their own.  The next block is waited
// for, and its first columns asked for, before the last ones of this block are added, so that the way to tensor memory and back passes under arithmetic.
// (All 64 columns of threads that have no more at once: 4096 x 14336, one token, 15.6 us against 14.8.)
template <int C, int SKIP, typename W, typename R>
__device__ __forceinline__ void add_blocks(Sums<C>& s, int blocks, W wait, R read) {
  constexpr int N = 32;
  uint32_t r[2][N], at;
  float f0, f1;
  wait(at, f0, f1);
  tmem_ld(at, r[0]);
#pragma unroll 1
  for (; blocks > 0; --blocks) {
    const float g0 = f0, g1 = f1;
#pragma unroll
    for (int c = 0; c < C; c += N) {
      uint32_t (&now)[N] = r[(c / N) & 1], (&then)[N] = r[(c / N + 1) & 1];
      tmem_wait_ld(now);
      if (c + N < C) {
        tmem_ld(at + c + N + (c + N >= 64 ? SKIP : 0), then);
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

// silu(gate) up = gate up / (1 + p^2), times p^2 where the gate is negative, with p = e^(-|gate| / 2) by the unit's own power of two: neither p^2 nor its reciprocal,
// which leave the range of fp32 beyond 87, stands alone.  What the exponent's rounding and that of log2(e) / 2 leave is put back, so down to gates of -174 a result
// that fp32 holds as a normal number is off by 2^-20 of it at most: p, which counts twice, 2^-22.5 and a rounding, the reciprocal 2^-23, a sum and four products a rounding each.
// (With e^-gate and its reciprocal, half the instructions, prompts take as long: 8192 x 28672 x 4096 776 us and 770.)
__device__ __forceinline__ float gated(float gate, float up) {
  constexpr float c = -0.721347511f, rest = -6.6749e-9f;              // c + rest / ln 2 = -log2(e) / 2
  const float g = fabsf(gate), t = g * c, off = fmaf(fmaf(g, c, -t), 0.693147181f, g * rest);
  float p, inv;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(p) : "f"(t));
  p = fmaf(p, off, p);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inv) : "f"(fmaf(p, p, 1.f)));
  if (gate < 0.f) { gate *= p; up *= p; }
  return gate * inv * up;
}

// 64 columns of a row from n0 on, rounded once, where its rows are 16-byte aligned; c0: where their sums begin.
template <int C>
__device__ __forceinline__ void store_row(const Fp8Params& p, const Sums<C>& s, int c0, int row, int n0) {
  bf16* dst = p.y + (int64_t)row * p.N + n0;
#pragma unroll
  for (int c = c0; c < c0 + 64; c += 8)
    if (n0 + c - c0 < p.N)
      *reinterpret_cast<uint4*>(dst + c - c0) = make_uint4(pack_bf2(s.v[c], s.v[c + 1]), pack_bf2(s.v[c + 2], s.v[c + 3]), pack_bf2(s.v[c + 4], s.v[c + 5]), pack_bf2(s.v[c + 6], s.v[c + 7]));
}

// The bias of SETS x 64 columns, SKIP apart, from n0 (even) on to a warp's own words in shared memory, two columns a word: asked for when a tile begins, there
// when it ends.  (Loads by each thread when it ends, 9472 x 4096 x 1408: 18 us of 74.)
template <int SETS, int SKIP>
__device__ __forceinline__ void ask_bias(const Fp8Params& p, uint32_t* own, int n0, int lane) {
#pragma unroll
  for (int h = 0; h < SETS; ++h) {
    const int n = n0 + h * SKIP + 2 * lane, left = min(max(p.N - n, 0), 2);
    const bf16* src = p.bias + (left ? n : 0);
    uint32_t* dst = own + h * 32 + lane;
    if ((reinterpret_cast<uintptr_t>(p.bias) & 3) == 0) {
      asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(s_addr(dst)), "l"(src), "r"(2 * left) : "memory");
    } else {
      uint32_t v = 0;
      if (left > 0) v = *reinterpret_cast<const uint16_t*>(src);
      if (left > 1) v |= (uint32_t)*reinterpret_cast<const uint16_t*>(src + 1) << 16;
      *dst = v;
    }
  }
}
template <int C>
__device__ __forceinline__ void add_bias(Sums<C>& s, const uint32_t* own) {
  asm volatile("cp.async.wait_all;" ::: "memory");
  __syncwarp();
#pragma unroll
  for (int c = 0; c < C; c += 8) {
    const uint4 b = *reinterpret_cast<const uint4*>(own + c / 2);
    s.v[c] += bf_lo(b.x); s.v[c + 1] += bf_hi(b.x); s.v[c + 2] += bf_lo(b.y); s.v[c + 3] += bf_hi(b.y);
    s.v[c + 4] += bf_lo(b.z); s.v[c + 5] += bf_hi(b.z); s.v[c + 6] += bf_lo(b.w); s.v[c + 7] += bf_hi(b.w);
  }
  __syncwarp();
}

// Rows that are not 16-byte aligned: a warp's 32 rows (from `row` on, `rows` of them there) of C columns, the second 64 of them SKIP behind the first.  8 rows
// of 64 columns at a time go through shared memory, in words as memory has them: a row that begins in the middle of a word has its columns one half further.
// A row's whole words go out at once, and the halves at its ends, of 8 rows at once: what is written piece by piece costs the L2 by the piece (from registers,
// a column of 32 rows at a time, 2048 x 4095 x 4096 took 105 us; 16 columns of two rows at a time 43).
constexpr int kNarrowRow = 144, kNarrow = 8 * kNarrowRow;      // bytes of a row (33 words, and none that meets another row's in a bank) and of a warp
template <int C, int SKIP>
__device__ __forceinline__ void store_narrow(const Fp8Params& p, const Sums<C>& s, int row, int rows, int n0, uint32_t buffer, int lane) {
  auto at = [&](int r, int n) { return reinterpret_cast<uint16_t*>(p.y) + (int64_t)(row + r) * p.N + n; };
  auto is_odd = [](const uint16_t* dst) { return (int)(reinterpret_cast<uintptr_t>(dst) >> 1) & 1; };
#pragma unroll
  for (int c0 = 0; c0 < C; c0 += 64) {
    const int n = n0 + c0 / 64 * SKIP, columns = min(p.N - n, 64);
    if (columns <= 0) break;
    uint32_t u[33];
    const bool half = is_odd(at(lane, n));
    u[0] = pack_bf2(half ? 0.f : s.v[c0], half ? s.v[c0] : s.v[c0 + 1]);
#pragma unroll
    for (int w = 1; w < 32; ++w) u[w] = pack_bf2(half ? s.v[c0 + 2 * w - 1] : s.v[c0 + 2 * w], half ? s.v[c0 + 2 * w] : s.v[c0 + 2 * w + 1]);
    u[32] = pack_bf2(s.v[c0 + 63], 0.f);
#pragma unroll 1
    for (int g = 0; g < 32 && g < rows; g += 8) {
      __syncwarp();
      if ((lane & 24) == g) {
        const uint32_t put = buffer + (lane & 7) * kNarrowRow;
#pragma unroll
        for (int k = 0; k < 8; ++k) asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(put + k * 16), "r"(u[4 * k]), "r"(u[4 * k + 1]), "r"(u[4 * k + 2]), "r"(u[4 * k + 3]) : "memory");
        asm volatile("st.shared.b32 [%0], %1;" ::"r"(put + 128), "r"(u[32]) : "memory");
      }
      __syncwarp();
      uint32_t v[8];
#pragma unroll
      for (int r = 0; r < 8; ++r) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v[r]) : "r"(buffer + r * kNarrowRow + lane * 4) : "memory");
#pragma unroll
      for (int r = 0; r < 8; ++r) {
        uint16_t* dst = at(g + r, n);
        const int c = 2 * lane - is_odd(dst);
        if (g + r < rows && c >= 0 && c + 1 < columns) *reinterpret_cast<uint32_t*>(dst + c) = v[r];
      }
      // the first column of a row that begins in a word's middle; the last of one that ends there
      const int r = (lane >> 1) & 7, c = lane & 1 ? columns - 1 : 0;
      uint16_t* dst = at(g + r, n);
      const int odd = is_odd(dst);
      if (lane < 16 && g + r < rows && ((c + odd) & 1) == 1 - (lane & 1)) {
        uint16_t e;
        asm volatile("ld.shared.u16 %0, [%1];" : "=h"(e) : "r"(buffer + r * kNarrowRow + (c + odd) * 2) : "memory");
        dst[c] = e;
      }
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
        u[i] = pack_bf2(s.v[c], s.v[c + 1]);
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
      h[c + i] = gated(g[i], u[i]);
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
  const fp8::Rows32 rows(__uint_as_float(m), factor);
  uint8_t* dst = p.codes + (int64_t)row * p.N + n * 128 + part * H;
  uint32_t marked = 0;
#pragma unroll
  for (int c = 0; c < H; c += 16) {
    uint32_t q[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = factor > 0.f ? rows.codes4(h[c + 4 * i], h[c + 4 * i + 1], h[c + 4 * i + 2], h[c + 4 * i + 3], marked, c / 4 + i) : 0u;
    *reinterpret_cast<uint4*>(dst + c) = make_uint4(q[0], q[1], q[2], q[3]);
  }
  for (; marked; marked &= marked - 1) {                         // (in place, 16 times unrolled: 71 us where this takes 66, 15 groups of 889 x 1792 x 768)
    const int at = __ffs(marked) - 1;
    float a = h[0], b = h[1], c = h[2], d = h[3];
#pragma unroll
    for (int j = 1; j < H / 4; ++j)
      if (j == at) { a = h[4 * j]; b = h[4 * j + 1]; c = h[4 * j + 2]; d = h[4 * j + 3]; }
    *reinterpret_cast<uint32_t*>(dst + 4 * at) = rows.settled4(a, b, c, d);
  }
  if (part == 0) p.out_scales[n * p.out_stride + row] = scale;
}

// -------------------------------------------------------------------------------------------------- tiles by single CTAs

// What a CTA does: blocks of K [kb0, kb1) of tiles [tile0, tile1).  With at least half as many tiles as SMs each is one CTA's, and as many CTAs work as make
// all have the same number (a weight stream needs bytes under way, not SMs); fewer are cut along K, into `splits` shares: of groups, where that saves more than
// the way through the workspace costs, 5 us (gated 8).  us cut and whole: 16 rows in 8 groups of 1024 x 1024 8.8 and 5.9, 8 of 2048 x 4096 15.2 and 15.1, of 1024 x
// 6144 14.4 and 15.7, 2 of 2048 x 14336 18.6 and 29.7; gated 256 x 1024 12.2 and 8.6, 256 x 3200 18.2 and 16.2, 1024 x 6144 20.4 and 25.3.
struct Work { int tile0, tile1, kb0, kb1, splits; };
// Blocks of K of a stage: the thread that issues the MMAs takes some 600 cycles from one pair of barriers to the next, and tiles of 128 columns have their
// data in 370; besides, boxes of 128 bytes a row are read at 5.7 TB/s and two neighbouring ones at 6.35.
__host__ __device__ constexpr int stream_sub(int nt) { return nt == 128 ? 2 : 1; }
__device__ __forceinline__ Work work_of(int tiles, int KB, int splits, int me, int sms) {
  if (splits == 0) splits = tiles == 0 || 2 * tiles >= sms || KB <= 32 ? 1 : max(1, min(min(sms / tiles, KB / 2), kMaxSplits));
  if (splits > 1) {
    const int tile = me / splits, piece = me - tile * splits;
    if (tile >= tiles) return Work{0, 0, 0, 0, splits};
    return Work{tile, tile + 1, KB * piece / splits, KB * (piece + 1) / splits, splits};
  }
  const int rounds = (tiles + sms - 1) / sms;
  if (rounds <= 1) return me < tiles ? Work{me, me + 1, 0, KB, 1} : Work{0, 0, 0, 0, 1};
  const int ctas = (tiles + rounds - 1) / rounds;
  if (me >= ctas) return Work{0, 0, 0, 0, 1};
  const int each = tiles / ctas, more = tiles - each * ctas;
  return Work{each * me + min(me, more), each * (me + 1) + min(me + 1, more), 0, KB, 1};
}

__device__ __forceinline__ void copy4(uint32_t dst, const float* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void push4(uint32_t dst, float a, float b, float c, float d) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst), "f"(a), "f"(b), "f"(c), "f"(d) : "memory");
}

__device__ __forceinline__ float4 lds4(uint32_t at) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(at) : "memory");
  return v;
}

__device__ __forceinline__ float lds1(uint32_t at) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
  return v;
}

// CLUSTER: the shares of a tile are a cluster's CTAs.  Each finishes its part of the tile's columns, groups of 8, and gets the others' sums of them through
// distributed shared memory; they are added in the order of K, so the result's bits are the same each time.
// Otherwise shares (of grouped rows, whose number of tiles the host does not know) go through the workspace: the last to arrive adds them, in that order too.
// Bound by the weights' way from memory, and at one or two tiles a CTA by what is before and behind it: about 2 us from the launch to the first bytes and 2
// to 3 for the last tile's sums, exchange and stores.  64 tokens: eight each of 128 experts, gated 1536 x 2048 (376 MB) 70.4 us, 5.3 TB/s; gated 28672 x 4096
// (119 MB) 25.5 us; 6144 x 4096 (26 MB) 10.8 us; one token, 4096 x 14336 (59 MB) 14.4 us.
template <int NT, bool GATED, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, 1)
fp8_stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Fp8Params p) {
  constexpr int C = NT / 2, SUB = stream_sub(NT), BUFS = 512 / (NT * SUB), SETS = NT / 128, SLOT = kSlotBytes / 4;
  static_assert(!GATED || NT == 256, "a gated tile holds 128 columns of each");
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * kMaxStages + 2 * BUFS];
  __shared__ uint32_t tmem_slot;
  __shared__ int last_flag;
  __shared__ uint32_t tops[GATED ? (CLUSTER ? 1 + kMaxSplits : 2) * 128 : 1];
  __shared__ __align__(16) uint32_t biases[GATED ? 4 : kSumWarps * 64];       // of each warp that adds up; of all columns
  __shared__ Groups<CLUSTER ? 1 : kMaxGroups> groups;
  const int stages = p.stages;
  const uint32_t block_bytes = (uint32_t)p.x_bytes + NT * 128, stage_bytes = SUB * block_bytes;
  const uint32_t base = s_addr(smem), bar0 = s_addr(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (kMaxStages + s); };
  auto tfull = [&](int b) { return bar0 + 8u * (2 * kMaxStages + b); };
  auto tempty = [&](int b) { return bar0 + 8u * (2 * kMaxStages + BUFS + b); };
  const int warp = uniform_warp(), lane = threadIdx.x & 31;

  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < stages; ++s) { bar_init(full(s), 33); bar_init(empty(s), 1); }      // (full: the tiles' copies, the factors' by 32 lanes)
    for (int b = 0; b < BUFS; ++b) { bar_init(tfull(b), 1); bar_init(tempty(b), kSumWarps); }
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  if (CLUSTER && GATED && threadIdx.x < 128) tops[threadIdx.x] = 0;
  if ((CLUSTER || !p.offsets) && threadIdx.x == 0) { groups.starts[0] = 0; groups.near[0] = make_int2(0, p.T); groups.starts[1] = (p.T + kRows - 1) / kRows * p.n_tiles; }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_launch_dependents();
  if (CLUSTER && !p.over) cluster_arrive_relaxed();
  if (!CLUSTER && p.offsets) {                      // which tiles there are is the kernel before's output
    pdl_wait();
    count_tiles(p, kRows, groups);
  }
  const int KB = p.KB;
  const Work work = work_of(same(groups.starts[p.E]), KB, p.splits, (int)blockIdx.x, (int)gridDim.x);
  const int e_first = work.tile0 < work.tile1 ? first_group(p, groups, work.tile0) : 0;
  // xs of the rows and ws of the columns, block of K by block of K, in a ring.  A slot is free again when its block is added up.  The block `stages` further
  // is then at the earliest on its way (its stage was freed by an MMA that began after the sums BUFS blocks before had been read).
  float* factors = reinterpret_cast<float*>(smem + stages * stage_bytes);
  const int slots = (stages + BUFS) * SUB;

  if (warp == 0) {
    regs_down<kOtherRegs>();
    if (elect_one()) {
      int stage = 0, e = e_first;
      uint32_t phase = 0;
      auto load_w = [&](int s, const Tile& t, int kb, int n) {
        const int row = t.e * p.w_rows;
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          if (u >= n) break;
          const uint32_t dst = base + s * stage_bytes + u * block_bytes + p.x_bytes;
#pragma unroll
          for (int h = 0; h < NT / 128; ++h) load_box(dst + h * kSlab, &map_w, full(s), (kb + u) * 128, row + (GATED ? t.n * 128 + h * p.N : t.n * NT + h * 128));
        }
      };
      auto load_x = [&](int s, const Tile& t, int kb, int n) {
        for (int u = 0; u < n; ++u)
          for (int r = 0; r < t.rows; r += 32) load_box(base + s * stage_bytes + u * block_bytes + r * 128, &map_x, full(s), (kb + u) * 128, t.row + r);
      };
      auto bytes_of = [&](const Tile& t, int n) { return (uint32_t)(n * (NT * 128 + (t.rows + 31) / 32 * 4096)); };
      // What the weights are is known before the kernel before has ended: the first tile's first blocks.
      int ahead = 0;
      if ((CLUSTER || !p.offsets) && work.tile0 < work.tile1) {
        const Tile t = find_tile<kRows, 0>(p, groups, work.tile0, e);
        for (int kb = work.kb0; ahead < p.ahead && kb < work.kb1; kb += SUB, ++ahead) {
          const int n = min(SUB, work.kb1 - kb);
          bar_expect(full(ahead), bytes_of(t, n));
          load_w(ahead, t, kb, n);
        }
      }
      pdl_wait();
      for (int tile = work.tile0; tile < work.tile1; ++tile) {
        const Tile t = find_tile<kRows, 0>(p, groups, tile, e);
        for (int kb = work.kb0; kb < work.kb1; kb += SUB) {
          const int n = min(SUB, work.kb1 - kb);
          if (ahead > 0) {
            --ahead;
          } else {
            mbar_wait(empty(stage), phase ^ 1);
            bar_expect(full(stage), bytes_of(t, n));
            load_w(stage, t, kb, n);
          }
          load_x(stage, t, kb, n);
          if (++stage == stages) { stage = 0; phase ^= 1; }
        }
      }
    }
  } else if (warp == 1) {
    regs_down<kOtherRegs>();
    pdl_wait();                                     // (nothing is there to multiply before; a wait at a barrier, limited in time, would span what is left of the kernel before)
    if (elect_one()) {
      constexpr uint32_t idesc = instr_desc(kRows, NT);
      int stage = 0, buf = 0;
      uint32_t phase = 0, buf_phase = 0;
      const uint64_t a0 = tile_desc(base), b0 = tile_desc(base + p.x_bytes);
      uint64_t a = a0, b = b0;
      bool f_there = false, t_there = false;
      for (int tile = work.tile0; tile < work.tile1; ++tile)
        for (int kb = work.kb0; kb < work.kb1; kb += SUB) {
          if (!f_there) mbar_wait(full(stage), phase);
          if (!t_there) mbar_wait(tempty(buf), buf_phase ^ 1);
          const int s1 = stage + 1 == stages ? 0 : stage + 1, v1 = buf + 1 == BUFS ? 0 : buf + 1;
          const uint32_t p1 = s1 == 0 ? phase ^ 1 : phase, w1 = v1 == 0 ? buf_phase ^ 1 : buf_phase;
          f_there = mbar_test(full(s1), p1);
          t_there = mbar_test(tempty(v1), w1 ^ 1);
          fence_after();
          const uint32_t d = tmem + buf * (NT * SUB);
#pragma unroll
          for (int u = 0; u < SUB; ++u) {
            if (u > 0 && kb + u >= work.kb1) break;
            const uint64_t off = (uint64_t)(u * (block_bytes >> 4));
#pragma unroll
            for (int k = 0; k < 4; ++k) mma8(d + u * NT, a + off + 2 * k, b + off + 2 * k, idesc, k > 0);
          }
          commit(tfull(buf));
          commit(empty(stage));
          a += stage_bytes >> 4; b += stage_bytes >> 4;
          if (s1 == 0) { a = a0; b = b0; }
          stage = s1; phase = p1; buf = v1; buf_phase = w1;
        }
    }
  } else if (warp == 2) {
    regs_down<kOtherRegs>();
    int stage = 0, slot = 0, e = e_first;
    uint32_t phase = 0;
    auto column = [&](const Tile& t, int kb) {           // of a tile's ws: lanes 0 (and 1) have a block of its columns each
      const int64_t block = (int64_t)t.e * p.w_blocks + (GATED ? t.n + lane * (p.N / 128) : min(t.n * SETS + lane, p.w_blocks - 1));
      return p.ws + block * p.KB + kb;
    };
    auto to = [&](int s, int i) { return s_addr(factors + s * SLOT + i); };
    int early = 0;
    if ((CLUSTER || !p.offsets) && work.tile0 < work.tile1) {
      const Tile t = same(find_tile<kRows, 0>(p, groups, work.tile0, e));
      early = min(p.ahead * SUB, work.kb1 - work.kb0);
      for (int i = 0; i < early; ++i)
        if (lane < SETS) copy4(to(i, 128 + lane), column(t, work.kb0 + i), true);
    }
    pdl_wait();
    for (int tile = work.tile0; tile < work.tile1; ++tile) {
      const Tile t = same(find_tile<kRows, 0>(p, groups, tile, e));
      const float* xs = p.xs + work.kb0 * p.xs_stride + t.row + lane;
      const float* ws = column(t, work.kb0);
      for (int kb = work.kb0; kb < work.kb1; kb += SUB) {
        mbar_wait(empty(stage), phase ^ 1);
#pragma unroll
        for (int u = 0; u < SUB; ++u) {
          if (kb + u < work.kb1) {
            for (int q = 0; q * 32 < t.rows; ++q) {
              const bool there = q * 32 + lane < t.rows;
              copy4(to(slot + u, q * 32 + lane), there ? xs + q * 32 : p.xs, there);
            }
            if (early > 0) --early;
            else if (lane < SETS) copy4(to(slot + u, 128 + lane), ws, true);
            xs += p.xs_stride;
            ++ws;
          }
        }
        asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full(stage)) : "memory");
        if (++stage == stages) { stage = 0; phase ^= 1; }
        if ((slot += SUB) == slots) slot = 0;
      }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
  } else if (warp == 3) {
    regs_down<kOtherRegs>();
    if constexpr (CLUSTER && !GATED) {               // (the others see it behind the cluster's barriers)
      if (p.bias) {
        pdl_wait();
        int e = 0;
        ask_bias<NT / 64, 64>(p, biases, find_tile<kRows, 0>(p, groups, work.tile0, e).n * NT, lane);
        asm volatile("cp.async.wait_all;" ::: "memory");
      }
    }
  } else {
    regs_up<kSumRegs>();
    const int q = warp & 3, part = (warp - 4) >> 2, tid = threadIdx.x - 128, lane128 = q * 32 + lane;
    pdl_wait();
    int buf = 0, slot = 0, e = e_first;
    uint32_t buf_phase = 0;
    for (int tile = work.tile0; tile < work.tile1; ++tile) {
      const Tile t = same(find_tile<kRows, 0>(p, groups, tile, e));
      const bool some = q * 32 < t.rows, there = lane128 < t.rows;
      const int row = t.row + lane128, n0 = t.n * NT + part * 64;
      Sums<C> s;
      s.clear();
      uint32_t* own = biases + (GATED ? 0 : (warp - 4) * 64);
      if (!GATED && !CLUSTER && p.bias) ask_bias<C / 64, 128>(p, own, n0, lane);
      const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + part * 64;
      int sub = 0, left = work.kb1 - work.kb0;
      auto read = [&] {
        if (--left == 0 || ++sub == SUB) {
          sub = 0;
          fence_before();
          bar_arrive_lane0(tempty(buf), lane);
          if (++buf == BUFS) { buf = 0; buf_phase ^= 1; }
          if ((slot += SUB) == slots) slot = 0;
        }
      };
      auto wait = [&](uint32_t& from, float& f0, float& f1) {
        if (SUB == 1 || sub == 0) {
          mbar_wait(tfull(buf), buf_phase);
          fence_after();
        }
        const float* f = factors + (slot + sub) * SLOT;
        f0 = f[lane128] * f[128];
        f1 = SETS == 2 ? f[lane128] * f[129] : f0;
        from = at + buf * (NT * SUB) + sub * NT;
      };
      if (some) {
        add_blocks<C, 64>(s, left, wait, read);
      } else {
        while (left > 0) {
          if (sub == 0) mbar_wait(tfull(buf), buf_phase);
          read();
        }
      }
      if constexpr (CLUSTER) {
        // Groups of 8 columns of each set: this CTA finishes [g0, g1) of 16.  Their sums lie there by sender, set, group, half and row, 16 bytes each; each is
        // finished by a lane of its row.  (Everything here runs once a launch and costs its way from the L2: rolled loops, and all sums by one path.)
        const int S = work.splits, me = (int)cluster_ctarank(), rows = p.quarters * 32, most = p.most;
        const uint32_t sums = p.over ? base : s_addr(factors + slots * SLOT);
        auto place = [&](int sender, int set, int g, int half, int r) { return sums + (uint32_t)((((sender * SETS + set) * most + g) * 2 + half) * rows + r) * 16u; };
        if (p.over) cluster_arrive();
        cluster_wait();                                   // (all have begun; or their MMAs have read what the sums are laid over)
        if (some) {
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const int g = part * 8 + i, owner = p.owner[g];
            const uint32_t to = mapa_u32(place(me, 0, g - p.first[owner], 0, lane128), owner);
#pragma unroll
            for (int set = 0; set < SETS; ++set)
#pragma unroll
              for (int half = 0; half < 2; ++half) {
                const float* v = &s.v[set * 64 + i * 8 + half * 4];
                push4(to + (uint32_t)((set * most * 2 + half) * rows) * 16u, v[0], v[1], v[2], v[3]);
              }
          }
        }
        cluster_arrive(); cluster_wait();
        const int g0 = p.first[me], mine = p.first[me + 1] - g0, items = mine * p.quarters;
        auto item = [&](int n, int& r, int& g) {          // a warp's n-th quarter of the rows and group
          g = n / p.quarters;
          r = (n - g * p.quarters) * 32 + lane;
        };
        auto sum_of = [&](int set, int g, int r, float (&v)[8]) {
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = 0.f;
#pragma unroll 1
          for (int from = 0; from < S; ++from)
#pragma unroll
            for (int half = 0; half < 2; ++half) {
              const float4 f = lds4(place(from, set, g, half, r));
              v[half * 4] += f.x; v[half * 4 + 1] += f.y; v[half * 4 + 2] += f.z; v[half * 4 + 3] += f.w;
            }
        };
        if (!GATED && !p.wide) {
          // rows that are not 16-byte aligned: four rows of a group at a time, a column a lane
          const int j = lane & 7;
#pragma unroll 1
          for (int r = (warp - 4) * 4 + (lane >> 3); r < t.rows; r += 4 * kSumWarps)
#pragma unroll 1
            for (int g = 0; g < mine; g += 4) {      // (reading beyond the last group, but not beyond what lies there)
              const int c = (g0 + g) * 8 + j;
              const uint32_t from0 = place(0, 0, g, j >> 2, r) + (j & 3) * 4, group = 2 * rows * 16, sender = SETS * most * group;
              float v[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 1
              for (int from = 0; from < S; ++from)
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += lds1(from0 + from * sender + min(k, most - 1 - g) * group);
              bf16* dst = p.y + (int64_t)(t.row + r) * p.N + t.n * NT + c;
#pragma unroll
              for (int k = 0; k < 4; ++k)
                if (g + k < mine && t.n * NT + c + 8 * k < p.N) dst[8 * k] = f2bf(p.bias ? v[k] + bf2f(reinterpret_cast<const bf16*>(biases)[c + 8 * k]) : v[k]);
            }
        } else
#pragma unroll 1
        for (int n = warp - 4; n < items; n += kSumWarps) {
          int r, g;
          item(n, r, g);
          float v[8];
          sum_of(0, g, r, v);
          if constexpr (GATED) {
            float u[8];
            sum_of(1, g, r, u);
            uint32_t top = 0;
#pragma unroll
            for (int j = 0; j < 8; ++j) {
              v[j] = gated(v[j], u[j]);
              top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
            }
            atomicMax(&tops[r], top);
            push4(mapa_u32(place(0, 0, g, 0, r), me), v[0], v[1], v[2], v[3]);      // (in the place of the first sender's sums)
            push4(mapa_u32(place(0, 0, g, 1, r), me), v[4], v[5], v[6], v[7]);
          } else if (r < t.rows && t.n * NT + (g0 + g) * 8 < p.N) {
            if (p.bias) {
              const uint4 b = *reinterpret_cast<const uint4*>(biases + (g0 + g) * 4);
              v[0] += bf_lo(b.x); v[1] += bf_hi(b.x); v[2] += bf_lo(b.y); v[3] += bf_hi(b.y);
              v[4] += bf_lo(b.z); v[5] += bf_hi(b.z); v[6] += bf_lo(b.w); v[7] += bf_hi(b.w);
            }
            *reinterpret_cast<uint4*>(p.y + (int64_t)(t.row + r) * p.N + t.n * NT + (g0 + g) * 8) =
                make_uint4(pack_bf2(v[0], v[1]), pack_bf2(v[2], v[3]), pack_bf2(v[4], v[5]), pack_bf2(v[6], v[7]));
          }
        }
        if constexpr (GATED) {
          // the block's largest magnitude over all CTAs
          sums_sync();
          if (tid < 128)
#pragma unroll 1
            for (int to = 0; to < S; ++to)
              asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(mapa_u32(s_addr(&tops[(1 + me) * 128 + tid]), to)), "r"(tops[tid]) : "memory");
          cluster_arrive(); cluster_wait();
#pragma unroll 1
          for (int n = warp - 4; n < items; n += kSumWarps) {
            int r, g;
            item(n, r, g);
            uint32_t top = 0;
            for (int c = 1; c <= S; ++c) top = max(top, tops[c * 128 + r]);
            float scale, factor;
            fp8::scale_of(__uint_as_float(top), scale, factor);
            const float4 a = lds4(place(0, 0, g, 0, r)), b = lds4(place(0, 0, g, 1, r));
            uint2 c = make_uint2(0, 0);
            if (factor > 0.f) {
              const fp8::Rows32 row(__uint_as_float(top), factor);
              uint32_t marked = 0;
              c.x = row.codes4(a.x, a.y, a.z, a.w, marked, 0);
              c.y = row.codes4(b.x, b.y, b.z, b.w, marked, 1);
              if (marked & 1) c.x = row.settled4(a.x, a.y, a.z, a.w);
              if (marked & 2) c.y = row.settled4(b.x, b.y, b.z, b.w);
            }
            if (r < t.rows) {
              *reinterpret_cast<uint2*>(p.codes + (int64_t)(t.row + r) * p.N + t.n * 128 + (g0 + g) * 8) = c;
              if (me == 0 && g == 0) p.out_scales[t.n * p.out_stride + t.row + r] = scale;
            }
          }
        }
      } else {
        if (work.splits > 1) {
          // To the workspace, [CTA][quarter][part][column / 4][lane] of 16 bytes.
          constexpr int kPer = (NT / 4) * 32;          // float4 of a quarter
          auto share_of = [&](int cta) { return reinterpret_cast<float4*>(p.part) + ((int64_t)cta * p.quarters + q) * kPer + part * (C / 4) * 32 + lane; };
          if (some) {
            float4* dst = share_of((int)blockIdx.x);
#pragma unroll
            for (int c = 0; c < C; c += 4) __stcg(dst + c / 4 * 32, make_float4(s.v[c], s.v[c + 1], s.v[c + 2], s.v[c + 3]));
          }
          sums_sync();
          if (tid == 0) {
            __threadfence();                              // (of what all threads of the barrier have stored)
            const bool mine = atomicAdd(p.count + tile, 1u) == (unsigned)(work.splits - 1);
            if (mine) p.count[tile] = 0;                  // ready for the next launch
            __threadfence();
            last_flag = mine;
          }
          sums_sync();
          if (last_flag == 0) continue;                   // (a share is all that its CTA has)
          s.clear();
          if (some)
#pragma unroll
            for (int h = 0; h < C; h += 64)
              for (int c = tile * work.splits; c < (tile + 1) * work.splits; ++c) {
                const float4* src = share_of(c) + h / 4 * 32;
                float4 v[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __ldcg(src + i * 32);
#pragma unroll
                for (int i = 0; i < 16; ++i) { s.v[h + 4 * i] += v[i].x; s.v[h + 4 * i + 1] += v[i].y; s.v[h + 4 * i + 2] += v[i].z; s.v[h + 4 * i + 3] += v[i].w; }
              }
        }
        if constexpr (GATED) {
          store_gated(p, s, row, there, t.n, tops, part, lane128);
        } else {
          if (p.bias) add_bias<C>(s, own);
          if (!p.wide) {
            if (some) store_narrow<C, 128>(p, s, row - lane, t.rows - q * 32, n0, s_addr(factors + slots * SLOT) + (warp - 4) * kNarrow, lane);
          } else if (there) {
#pragma unroll
            for (int h = 0; h < C / 64; ++h) store_row<C>(p, s, h * 64, row, n0 + h * 128);
          }
        }
      }
    }
  }
  if (CLUSTER && warp < 4) {                        // the barriers that the others take, for all threads take part
    if (p.over) cluster_arrive();
    cluster_wait();
    cluster_arrive(); cluster_wait();
    if (GATED) { cluster_arrive(); cluster_wait(); }
  }
  fence_before();
  __syncthreads();
  if (warp == 2) {
    fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
}

// -------------------------------------------------------------------------------------------------------------- pairs

// A block of K is 32 KB of codes and 512 cycles of MMAs a CTA; its 128 x 256 sums are 256 cycles of the fp32 pipe.  Both run side by side: tensor memory holds
// two blocks, and the first and the second 128 columns of each are handed over apart, as soon as their four warps have read them.  Six stages and 2 KB a warp
// through which rows are stored; four stages and a whole tile stored by copies from shared memory took 410 us where this took 399.
// Bound by the power limit when it runs over and over, else by the 585 cycles that a block of K takes and by a tile's end (3000 cycles, gated 3900, under which
// two blocks of the next tile are multiplied).  8192 tokens: 4096 x 14336 377 us (2.5 PFLOP/s; over and over 450; copies and MMAs alone 334), gated 28672 x
// 4096 808 us (2.4 PFLOP/s; 938; 655).  12288 rows of 64 experts, 2048 x 1408 (253 MB): 69 us, gated 2816 x 2048 127 us.
template <bool GATED, bool WIDE>
__global__ void __launch_bounds__(kThreads, 1)
fp8_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const Fp8Params p) {
  constexpr int C = 128, STAGES = kPairStages;
  constexpr uint32_t kStage = 2 * kSlab;
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  __shared__ uint64_t bars[2 * STAGES + 8 + kPairSlots];
  __shared__ uint32_t tmem_slot;
  __shared__ uint32_t tops[GATED ? 256 : 1];
  __shared__ __align__(16) uint32_t biases[GATED ? 4 : kSumWarps * 64];       // of each warp that adds up
  __shared__ int4 tiles[16];                        // n, row, rows of the tiles under way: at most one a block of K of the rings, and the last one
  __shared__ Groups<kMaxGroups> groups;
  const uint32_t base = s_addr(smem), bar0 = s_addr(bars);
  auto full = [&](int s) { return bar0 + 8u * s; };
  auto empty = [&](int s) { return bar0 + 8u * (STAGES + s); };
  auto tfull = [&](int b) { return bar0 + 8u * (2 * STAGES + b); };
  auto tempty = [&](int b) { return bar0 + 8u * (2 * STAGES + 4 + b); };
  const Told told{bar0 + 8u * (2 * STAGES + 8)};    // factors, and with a tile's first ones its place
  const int warp = uniform_warp(), lane = threadIdx.x & 31, rank = (int)cluster_ctarank();

  if (warp == 0 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
  }
  if (warp == 1 && lane == 0) {
    for (int s = 0; s < STAGES; ++s) { bar_init(full(s), 3); bar_init(empty(s), 2); }       // (full: the leader's copies, both CTAs' factors)
    for (int b = 0; b < 4; ++b) { bar_init(tfull(b), 1); bar_init(tempty(b), kSumWarps); }       // (of two blocks, the first and the second 128 columns)
    told.init(kPairSlots);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 2) {
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(&tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
  }
  if (!p.offsets && threadIdx.x == 0) { groups.starts[0] = 0; groups.near[0] = make_int2(0, p.T); groups.starts[1] = (p.T + 2 * kRows - 1) / (2 * kRows) * p.n_tiles; }
  fence_before();
  __syncthreads();
  fence_after();
  const uint32_t tmem = tmem_slot;
  pdl_launch_dependents();
  cluster_arrive(); cluster_wait();                 // the peer's barriers are there
  pdl_wait();
  if (p.offsets) count_tiles(p, 2 * kRows, groups);
  const int KB = p.KB, total = same(groups.starts[p.E]), first = (int)blockIdx.x >> 1, step = (int)gridDim.x >> 1;
  const int e_first = first < total ? first_group(p, groups, first) : 0;
  float* factors = reinterpret_cast<float*>(smem + STAGES * kStage + (GATED ? 0 : kSumWarps * 2048));

  if (warp == 0 || warp == 3) {
    // the copies and factors of kPairBatch blocks of K by one of the two, of as many by the other
    regs_down<kOtherRegs>();
    int stage = 0, slot = 0, tile = 0, e = e_first, turn = 1 - (warp & 1);
    uint32_t phase = 0;
    const uint32_t lead0 = mapa_u32(full(0), 0);
    for (int w = first; w < total; w += step) {
      const Tile t = same(find_tile<2 * kRows, kPairBand>(p, groups, w, e));
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
          if (lane == 0) {
            told.tell(slot);
            bar_arrive_at(lead);                     // (so that when a block's sums are there its factors mostly are)
          }
          if (++stage == STAGES) { stage = 0; phase ^= 1; }
          if (++slot == kPairSlots) slot = 0;
        }
      }
    }
  } else if (warp < 4) {
    regs_down<kOtherRegs>();
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
    regs_up<kSumRegs>();
    const int q = warp & 3, part = (warp - 4) >> 2, lane128 = q * 32 + lane;
    const uint32_t lead_tempty = mapa_u32(tempty(part), 0);
    int buf = 0, slot = 0, tile = 0;
    uint32_t buf_phase = 0, slot_phase = 0;
    for (int w = first; w < total; w += step) {
      told.wait(slot, slot_phase);
      mbar_wait(tfull(2 * buf + part), buf_phase);
      const int4 found = tiles[tile++ & 15];
      const Tile t = same(Tile{0, found.x, found.y, found.z});
      const int mine = rank * kRows + lane128;
      const bool some = rank * kRows + q * 32 < t.rows, there = mine < t.rows;
      const int row = t.row + mine, n0 = t.n * 256 + part * 128;
      Sums<C> s;
      s.clear();
      uint32_t* own = biases + (GATED ? 0 : (warp - 4) * 64);
      if (!GATED && p.bias) ask_bias<2, 64>(p, own, n0, lane);
      const uint32_t at = tmem + ((uint32_t)(q * 32) << 16) + part * 128;
      bool seen = true;                               // a slot is asked for a block ahead (where it is wanted, 4 % more)
      auto read = [&] {
        fence_before();
        bar_arrive_lane0(lead_tempty + 16u * buf, lane);
        if (++buf == 2) { buf = 0; buf_phase ^= 1; }
        if (++slot == kPairSlots) { slot = 0; slot_phase ^= 1; }
      };
      auto wait = [&](uint32_t& from, float& f0, float& f1) {
        if (!seen) told.wait(slot, slot_phase);
        const bool last = slot + 1 == kPairSlots;
        seen = told.test(last ? 0 : slot + 1, slot_phase ^ last);
        const float* f = factors + slot * 256 + lane128;
        f0 = f[GATED ? 0 : part * 128];
        f1 = GATED ? f[128] : f0;
        mbar_wait(tfull(2 * buf + part), buf_phase);
        fence_after();
        from = at + buf * 256;
      };
      if (some) {
        add_blocks<C, 0>(s, KB, wait, read);
      } else {
        for (int kb = 0; kb < KB; ++kb) { mbar_wait(tfull(2 * buf + part), buf_phase); read(); }
      }
      if (!GATED && p.bias) add_bias<C>(s, own);
      if constexpr (GATED) {
        store_gated(p, s, row, there, t.n, tops, part, lane128);
      } else if (some) {
        const uint32_t buffer = base + STAGES * kStage + (warp - 4) * 2048;
        if constexpr (WIDE) store_rows<C>(p, s, row - lane, t.rows - (mine - lane), n0, buffer, lane);
        else store_narrow<C, 64>(p, s, row - lane, t.rows - (mine - lane), n0, buffer, lane);
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
  const CUresult r = with_context(CUDA_ERROR_INVALID_CONTEXT, fp8_pair_kernel<false, true>, [&] {
    return enc(m, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
  KGE_REQUIRE(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled failed (%d) rows=%lld cols=%lld", (int)r, (long long)rows, (long long)cols);
  return 0;
}

static bool aligned_to(const void* p, int n) { return ((uintptr_t)p & (n - 1)) == 0; }

static int sm_count() {
  int dev = 0, n = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return 0;
  return n < kMaxCtas ? n : kMaxCtas;
}

// How many clusters of `size` CTAs, one an SM, run at once.
static int max_clusters(int size) {
  static std::atomic<int> cache[kMaxSplits + 1];
  int n = cache[size].load(std::memory_order_relaxed);
  if (n == 0) {
    auto kern = fp8_stream_kernel<128, false, true>;
    int got = 0;
    if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem - kOwn) == cudaSuccess) {
      cudaLaunchConfig_t cfg = {};
      cfg.gridDim = dim3(size * 64); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = kSmem - kOwn;
      cudaLaunchAttribute attr[1];
      attr[0].id = cudaLaunchAttributeClusterDimension;
      attr[0].val.clusterDim.x = size; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
      cfg.attrs = attr; cfg.numAttrs = 1;
      if (cudaOccupancyMaxActiveClusters(&got, kern, &cfg) != cudaSuccess) { (void)cudaGetLastError(); got = 0; }
    }
    n = got + 1;
    cache[size].store(n, std::memory_order_relaxed);
  }
  return n - 1;
}

static int quarters_of(int T) { return ((T < kRows ? T : kRows) + 31) / 32; }
// What the sums of a cluster's shares take of shared memory, and how many stages are left.
static int sums_bytes(int splits, int sets, int quarters) { return splits > 1 ? splits * ((16 + splits - 1) / splits) * sets * 2 * quarters * 32 * 16 : 0; }
static int stage_bytes_of(int nt, int quarters) { return stream_sub(nt) * (quarters * 4096 + nt * 128 + kSlotBytes); }
static int stages_beside(int bytes, int nt, int quarters) {
  const int n = (kSmem - kOwn - 1024 - 512 / nt * kSlotBytes - bytes) / stage_bytes_of(nt, quarters);
  return n < kMaxStages ? n : kMaxStages;
}
// What a tile's end takes of shared memory beside the stages: a cluster's sums, if two stages are left (else they lie over the stages: gated 128 rows); without
// a cluster, 9 KB for rows that are not 16-byte aligned.
static int end_bytes(int nt, int splits, int quarters, int wide) {
  if (splits <= 1) return wide ? 0 : kSumWarps * kNarrow;
  const int sums = sums_bytes(splits, nt / 128, quarters);
  return stages_beside(sums, nt, quarters) >= 2 ? sums : 0;
}
static int stream_stages(int nt, int splits, int quarters, int wide) { return stages_beside(end_bytes(nt, splits, quarters, wide), nt, quarters); }
// Shares of K of a dense problem's tiles: the most that run at once.
static int plan_splits(int64_t tiles, int KB, int sms) {
  if (2 * tiles >= sms) return 1;
  for (int s = kMaxSplits; s > 1; --s)
    if (tiles * s <= sms && KB >= 2 * s && tiles <= max_clusters(s)) return s;
  return 1;
}
// Which kernel a dense problem takes, by what each is measured to need: a block of K 0.37 us a tile of the pair kernel and 1.8 for the tile's end (4.4 where
// rows are not 16-byte aligned); 0.38 a tile of 128 columns of the other and 0.70 of 256, and 1.5 for its end; 0.45 and 0.70 of a share, for there the rings
// are not yet full, and 0.7 (gated 1.5) of every 32 rows for the exchange; 5 us for start and end.  us by pairs and by single CTAs: 128 x 28672 x 4096 37.2 and
// 29.1, 256 38.2 and 51.5, 512 64 and 98; 256 x 4096 x 4096 18.7 and 13.0, 512 19.4 and 16.7, 1024 20.4 and 23.0; 898 x 491 x 512 11.0 and 8.4; gated 128 x
// 28672 x 4096 36.5 and 26.8, 256 37.6 and 47.2; 1112 x 256 x 10240 31.5 and 16.9.  Of 45 dense shapes drawn at random the slower one was taken for three, by
// 10 % and more: all of 12 us and less.
static bool use_pairs(int T, int N, int KB, bool gated, int sms) {
  auto up = [](int64_t a, int64_t b) { return (a + b - 1) / b; };
  const int64_t wide = up(N, gated ? 128 : 256);
  const double pairs = up(up(T, 2 * kRows) * wide, sms / 2) * (KB * 0.37 + (gated || N % 8 == 0 ? 1.8 : 4.4));
  double single = up(up(T, kRows) * wide, sms) * (KB * 0.70 + 1.5);
  const int64_t tiles = up(T, kRows) * (gated ? wide : up(N, 128));
  const int splits = plan_splits(tiles, KB, sms);
  if (splits > 1) single = up(KB, splits) * (gated ? 0.70 : 0.45) + (gated ? 1.5 : 0.7) * quarters_of(T);
  else if (!gated && 2 * up(T, kRows) * wide < sms) single = up(tiles, sms) * (KB * 0.38 + 1.5);
  return pairs < single;
}

template <int NT, bool GATED>
static int launch_stream(Fp8Params& p, const void* x, const void* w, int K, cudaStream_t st) {
  p.quarters = quarters_of(p.T);
  p.x_bytes = p.quarters * 4096;
  p.n_tiles = (p.N + (GATED ? 128 : NT) - 1) / (GATED ? 128 : NT);
  const int sms = sm_count();
  const int64_t tiles = (int64_t)((p.T + kRows - 1) / kRows) * p.n_tiles;
  p.splits = 0;                                            // grouped: by the number of tiles, on the device
  if (!p.offsets) p.splits = GATED || NT == 128 ? plan_splits(tiles, p.KB, sms) : 1;
  const bool cluster = p.splits > 1;
  if (cluster) {
    p.most = (16 + p.splits - 1) / p.splits;
    for (int c = 0; c <= p.splits; ++c) p.first[c] = (uint8_t)(16 * c / p.splits);
    for (int c = 0; c < p.splits; ++c)
      for (int g = p.first[c]; g < p.first[c + 1]; ++g) p.owner[g] = (uint8_t)c;
  }
  p.wide = GATED || (p.N % 8 == 0 && aligned_to(p.y, 16));
  p.stages = stream_stages(NT, p.splits, p.quarters, p.wide);
  p.over = cluster && end_bytes(NT, p.splits, p.quarters, p.wide) == 0;
  KGE_REQUIRE(p.stages >= 2 && (!p.over || p.stages * stage_bytes_of(NT, p.quarters) >= sums_bytes(p.splits, NT / 128, p.quarters)), "kge_gemm_fp8: internal: %d stages", p.stages);
  p.ahead = p.stages;
  // an MMA reads 128 rows of tokens from where they begin, and finds others' bytes behind the last: never beyond the stage's weights
  static_assert(NT * 128 >= kRows * 128, "");
  const int smem = p.stages * stage_bytes_of(NT, p.quarters) + 512 / NT * kSlotBytes + end_bytes(NT, p.splits, p.quarters, p.wide) + 1024;
  CUtensorMap mw, mx;
  if (int rc = encode_map(&mw, w, (int64_t)p.E * p.w_rows, K, 128)) return rc;
  if (int rc = encode_map(&mx, x, p.T, K, 32)) return rc;
  auto kern = fp8_stream_kernel<NT, GATED, false>;
  if constexpr (GATED || NT == 128) {
    if (cluster) kern = fp8_stream_kernel<NT, GATED, true>;
  }
  // the function's limit, for every size: one set for this call could be lowered by another thread's before the launch
  KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, kSmem - kOwn));
  prefer_max_shared(kern);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(cluster ? tiles * p.splits : sms)); cfg.blockDim = dim3(kThreads); cfg.dynamicSmemBytes = smem; cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = (p.offsets ? pdl_for_this_launch() : pdl_for_weights(st)) ? 1 : 0;      // (grouped rows wait before they read anything)
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = p.splits; attr[1].val.clusterDim.y = 1; attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr; cfg.numAttrs = cluster ? 2 : 1;
  KGE_CUDA_OK(cudaLaunchKernelEx(&cfg, kern, mw, mx, p));
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
  auto kern = fp8_pair_kernel<GATED, true>;
  if constexpr (!GATED) {
    if (!p.wide) kern = fp8_pair_kernel<GATED, false>;
  }
  KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
  prefer_max_shared(kern);
  const int sms = sm_count();
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
  return kCounters * 4 + (int64_t)kMaxCtas * quarters * 256 * 128;
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
  KGE_REQUIRE(tiles < (1ll << 31) && tiles * p.KB < (1ll << 31), "%s: %lld tiles of %d blocks in one call", name, (long long)tiles, p.KB);
  KGE_REQUIRE(workspace && workspace_bytes >= workspace_bytes_of(p.T) && aligned_to(workspace, 16), "%s: needs a workspace of %lld bytes, 16-byte aligned", name,
              (long long)workspace_bytes_of(p.T));
  p.count = (unsigned int*)workspace;
  p.part = (float*)((uint8_t*)workspace + kCounters * 4);
  const int sms = sm_count();
  if (sms < 2) {
    set_error("%s: no CUDA device", name);
    return -2;
  }
  // Groups: by their mean size.  64 of 2048 x 1408, us by pairs and by single CTAs: 96 rows each 59.3 and 59.7, 192 71.5 and 85.9; 16 of 2048 x 2048: 128 25.7
  // and 30.8, 256 33.5 and 44.2.
  const bool pairs = p.offsets ? p.T / p.E > 96 : use_pairs(p.T, p.N, p.KB, gated, sms);
#ifndef KGE_HALF
  if (gated) return pairs ? launch_pairs<true>(p, x, w, K, st) : launch_stream<256, true>(p, x, w, K, st);
#endif
  if (pairs) return launch_pairs<false>(p, x, w, K, st);
  // Tiles of 256 columns where they are enough for whole tiles a CTA: 64 tokens, us with 128 and 256, 28672 x 4096 27.5 and 25.9, 128256 x 4096 96.5 and 97.4,
  // 128 experts of 2048 x 768, 512 rows, 39.2 and 38.6.  Cut along K they have less to show (4096 x 4096 8.8 and 10.3).
  const int64_t groups = p.offsets && p.T < p.E ? p.T : p.E, wide = ((int64_t)(p.T / p.E + kRows - 1) / kRows + (p.T < p.E)) * groups * ((p.N + 255) / 256);
  return 2 * wide >= sms ? launch_stream<256, false>(p, x, w, K, st) : launch_stream<128, false>(p, x, w, K, st);
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
