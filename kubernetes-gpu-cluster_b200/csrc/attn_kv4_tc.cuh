// Prompt attention over the 4-bit key-value cache (layout: kv4.cuh).  Included by attn_tc.cu inside its namespaces (tiles, descriptors, MMA
// wrappers), behind attn_pair.cuh, whose plan it shares: two query tiles of 128 rows per CTA with four softmax warps and an issuer each, scores
// and probabilities in TMEM, work from the hardware's queue of CTAs not yet launched.
//
// What differs is how keys and values become operands.  A producer brings the groups of 64 keys as they lie in the pages (hd + 8 bytes a key, a
// quarter of 16-bit rows) into a ring, and four warps of their own turn codes into the 128-byte-swizzled tiles that the MMAs read: n - 8, which is
// exact, of keys in the model's type, as Q is, of values in float16, as the weights are in either build.  The two numbers of a row are applied in
// fp32 by the softmax (z = low + 8 s):
//   x = scale (s_k S + z_k sum(q))       e = 2^(x - X)       P = 2^-M e s_v       out = (sum P (n - 8) + sum 2^-M e z_v) / (2^-M sum e)
// so besides the result only P is rounded to 16 bits, and nothing that a query gets hangs on rows that it does not see, not even in its last bit:
// scores, numbers, X and M are its own, and masked weights are zeros that meet finite codes.  (Rows as float16 numbers with a power of two for a tile
// save the 64 shared loads of 16 bytes a tile and thread that the numbers cost, 182 us against 206 below, but a tile's largest row decides what the
// others keep: a key 10^5 times as large spoilt queries in front of it.)
// X is the largest score of the first tile in which a row sees keys, M its largest x_j + m_j - X with m_j = log2 of max(2^-6 s_v, 2^-90 |z_v|,
// 2^-90): P is at most 2^6 then, and 2^-M e z_v and the sums stay finite whatever the values are.  They move when a P may pass 2^14 (or z_v's sums
// 2^98) or an e 2^60, so weights lose bits 2^20 below the largest.  (One number X + M for both: 3 % less time, but a large score swallows the M, and
// where values are large their small e end before they count for nothing in sum e.)
// Error against 64 bits, largest: bfloat16 0.0017, float16 0.0003, of which the result's own rounding is 0.0016 and 0.00021.
// The turning warps need few registers and the softmax many: 512 threads start with 128 each, and setmaxnreg hands 40 of each of eight warps'
// to the eight softmax warps (168 and 88: 128 (2 x 168 + 2 x 88) = 65536, what the launch holds).
//   * Rows that read as NaN (kv4.cuh) must not reach queries that do not see them: such a key has s_v = z_v = 0 here and s_k is NaN, so every query
//     that sees it gets NaN from its score and no other does.
//   * Rows behind the last key are zeros, whatever the page holds.
//   * A window with first tokens that stay visible: tiles of the first tokens, then those of the windows; only tiles at a border are masked.
namespace atc4 {
using namespace atc;
using atc2::max3; using atc2::tma_load_3d; using atc2::tmem_ld32_nowait; using atc2::tmem_st16; using atc2::tmem_wait_st;

constexpr int kThreads = 512;                  // warps 0-3 and 4-7: softmax of the two query tiles; 8 and 9: their MMAs; 10: copies; 12-15: codes to tiles
constexpr int NST = 3, NRAW = 3;               // K tiles and as many V tiles; tiles of codes
constexpr int kSoftmaxRegs = 168, kOtherRegs = 88;
static_assert(2 * kSoftmaxRegs + 2 * kOtherRegs == 4 * 128, "the register shares are what the launch holds");
constexpr int kNumbers = 1024 + 256 + 16;      // of a stage: per pair of keys (s, s, z, z) of the keys and of the values; m of each key; the largest of 32 each
constexpr float kLeastTop = 6.f, kRoom = 90.f, kScoreRoom = 60.f;       // log2 of a row's largest P when M is set; of 2^-M z_v; of e
template <int HD> constexpr int raw_bytes() { return 4 * kv4::group_bytes(HD); }
template <int HD> constexpr int smem_bytes() { return (2 * 128 + 2 * NST * BNK) * HD * 2 + NRAW * raw_bytes<HD>() + NST * kNumbers + 512 + 8 * 4096 + 128 * 16; }

// n0, n1: key tiles of the two query tiles; n1 < 0: no more work.  split: one query tile, its even key tiles are the first warps', its odd ones
// the second's.  Tile j holds the keys from 64 j (j < ptiles: first tokens that stay visible) or from 64 (tile_lo + j - ptiles).
struct __align__(16) Item { int q0, tok0, ntok0, ntok1, ctx0, kvh, n0, n1, split, ptiles, tile_lo, kv_len; };

struct KvArgs {
  const uint8_t* cache;
  const int32_t *table, *lens, *qsl;
  int max_blocks, flat, per, H, KV, bs_shift, window, first, skip_single;
  float scale_log2;
};

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes, uint32_t bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}
__device__ __forceinline__ void st_shared16(uint32_t dst, const uint32_t (&v)[4]) {
  asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(dst), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]) : "memory");
}
// eight codes n -> eight float16 numbers n - 8, in order
__device__ __forceinline__ void expand(uint32_t w, uint32_t (&r)[4]) {
#pragma unroll
  for (int p = 0; p < 4; ++p) {
    const uint32_t u = p < 2 ? w : w >> 8;               // 0x6400 | n = 1024 + n; 0x6400 | n << 4 = 1024 + 16 n
    if (p & 1) asm("fma.rn.f16x2 %0, %1, %2, %3;" : "=r"(r[p]) : "r"((u & 0x00f000f0u) | 0x64006400u), "r"(0x2c002c00u), "r"(0xd480d480u));
    else asm("sub.rn.f16x2 %0, %1, %2;" : "=r"(r[p]) : "r"((u & 0x000f000fu) | 0x64006400u), "r"(0x64086408u));
  }
}
// the same as numbers of the model's type
__device__ __forceinline__ void expand_key(uint32_t w, uint32_t (&r)[4]) {
#ifdef KGE_HALF
  expand(w, r);
#else
#pragma unroll
  for (int p = 0; p < 4; ++p) asm("sub.rn.bf16x2 %0, %1, %2;" : "=r"(r[p]) : "r"(((w >> (4 * p)) & 0x000f000fu) | 0x43004300u), "r"(0x43084308u));      // 0x4300 | n = 128 + n
#endif
}
__device__ __forceinline__ uint32_t pack_h2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}
__device__ __forceinline__ bool finite2(uint32_t p) {    // both 16-bit numbers of a row
#ifdef KGE_HALF
  return (p & 0x7c00u) != 0x7c00u && (p & 0x7c000000u) != 0x7c000000u;
#else
  return (p & 0x7f80u) != 0x7f80u && (p & 0x7f800000u) != 0x7f800000u;
#endif
}

template <int HD>
__global__ void __launch_bounds__(kThreads, 1)
attn_kv4_tc_kernel(const __grid_constant__ CUtensorMap tm_q8, const __grid_constant__ CUtensorMap tm_q1, bf16* __restrict__ out, const KvArgs ka) {
  constexpr uint32_t Q_TILE = 128 * HD * 2, TILE = BNK * HD * 2, RAW = (uint32_t)(4 * kv4::group_bytes(HD)), GB = (uint32_t)kv4::group_bytes(HD);
  constexpr uint32_t S_COL = 256;              // TMEM: O0 and O1, then per query tile the scores (64 columns) and two buffers of probabilities (32 each)
  constexpr uint32_t IDESC_S = (1u << 4) | KGE_IDESC_AB | ((uint32_t)(BNK >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
  constexpr uint32_t IDESC_O = (1u << 4) | (1u << 16) | ((uint32_t)(HD >> 3) << 17) | ((uint32_t)(BM >> 4) << 24);
  extern __shared__ __align__(1024) uint8_t smem_raw[];
  if ((s_addr(smem_raw) & 1023u) != 0) __trap();
  const uint32_t sQ = s_addr(smem_raw), sK = sQ + 2 * Q_TILE, sV = sK + NST * TILE;
  uint8_t* raw = smem_raw + 2 * Q_TILE + 2 * NST * TILE;
  uint8_t* numbers = raw + NRAW * RAW;
  uint8_t* tail = numbers + NST * kNumbers;
  uint8_t* stage_out = tail + 512;
  float4* part = reinterpret_cast<float4*>(stage_out + 8 * 4096);
  const uint32_t bar0 = s_addr(tail);
  Item* items = reinterpret_cast<Item*>(tail + 288);                   // 2 slots of 48 bytes
  const uint32_t clc_resp = bar0 + 384;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(tail + 400);
  static_assert(sizeof(Item) == 48, "two items lie between the barriers and the answers to requests for work");
  // Barriers; tiles are counted over all items of the CTA.  A parity wait holds only while no later phase of its barrier can complete: what
  // completes the next phase needs something that the waiter does after the wait (p_full and o_full, which may run a tile ahead of their
  // waiters, are pairs for that).  No stage is handed back before it was filled: an issuer without work for a tile waits for it too.
  //   raw_full(r)   the four turning warps, before they arrive on raw_empty(r), without which the producer does not refill it
  //   raw_empty(r)  the producer, before the copy that the next phase of raw_full(r) counts
  //   k_full, v_full: 4 arrivals of the turning warps; k_empty, v_empty: a commit of each issuer, waited for by the turning warps before they
  //   write the stage again.  The numbers of a stage are written with its values and read by the softmax, which waits for v_full too: the
  //   next phase of it needs v_empty, that a P V, and that the P of the waiter
  //   q_empty       a commit of each issuer, and the softmax warps, which have summed their rows of Q
  auto k_full = [&](int s) { return bar0 + 8u * s; };
  auto k_empty = [&](int s) { return bar0 + 24u + 8u * s; };
  auto v_full = [&](int s) { return bar0 + 48u + 8u * s; };
  auto v_empty = [&](int s) { return bar0 + 72u + 8u * s; };
  auto raw_full = [&](int s) { return bar0 + 96u + 8u * s; };
  auto raw_empty = [&](int s) { return bar0 + 120u + 8u * s; };
  auto s_full = [&](int a) { return bar0 + 144u + 8u * a; };
  auto s_read = [&](int a) { return bar0 + 160u + 8u * a; };
  auto p_full = [&](int a, int t) { return bar0 + 176u + 16u * a + 8u * (t & 1); };
  auto o_full = [&](int a, int t) { return bar0 + 208u + 16u * a + 8u * (t & 1); };
  auto item_full = [&](int s) { return bar0 + 240u + 8u * s; };
  auto item_empty = [&](int s) { return bar0 + 256u + 8u * s; };
  const uint32_t q_full = bar0 + 272u, q_empty = bar0 + 280u, clc_full = bar0 + 408u;
  const int warp = uniform_warp(), lane = threadIdx.x & 31;
  const int G = ka.H / ka.KV, TT = BM / G, TI = ka.per * TT;           // tokens of a query tile, of an item

  if (warp == 8) {
    if (lane == 0) {
      for (int s = 0; s < NST; ++s) { mbar_init(k_full(s), 4); mbar_init(k_empty(s), 2); mbar_init(v_full(s), 4); mbar_init(v_empty(s), 2); }
      for (int s = 0; s < NRAW; ++s) { mbar_init(raw_full(s), 1); mbar_init(raw_empty(s), 4); }
      for (int a = 0; a < 2; ++a) {
        mbar_init(s_full(a), 1); mbar_init(s_read(a), 4);
        for (int t = 0; t < 2; ++t) { mbar_init(p_full(a, t), 4); mbar_init(o_full(a, t), 1); }
        mbar_init(item_full(a), 1); mbar_init(item_empty(a), 14);      // 8 softmax warps, 2 issuers, 4 turning warps
      }
      mbar_init(q_full, 1); mbar_init(q_empty, 10); mbar_init(clc_full, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(s_addr(tmem_slot)), "n"(512) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (warp == 10 && lane == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&tm_q8) : "memory");
  }
  tc_before();
  __syncthreads();
  tc_after();
  const uint32_t tmem = *tmem_slot;
  pdl_launch_dependents();
  pdl_wait();

  if (warp >= 8) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    if (warp == 10) {
      // ------------------------------------------------------------------ work items, Q, tiles of codes
      int bx = blockIdx.x, by = blockIdx.y, bz = blockIdx.z;
      const bool leader = elect_one();
      const int bs = 1 << ka.bs_shift, box = bs < BNK ? bs : BNK;      // keys of one copy
      uint32_t nraw = 0, ni = 0, nclc = 0;
      while (true) {
        int rank = bz, kvh = bx, b = by;
        auto tokens = [&](int r) {                                     // of request r, for this kernel
          const int n = ka.qsl[r + 1] - ka.qsl[r];
          return ka.skip_single && n == 1 ? 0 : n;
        };
        if (ka.flat) {
          // work number bx / KV in the requests' order from the last to the first, without gaps: 32 requests at a time
          kvh = bx % ka.KV;
          rank = bx / ka.KV;
          by = 0;
          for (b = -1; b < 0;) {
            const int r = by + lane, mine = r < ka.flat ? (tokens(ka.flat - 1 - r) + TI - 1) / TI : 0;
            int upto = mine;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
              const int v = __shfl_up_sync(0xffffffffu, upto, o);
              if (lane >= o) upto += v;
            }
            const uint32_t past = __ballot_sync(0xffffffffu, upto > rank);
            if (past) {
              const int l = __ffs(past) - 1;
              rank -= __shfl_sync(0xffffffffu, upto - mine, l);
              b = ka.flat - 1 - by - l;
            } else {
              rank -= __shfl_sync(0xffffffffu, upto, 31);
              by += 32;
              if (by >= ka.flat) { b = 0; rank = -1; }                 // more CTAs than work
            }
          }
        }
        const int32_t* btab = ka.table + (int64_t)b * ka.max_blocks;
        const int q0 = ka.qsl[b], q_len = tokens(b);
        const int tok0 = rank < 0 || q_len <= 0 ? -1 : ((q_len + TI - 1) / TI - 1 - rank) * TI;
        if (tok0 >= 0) {
          // (a length below the rows: the first of them have no key, ctx0 is negative, and what they get is zeros)
          const int ctx0 = min(max(ka.lens[b], 0), ka.max_blocks << ka.bs_shift) - q_len;
          const int ntok0 = min(TT, q_len - tok0), ntok1 = max(0, min(TI - TT, q_len - tok0 - TT));
          const int kv_len = ctx0 + tok0 + ntok0 + ntok1;
          const int tile_lo = ka.window > 0 ? max(0, ctx0 + tok0 - ka.window + 1) / BNK : 0;
          const int ptiles = min((min(ka.first, max(0, kv_len - ka.window)) + BNK - 1) / BNK, tile_lo);
          const int n = max(1, ptiles + (kv_len + BNK - 1) / BNK - tile_lo), split = ntok1 == 0 && n > 1;
          const int n0 = split ? (n + 1) / 2 : max(1, ptiles + (ctx0 + tok0 + ntok0 + BNK - 1) / BNK - tile_lo), n1 = split ? n / 2 : (ntok1 ? n : 0);
          const int slot = ni & 1;
          if (ni >= 2) mbar_wait(item_empty(slot), ((ni >> 1) - 1) & 1);
          if (leader) {
            Item it;
            it.q0 = q0; it.tok0 = tok0; it.ntok0 = ntok0; it.ntok1 = ntok1; it.ctx0 = ctx0; it.kvh = kvh; it.n0 = n0; it.n1 = n1; it.split = split;
            it.ptiles = ptiles; it.tile_lo = tile_lo; it.kv_len = kv_len;
            items[slot] = it;
            mbar_arrive(item_full(slot));
          }
          __syncwarp();
          // Q: boxes of 8 tokens, single tokens for the rest, so that nothing beyond the request's rows is read
          if (ni > 0) mbar_wait(q_empty, (ni - 1) & 1);
          if (leader) {
            mbar_expect_tx(q_full, (uint32_t)((ntok0 + ntok1) * G * HD * 2));
#pragma unroll 1
            for (int a = 0; a < 2; ++a) {
              const int nt = a ? ntok1 : ntok0, full = TT >= 8 ? nt & ~7 : 0;
              for (int t = 0; t < nt; t += t < full ? 8 : 1)
#pragma unroll
                for (int h = 0; h < HD / 64; ++h)
                  tma_load_3d(sQ + a * Q_TILE + (uint32_t)(h * (128 * 128) + t * G * 128), t < full ? &tm_q8 : &tm_q1, q_full, h * 64, kvh * G, q0 + tok0 + a * TT + t);
            }
          }
          __syncwarp();
          // a copy per block of a tile; a lane a copy.  The block ids of the next tile are read while this one's stage is waited for.
          auto block_of = [&](int j) {
            const int key = (j < ptiles ? j : tile_lo + j - ptiles) * BNK + lane * box;
            return j < n && lane * box < BNK && key < kv_len ? btab[key >> ka.bs_shift] : -1;
          };
          int blk = block_of(0);
          for (int j = 0; j < n; ++j, ++nraw) {
            const int st = nraw % NRAW, key0 = (j < ptiles ? j : tile_lo + j - ptiles) * BNK;
            const int groups = min(4, max(0, (kv_len - key0 + 15) >> 4));
            const int mine = blk, first = lane * (box >> 4), count = min(box >> 4, groups - first);
            blk = block_of(j + 1);
            if (nraw >= (uint32_t)NRAW) mbar_wait(raw_empty(st), (nraw / NRAW - 1) & 1);
            const uint32_t dst = s_addr(raw) + st * RAW;
            if (leader) mbar_expect_tx(raw_full(st), (uint32_t)groups * GB);
            __syncwarp();
            if (mine >= 0 && count > 0) {
              const int in_block = (key0 + lane * box) & (bs - 1);
              bulk_load(dst + first * GB, ka.cache + ((((int64_t)mine * ka.KV + kvh) << (ka.bs_shift - 4)) + (in_block >> 4)) * GB, (uint32_t)count * GB, raw_full(st));
            }
          }
          ++ni;
        }
        // the next item, asked for with the last tiles of this one in flight (attn_pair.cuh)
        if (leader) {
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          mbar_expect_tx(clc_full, 16);
          asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];" ::"r"(clc_resp), "r"(clc_full) : "memory");
        }
        __syncwarp();
        mbar_wait(clc_full, nclc & 1);
        ++nclc;
        uint32_t ok, x = 0, y = 0, z = 0;
        asm volatile(
            "{\n.reg .b128 h;\n.reg .pred p;\nld.shared.b128 h, [%4];\n"
            "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, h;\nselp.u32 %0, 1, 0, p;\n"
            "mov.b32 %1, 0;\nmov.b32 %2, 0;\nmov.b32 %3, 0;\n"
            "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {%1, %2, %3, _}, h;\n}"
            : "=r"(ok), "=r"(x), "=r"(y), "=r"(z) : "r"(clc_resp) : "memory");
        __syncwarp();
        if (!ok) break;
        bx = (int)x; by = (int)y; bz = (int)z;
      }
      const int slot = ni & 1;
      if (ni >= 2) mbar_wait(item_empty(slot), ((ni >> 1) - 1) & 1);
      if (leader) {
        items[slot].n1 = -1;
        mbar_arrive(item_full(slot));
      }
    } else if (warp == 8 || warp == 9) {
      // ------------------------------------------------------------------ MMA issuer of query tile a
      if (elect_one()) {
        const int a = warp - 8;
        const uint32_t t_s = tmem + S_COL + a * 128, t_o = tmem + a * 128;
        uint32_t ns = 0, np = 0, nk = 0;                 // score tiles and products P V issued so far, key tiles
        for (uint32_t ni = 0;; ++ni) {
          mbar_wait(item_full(ni & 1), (ni >> 1) & 1);
          const int n0 = items[ni & 1].n0, n1 = items[ni & 1].n1, split = items[ni & 1].split;
          mbar_arrive(item_empty(ni & 1));
          if (n1 < 0) break;
          const int n = split ? n0 + n1 : max(n0, n1), na = a ? n1 : n0, ahead = 1 + split;
          const uint64_t qd = desc_kmajor(sQ + (split ? 0 : a) * Q_TILE);
          mbar_wait(q_full, ni & 1);
          bool first = true;                             // no product P V of this item yet
          for (int j = -ahead; j < n; ++j) {
            const int js = j + ahead;
            if (js < n) {                                // S of a tile ahead, once the softmax has read the one before
              const int st = (nk + js) % NST;
              mbar_wait(k_full(st), ((nk + js) / NST) & 1);         // also without work for it: the stage is not handed back before it is filled
              if (split ? (js & 1) == a : js < na) {
                if (ns > 0) mbar_wait(s_read(a), (ns - 1) & 1);
                tc_after();
                const uint64_t kd = desc_kmajor(sK + st * TILE);
#pragma unroll
                for (int k = 0; k < HD / 16; ++k) {
                  const uint32_t qoff = (uint32_t)((k >> 2) * (128 * 128) + (k & 3) * 32), koff = (uint32_t)((k >> 2) * (BNK * 128) + (k & 3) * 32);
                  tc_mma(t_s, qd + (qoff >> 4), kd + (koff >> 4), IDESC_S, k > 0 ? 1u : 0u);
                }
                tc_commit(s_full(a));
                ++ns;
              }
              tc_commit(k_empty(st));
              if (js + 1 == n) tc_commit(q_empty);
            }
            if (j >= 0) {                                // P V of tile j
              const int st = (nk + j) % NST;
              mbar_wait(v_full(st), ((nk + j) / NST) & 1);
              if (split ? (j & 1) == a : j < na) {
                mbar_wait(p_full(a, np), (np >> 1) & 1);
                tc_after();
                const uint64_t vd = desc_mnmajor(sV + st * TILE);
                const uint32_t t_p = t_s + 64 + (np & 1) * 32;
#pragma unroll
                for (int k = 0; k < BNK / 16; ++k)
                  tc_mma_ts(t_o, t_p + k * 8, vd + (uint32_t)((k * 16 * 128) >> 4), IDESC_O, (!first || k > 0) ? 1u : 0u);
                tc_commit(o_full(a, np));
                ++np;
                first = false;
              }
              tc_commit(v_empty(st));
            }
          }
          nk += n;
        }
      }
    } else if (warp >= 12) {
      // ------------------------------------------------------------------ codes to tiles: a quarter of a row's words per thread
      constexpr int W = HD / 32;                         // words of a thread's share: chunks W t .. W t + W - 1 of 16 bytes
      const int d = threadIdx.x - 384, t = d & 3, s = d >> 2;
      // rows whose stores share a wavefront lie in complementary halves of the swizzle: two apart (chunks 0, 4 and, of lanes t >= 2, 1, 5) or,
      // for 64 dimensions, one apart
      const int tok = HD == 128 ? ((s & 1) << 1) | ((s >> 1) & 1) | (s & 12) : s & 15;
      const bool swap = HD == 128 && (t & 2);
      uint32_t nk = 0;
      for (uint32_t ni = 0;; ++ni) {
        mbar_wait(item_full(ni & 1), (ni >> 1) & 1);
        const Item it = items[ni & 1];
        __syncwarp();
        if (lane == 0) mbar_arrive(item_empty(ni & 1));
        if (it.n1 < 0) break;
        const int n = it.split ? it.n0 + it.n1 : max(it.n0, it.n1);
        for (int j = 0; j < n; ++j, ++nk) {
          const int st = nk % NST, rs = nk % NRAW;
          const int left = it.kv_len - (j < it.ptiles ? j : it.tile_lo + j - it.ptiles) * BNK;      // keys from this tile on
          mbar_wait(raw_full(rs), (nk / NRAW) & 1);
          // everything that this thread needs of the tile's codes is read at once
          const uint8_t* pairs = raw + rs * RAW + ((d & 63) >> 4) * GB + 16 * HD + (d & 15) * 4;       // the numbers of key d
          const uint32_t pk = *reinterpret_cast<const uint32_t*>(pairs), pv = *reinterpret_cast<const uint32_t*>(pairs + 64);
          uint32_t w[2][2][4];                           // of keys and values: W words of two rows
#pragma unroll
          for (int pass = 0; pass < 2; ++pass) {
            const int grp = (s >> 4) + 2 * pass;
#pragma unroll
            for (int part_v = 0; part_v < 2; ++part_v) {
              const int at = part_v ? 8 * HD + tok * (HD / 2) + 4 * kv4::value_word(HD, tok, W * t) : kv4::key_row(tok) * (HD / 2) + 4 * W * t;
              const uint8_t* src = raw + rs * RAW + grp * GB + at;
              if (HD == 128) {
                const uint4 u = *reinterpret_cast<const uint4*>(src);
                w[part_v][pass][0] = u.x; w[part_v][pass][1] = u.y; w[part_v][pass][2] = u.z; w[part_v][pass][3] = u.w;
              } else {
                const uint2 u = *reinterpret_cast<const uint2*>(src);
                w[part_v][pass][0] = u.x; w[part_v][pass][1] = u.y;
              }
            }
          }
#pragma unroll
          for (int part_v = 0; part_v < 2; ++part_v) {
            if (nk >= (uint32_t)NST) mbar_wait(part_v ? v_empty(st) : k_empty(st), (nk / NST - 1) & 1);
            const uint32_t dst = (part_v ? sV : sK) + st * TILE;
#pragma unroll
            for (int pass = 0; pass < 2; ++pass) {
              const int row = ((s >> 4) + 2 * pass) * 16 + tok;
#pragma unroll
              for (int i = 0; i < W; ++i) {
                // (a row behind the last key: the other warps multiply it with weights of zero)
                const uint32_t x = row >= left ? 0x88888888u : swap ? w[part_v][pass][i ^ 1] : w[part_v][pass][i];
                uint32_t r[4];
                if (part_v) expand(x, r);
                else expand_key(x, r);
                st_shared16(dst + tile_off<BNK>(row, W * t + (swap ? i ^ 1 : i)), r);
              }
            }
            if (part_v && d < 64) {                      // warps 12 and 13: the numbers of key d
              const bool there = d < left, fine = finite2(pk) && finite2(pv);
              const float nan = __uint_as_float(0x7fffffffu);
              const float sk = there ? (fine ? bf_lo(pk) : nan) * ka.scale_log2 : 0.f, zk = there && fine ? fmaf(8.f, bf_lo(pk), bf_hi(pk)) * ka.scale_log2 : 0.f;
              const float sv = there && fine ? bf_lo(pv) : 0.f, zv = there && fine ? fmaf(8.f, sv, bf_hi(pv)) : 0.f;
              float* to = reinterpret_cast<float*>(numbers + st * kNumbers) + (d >> 1) * 8 + (d & 1);
              to[0] = sk; to[2] = zk; to[4] = sv; to[6] = zv;
              const float m = fmaxf(fmaxf(__log2f(sv) - kLeastTop, __log2f(fabsf(zv)) - kRoom), -kRoom);
              float* ms = reinterpret_cast<float*>(numbers + st * kNumbers + 1024);
              ms[d] = m;
              const int most = __reduce_max_sync(0xffffffffu, __float2int_ru(m));
              if (lane == 0) ms[64 + (d >> 5)] = (float)most;
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(part_v ? v_full(st) : k_full(st));
            if (!part_v && lane == 0) mbar_arrive(raw_empty(rs));      // (what was read of it has been used or lies in registers)
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ softmax: one row per thread
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    const int a = warp >> 2, r = threadIdx.x & 127, tk = r / G;
    const uint32_t t_row = tmem + ((uint32_t)((warp & 3) * 32) << 16);
    const uint32_t t_s = t_row + S_COL + a * 128, t_o = t_row + a * 128;
    uint32_t ns = 0, nk = 0;                                           // tiles of this group, key tiles of the items before
    for (uint32_t ni = 0;; ++ni) {
      mbar_wait(item_full(ni & 1), (ni >> 1) & 1);
      const Item it = items[ni & 1];
      __syncwarp();
      if (lane == 0) mbar_arrive(item_empty(ni & 1));
      if (it.n1 < 0) break;
      const int n = a ? it.n1 : it.n0, n_item = it.split ? it.n0 + it.n1 : max(it.n0, it.n1);
      const int qt = it.split ? 0 : a;                                 // the query tile of these warps
      // sum(q) of this thread's row
      mbar_wait(q_full, ni & 1);
      float qsum = 0.f;
      if (n > 0) {
        const uint8_t* row = smem_raw + qt * Q_TILE;
#pragma unroll
        for (int c = 0; c < HD / 8; ++c) {
          const uint4 u = *reinterpret_cast<const uint4*>(row + tile_off<128>(r, c));
          qsum += ((bf_lo(u.x) + bf_hi(u.x)) + (bf_lo(u.y) + bf_hi(u.y))) + ((bf_lo(u.z) + bf_hi(u.z)) + (bf_lo(u.w) + bf_hi(u.w)));
        }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(q_empty);
      if (n <= 0) { nk += n_item; continue; }
      const f2 qs2 = pk(qsum, qsum);
      const bool row_ok = tk < (qt ? it.ntok1 : it.ntok0);
      const int row_tok = it.tok0 + qt * TT + tk;
      const int lim = row_ok ? it.ctx0 + row_tok : -1;                 // last visible key of this row
      const int lo_row = ka.window > 0 ? lim - ka.window + 1 : 0;      // the window's first key; below it only the first tokens
      float x_ref = -INFINITY, m_ref = 0.f, g = 1.f, l = 0.f, zs = 0.f;      // X (none yet: -inf), M and 2^-M
      // the second group's exponentials start when the first's of its first tile are done (attn_pair.cuh)
      const bool turns = it.n1 >= 3;
      for (int j = 0; j < n; ++j) {
        mbar_wait(s_full(a), ns & 1);
        tc_after();
        uint32_t sv[BNK];
#pragma unroll
        for (int c = 0; c < BNK; c += 32) tmem_ld32_nowait(t_s + c, &sv[c]);
        tmem_wait_ld(sv);
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(s_read(a));                         // the next tile's scores may be written
        const int jt = it.split ? 2 * j + a : j, kbase = (jt < it.ptiles ? jt : it.tile_lo + jt - it.ptiles) * BNK;
        const int vis = lim - kbase, from = lo_row - kbase, keep = ka.first - kbase;      // column i is visible: i <= vis and (i >= from or i < keep)
        const int st = (nk + jt) % NST;
        mbar_wait(v_full(st), ((nk + jt) / NST) & 1);                  // the numbers of the tile's keys and values
        const ulonglong2* num = reinterpret_cast<const ulonglong2*>(numbers + st * kNumbers);
#pragma unroll
        for (int i = 0; i < BNK / 2; ++i) {
          const ulonglong2 sz = num[2 * i];
          float x0, x1;
          upk(fma2(pk(__uint_as_float(sv[2 * i]), __uint_as_float(sv[2 * i + 1])), sz.x, mul2(qs2, sz.y)), x0, x1);
          sv[2 * i] = __float_as_uint(x0); sv[2 * i + 1] = __float_as_uint(x1);
        }
        if (!__all_sync(0xffffffffu, vis >= BNK - 1 && (from <= 0 || keep >= BNK))) {
#pragma unroll
          for (int i = 0; i < BNK; ++i) sv[i] = i <= vis && (i >= from || i < keep) ? sv[i] : 0xff800000u;
        }
        // Whether X and M have to be set or moved: not where the largest score and the largest m of the tile, be it of keys that this row does not
        // see, stay below their bounds; else the row's own keys say.
        float mxa[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
        for (int i = 0; i < BNK; i += 8)
#pragma unroll
          for (int k = 0; k < 4; ++k) mxa[k] = max3(mxa[k], __uint_as_float(sv[i + 2 * k]), __uint_as_float(sv[i + 2 * k + 1]));
        const float2 m_most = *reinterpret_cast<const float2*>(numbers + st * kNumbers + 1024 + 256);
        const float high = max3(fmaxf(mxa[0], mxa[1]), mxa[2], mxa[3]);          // -inf: no key, or only NaN rows
        if (__any_sync(0xffffffffu, (high - x_ref) + fmaxf(fmaxf(m_most.x, m_most.y) - m_ref, kRescaleThreshold - kScoreRoom) > kRescaleThreshold)) {
          const float x_new = fmaxf(x_ref, high), dx = x_new - x_ref;
          const ulonglong2* lg = num + 64;
          const f2 nx2 = pk(-x_new, -x_new);
          float top[2] = {-INFINITY, -INFINITY};
#pragma unroll
          for (int i = 0; i < BNK; i += 4) {
            const ulonglong2 m = lg[i / 4];
            float x0, x1, x2, x3;
            upk(add2(add2(pk(__uint_as_float(sv[i]), __uint_as_float(sv[i + 1])), nx2), m.x), x0, x1);
            upk(add2(add2(pk(__uint_as_float(sv[i + 2]), __uint_as_float(sv[i + 3])), nx2), m.y), x2, x3);
            top[i / 4 & 1] = max3(max3(top[i / 4 & 1], x0, x1), x2, x3);
          }
          const float m_new = max3(top[0], top[1], m_ref - dx), up = dx + (m_new - m_ref);
          const bool grow = up > kRescaleThreshold || dx > kScoreRoom;
          if (__any_sync(0xffffffffu, grow)) {
            float alpha = 1.f;
            if (grow) {
              alpha = exp2f(-up);
              l *= exp2f(-dx);
              zs *= alpha;
              x_ref = x_new;
              m_ref = m_new;
              g = exp2f(-m_new);
            }
            if (j > 0) {
              mbar_wait(o_full(a, ns - 1), ((ns - 1) >> 1) & 1);       // P V of the tile before
              tc_after();
#pragma unroll 1
              for (int c = 0; c < HD; c += 16) {
                uint32_t v[16];
                asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                             : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]),
                               "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]) : "r"(t_o + c));
                tmem_wait_ld(v);
#pragma unroll
                for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
                tmem_st16(t_o + c, v);
              }
            }
          }
        }
        const float base = (x_ref == -INFINITY) ? 0.f : x_ref;
        const f2 nb2 = pk(-base, -base), g2 = pk(g, g);
        f2 rs[2] = {0, 0}, zr[2] = {0, 0};
        if (ns >= 2) { mbar_wait(o_full(a, ns), ((ns - 2) >> 1) & 1); tc_after(); }       // P V of two tiles before has read this buffer
        if (turns && j == 0 && a == 1) asm volatile("bar.sync 1, 256;" ::: "memory");
        const uint32_t t_p = t_s + 64 + (ns & 1) * 32;
#pragma unroll
        for (int c = 0; c < BNK; c += 32) {
          uint32_t pkd[16];
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            float p0, p1;
            upk(add2(pk(__uint_as_float(sv[c + 2 * i]), __uint_as_float(sv[c + 2 * i + 1])), nb2), p0, p1);
            const f2 e = pk(ex2_ftz(p0), ex2_ftz(p1));                 // masked: -inf -> 0
            const ulonglong2 sz = num[c + 2 * i + 1];
            rs[i & 1] = add2(rs[i & 1], e);
            const f2 eg = mul2(e, g2);
            zr[i & 1] = fma2(eg, sz.y, zr[i & 1]);
            upk(mul2(eg, sz.x), p0, p1);
            pkd[i] = pack_h2(p0, p1);
          }
          tmem_st16(t_p + c / 2, pkd);
        }
        if (turns && j == 0 && a == 0) asm volatile("bar.arrive 1, 256;" ::: "memory");
        tmem_wait_st();
        tc_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(p_full(a, ns));
        ++ns;
        l += sum2(add2(rs[0], rs[1]));
        zs += sum2(add2(zr[0], zr[1]));
      }
      mbar_wait(o_full(a, ns - 1), ((ns - 1) >> 1) & 1);
      tc_after();
      float mine = 1.f, other = 0.f;                                   // weights of the two halves of a split row
      if (it.split) {
        if (a) part[r] = make_float4(x_ref, m_ref, l, zs);
        tc_before();
        asm volatile("bar.sync 2, 256;" ::: "memory");
        tc_after();
        if (!a) {
          const float4 p1 = part[r];                                   // (a half that saw nothing but NaN keeps it)
          const bool none0 = x_ref == -INFINITY, none1 = p1.x == -INFINITY;
          const float x_new = fmaxf(x_ref, p1.x), up = (p1.x - x_ref) + (p1.y - m_ref);       // X; the other half's X + M less this one's
          mine = none0 ? 0.f : exp2f(-fmaxf(up, 0.f));
          other = none1 ? 0.f : exp2f(fminf(up, 0.f));
          l = (none0 ? (l == l ? 0.f : l) : l * exp2f(x_ref - x_new)) + (none1 ? (p1.z == p1.z ? 0.f : p1.z) : p1.z * exp2f(p1.x - x_new));
          zs = zs * mine + p1.w * other;
          g = exp2f(none0 || up > 0.f ? (x_new - p1.x) - p1.y : (x_new - x_ref) - m_ref);
        }
      }
      const float inv = l > 0.f ? 1.f / (l * g) : l == l ? 0.f : l;
      // a warp turns its 32 rows in shared memory, 64 columns at a time, and stores 128 contiguous bytes of four rows at once
      uint8_t* stage = stage_out + warp * 4096;
      const int srow = lane >> 3, schunk = lane & 7;
      const uint32_t rows_ok = __ballot_sync(0xffffffffu, row_ok);
#pragma unroll 1
      for (int c = 0; c < HD && !(it.split && a); c += 64) {
        uint32_t v[64];
        tmem_ld32_nowait(t_o + c, v);
        tmem_ld32_nowait(t_o + c + 32, v + 32);
        tmem_wait_ld(v);
        if (it.split) {
#pragma unroll
          for (int h = 0; h < 64; h += 32) {
            uint32_t u[32];
            tmem_ld32_nowait(t_o + 128 + c + h, u);
            tmem_wait_ld(u);
#pragma unroll
            for (int i = 0; i < 32; ++i) v[h + i] = __float_as_uint(__uint_as_float(v[h + i]) * mine + __uint_as_float(u[i]) * other);
          }
        }
        tc_before();                                                   // the next item's first P V comes behind p_full of these warps
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 64; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) + zs);
#pragma unroll
        for (int i = 0; i < 64; i += 8) {
          uint4 w;
          w.x = pack_bf2(__uint_as_float(v[i]) * inv, __uint_as_float(v[i + 1]) * inv);
          w.y = pack_bf2(__uint_as_float(v[i + 2]) * inv, __uint_as_float(v[i + 3]) * inv);
          w.z = pack_bf2(__uint_as_float(v[i + 4]) * inv, __uint_as_float(v[i + 5]) * inv);
          w.w = pack_bf2(__uint_as_float(v[i + 6]) * inv, __uint_as_float(v[i + 7]) * inv);
          *reinterpret_cast<uint4*>(stage + lane * 128 + (((i >> 3) ^ (lane & 7)) << 4)) = w;
        }
        __syncwarp();
#pragma unroll
        for (int i = 0; i < 32; i += 4) {
          const int row = i + srow, rr = (warp & 3) * 32 + row, t2 = rr / G;
          const uint4 w = *reinterpret_cast<const uint4*>(stage + row * 128 + ((schunk ^ (row & 7)) << 4));
          if ((rows_ok >> row) & 1)
            *reinterpret_cast<uint4*>(out + ((int64_t)(it.q0 + it.tok0 + qt * TT + t2) * ka.H + it.kvh * G + rr - t2 * G) * HD + c + schunk * 8) = w;
        }
      }
      if (it.split) asm volatile("bar.sync 3, 256;" ::: "memory");     // O1 and the sums are read
      nk += n_item;
    }
  }
  tc_before();
  __syncthreads();
  if (warp == 8) {
    tc_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(512) : "memory");
  }
}

template <int HD>
static int launch(bf16* out, const bf16* q, int q_stride, KvArgs ka, int B, int T, int max_q_len, int max_seq_len, cudaStream_t st) {
  const int G = ka.H / ka.KV, TT = BM / G;
  int by_request = 0;
  ka.per = 2;
  dim3 grid = tc_grid(B, T, max_q_len, ka.per * TT, ka.KV, by_request);
  auto items = [&] { return by_request ? ka.KV * ((int64_t)T / (ka.per * TT) + B) : (int64_t)grid.x * grid.y * grid.z; };
  // One query tile an item and its key tiles shared out (attn_pair.cuh), where items of two tiles leave SMs without work.  us of an item each / two tiles
  // an item, 32 / 8 heads of 128, bfloat16 (float16 within 1 %), requests x rows behind cached keys, items of two tiles:
  //    1 x 64    (8)    9.4 / 10.5      4 x 192 (96)  17.4 / 13.2      1 x 256 + 2000  (32)  45.9 / 62.4
  //    1 x 256  (32)   12.3 / 14.1      4 x 256 (128) 18.5 / 14.5      1 x 512 + 2000  (64)  50.4 / 68.6
  //    1 x 640  (80)   18.4 / 22.5      8 x 128 (128) 17.7 / 12.4      1 x 1024 + 2000 (128) 92.6 / 81.5
  //    1 x 1024 (128)  27.9 / 31.6      4 x 300 (160) 25.8 / 18.1      2 x 512 + 4000  (128)  147 / 116
  //    1 x 1184 (152)  37.2 / 37.1      1 x 2048 (256) 81.4 / 58.7     5 x 256 + 600   (160) 50.5 / 45.4
  // so: up to 74 of them, and up to 148 where contexts are long enough that the last rows' items decide.  Rows behind many more cached keys have items
  // alike: there the second half of that gives up 14 to 27 %.
  if (items() <= 74 || (items() <= 148 && max_seq_len >= 512)) {
    ka.per = 1;
    grid = tc_grid(B, T, max_q_len, ka.per * TT, ka.KV, by_request);
  }
  if (by_request) grid = dim3((unsigned)items());
  ka.flat = by_request ? B : 0;
  CUtensorMap tq8, tq1;
  if (int rc = make_tmap_q(&tq1, q, q_stride, HD, ka.H, G, 1)) return rc;
  tq8 = tq1;
  if (TT >= 8) { if (int rc = make_tmap_q(&tq8, q, q_stride, HD, ka.H, G, 8)) return rc; }
  auto kern = attn_kv4_tc_kernel<HD>;
  KGE_CUDA_OK(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem_bytes<HD>()));
  KGE_CUDA_OK(launch_pdl(kern, grid, dim3(kThreads), smem_bytes<HD>(), st, tq8, tq1, out, ka));
  return 0;
}
}  // namespace atc4

// Requests with more than one token (skip_single), or all of them.
int paged_attn_kv4_tc(bf16* out, const bf16* q, int q_stride, const uint8_t* cache, const int32_t* bt, int max_blocks, const int32_t* sl, const int32_t* qsl, int B, int T,
                      int max_q_len, int max_seq_len, int H, int KV, int hd, int bs, float scale, int window, int first, bool skip_single, cudaStream_t st) {
  atc4::KvArgs ka;
  ka.cache = cache; ka.table = bt; ka.lens = sl; ka.qsl = qsl;
  ka.max_blocks = max_blocks; ka.flat = 0; ka.per = 1; ka.H = H; ka.KV = KV; ka.window = window; ka.first = window > 0 ? first : 0; ka.skip_single = skip_single;
  ka.bs_shift = 4;
  while ((1 << ka.bs_shift) < bs) ++ka.bs_shift;
  ka.scale_log2 = scale * atc::kLog2e;
  const int seen = window > 0 && window < max_seq_len ? window : max_seq_len;
  return hd == 128 ? atc4::launch<128>(out, q, q_stride, ka, B, T, max_q_len, seen, st) : atc4::launch<64>(out, q, q_stride, ka, B, T, max_q_len, seen, st);
}
