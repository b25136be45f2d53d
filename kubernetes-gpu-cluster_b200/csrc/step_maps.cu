// The tables of a step (block table, slots, positions, row offsets) from its requests' lengths, on the GPU: a decode loop that never asks
// the host, or a captured step whose lengths change, needs no metadata copied in.
//
// Three prefix sums over the requests (rows, blocks, and the rows that are left), then one thread per row.  The operations are nothing and
// the bytes little (24 a request, 12 a row): what it costs is its chain - lengths, three sums, a search, a block id.  Every CTA of a cluster
// makes the sums for itself and then takes its share of the rows, so that no CTA waits for another's sums; the cluster's barrier lies
// between the last read of what the caller may pass as output too (lengths, place in the free list) and the first write.
// Back to back 64 requests of a token each take 4.1 us, 512 with 8192 rows 6.0.
#include "common.cuh"
#include "kge.h"

namespace kge {

constexpr int kMapThreads = 512, kMapCtas = 8, kMapRequests = 8192;

struct MapArgs {
  int32_t *table, *lens, *qsl, *positions, *counts;
  int64_t* slots;
  const int32_t *cached, *fresh, *free_blocks, *first;      // (cached may be lens, first may be counts + 2)
  int num_free, max_blocks, B, T, shift;
};

// exclusive sum over the block's threads; `red`: 33 numbers of shared memory; total: of all
__device__ __forceinline__ long long block_excl(long long v, long long* red, long long& total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  long long x = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const long long y = __shfl_up_sync(0xffffffffu, x, o); if (lane >= o) x += y; }
  __syncthreads();
  if (lane == 31) red[warp] = x;
  __syncthreads();
  long long w = lane < nw ? red[lane] : 0, ws = w;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) { const long long y = __shfl_up_sync(0xffffffffu, ws, o); if (lane >= o) ws += y; }
  total = __shfl_sync(0xffffffffu, ws, 31);
  return x - v + (warp ? __shfl_sync(0xffffffffu, ws, warp - 1) : 0);
}

__global__ void __launch_bounds__(kMapThreads) step_maps_kernel(const MapArgs a) {
  extern __shared__ int sh[];
  int *s_c = sh, *s_n = s_c + a.B, *s_at = s_n + a.B, *s_got = s_at + a.B, *s_q = s_got + a.B;      // s_q: [B + 1]
  __shared__ long long red[33];
  pdl_launch_dependents();
  pdl_wait();
  const int rank = (int)blockIdx.x, ctas = (int)gridDim.x, tid = threadIdx.x, bs = 1 << a.shift;
  const int64_t most = (int64_t)a.max_blocks << a.shift;
  const int first = min(max(*a.first, 0), a.num_free);
  for (int b = tid; b < a.B; b += kMapThreads) { s_c[b] = (int)min((int64_t)max(a.cached[b], 0), most); s_n[b] = max(a.fresh[b], 0); }
  __syncthreads();
  const int per = (a.B + kMapThreads - 1) / kMapThreads, lo = min(a.B, tid * per), hi = min(a.B, lo + per);
  long long sum = 0, wanted = 0, total, asked;
  for (int b = lo; b < hi; ++b) { wanted += s_n[b]; s_n[b] = (int)min((int64_t)s_n[b], most - s_c[b]); sum += s_n[b]; }
  block_excl(wanted, red, asked);
  long long run = block_excl(sum, red, total);
  // rows: as many as T has left
  long long need_sum = 0;
  for (int b = lo; b < hi; ++b) {
    const int n = s_n[b];
    s_n[b] = (int)max(0ll, min((long long)n, a.T - run));
    run += n;
    need_sum += ((s_c[b] + (int64_t)s_n[b] + bs - 1) >> a.shift) - ((s_c[b] + (int64_t)bs - 1) >> a.shift);
  }
  // blocks: as many as the list has left, request after request
  long long needed;
  long long at = first + block_excl(need_sum, red, needed);
  long long rows = 0;
  for (int b = lo; b < hi; ++b) {
    const int64_t held = (s_c[b] + (int64_t)bs - 1) >> a.shift, need = ((s_c[b] + (int64_t)s_n[b] + bs - 1) >> a.shift) - held;
    const int64_t got = max((int64_t)0, min(need, (int64_t)(a.num_free - at)));
    if (got < need) s_n[b] = (int)min((int64_t)s_n[b], ((held + got) << a.shift) - s_c[b]);
    s_at[b] = (int)min(at, (long long)a.num_free); s_got[b] = (int)got;
    at += need;
    rows += s_n[b];
  }
  long long all;
  run = block_excl(rows, red, all);
  for (int b = lo; b < hi; ++b) { s_q[b] = (int)run; run += s_n[b]; }
  if (tid == 0) s_q[a.B] = (int)all;
  if (ctas > 1) { cluster_arrive_relaxed(); cluster_wait(); }
  __syncthreads();
  const int rows_all = (int)all;
  for (int t = rank * kMapThreads + tid; t < a.T; t += ctas * kMapThreads) {
    int pos = 0;
    int64_t slot = -1;
    if (t < rows_all) {
      int l = 0, h = a.B;                              // the last request that begins at or before t and has rows
      while (h - l > 1) { const int m = (l + h) >> 1; if (s_q[m] <= t) l = m; else h = m; }
      const int c = s_c[l];
      pos = c + t - s_q[l];
      const int i = pos >> a.shift, held = (int)((c + (int64_t)bs - 1) >> a.shift);
      const int blk = i < held ? a.table[(int64_t)l * a.max_blocks + i] : a.free_blocks[s_at[l] + i - held];
      slot = ((int64_t)blk << a.shift) + (pos & (bs - 1));
    }
    a.positions[t] = pos;
    a.slots[t] = slot;
  }
  // table entries: a warp a request
  const int lane = tid & 31;
  for (int b = rank * (kMapThreads / 32) + (tid >> 5); b < a.B; b += ctas * (kMapThreads / 32)) {
    const int held = (int)((s_c[b] + (int64_t)bs - 1) >> a.shift);
    for (int i = lane; i < s_got[b]; i += 32) a.table[(int64_t)b * a.max_blocks + held + i] = a.free_blocks[s_at[b] + i];
  }
  if (rank == 0) {
    for (int b = tid; b < a.B; b += kMapThreads) { a.lens[b] = s_c[b] + s_n[b]; a.qsl[b] = s_q[b]; }
    if (tid == 0) {
      const int taken = (int)min(needed, (long long)(a.num_free - first));
      a.qsl[a.B] = rows_all;
      a.counts[0] = rows_all;
      a.counts[1] = (int)min(asked, 0x7fffffffll);
      a.counts[2] = first + taken;
      a.counts[3] = (int)(needed - taken);
    }
  }
}

}  // namespace kge

using namespace kge;

extern "C" int kge_step_maps(int32_t* block_table, int max_blocks_per_seq, int32_t* seq_lens, int32_t* query_start_loc, int32_t* positions, int64_t* slot_mapping,
                             int32_t* counts, const int32_t* cached_lens, const int32_t* new_lens, const int32_t* free_blocks, int num_free, const int32_t* free_first, int B,
                             int T, int block_size, void* stream) {
  KGE_REQUIRE(block_table && seq_lens && query_start_loc && positions && slot_mapping && counts && cached_lens && new_lens && free_first && (free_blocks || num_free == 0),
              "kge_step_maps: null pointer");
  KGE_REQUIRE(block_size > 0 && (block_size & (block_size - 1)) == 0, "kge_step_maps: block_size=%d must be a power of two", block_size);
  KGE_REQUIRE(B >= 0 && B <= kMapRequests, "kge_step_maps: %d requests (at most %d)", B, kMapRequests);
  KGE_REQUIRE(T >= 0 && T <= (1 << 30) && num_free >= 0 && max_blocks_per_seq > 0 && (int64_t)max_blocks_per_seq * block_size < (1ll << 31),
              "kge_step_maps: %d rows, %d free blocks, %d blocks of %d tokens a request", T, num_free, max_blocks_per_seq, block_size);
  MapArgs a;
  a.table = block_table; a.lens = seq_lens; a.qsl = query_start_loc; a.positions = positions; a.counts = counts; a.slots = slot_mapping;
  a.cached = cached_lens; a.fresh = new_lens; a.free_blocks = free_blocks; a.first = free_first;
  a.num_free = num_free; a.max_blocks = max_blocks_per_seq; a.B = B; a.T = T; a.shift = 0;
  while ((1 << a.shift) < block_size) ++a.shift;
  const size_t smem = (size_t)(5 * B + 1) * 4;
  // (48 KB would hold the kernel's static shared memory too, so every launch says what the largest needs)
  KGE_CUDA_OK(cudaFuncSetAttribute(step_maps_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (5 * kMapRequests + 1) * 4));
  const int ctas = T > 2 * kMapThreads ? kMapCtas : 1;
  prefer_max_shared(step_maps_kernel);
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(kMapThreads); cfg.dynamicSmemBytes = smem; cfg.stream = (cudaStream_t)stream;
  cudaLaunchAttribute attr[2];
  int n = 0;
  if (ctas > 1) {
    attr[n].id = cudaLaunchAttributeClusterDimension;
    attr[n].val.clusterDim.x = ctas; attr[n].val.clusterDim.y = 1; attr[n].val.clusterDim.z = 1;
    ++n;
  }
  if (pdl_for_this_launch()) {
    attr[n].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[n].val.programmaticStreamSerializationAllowed = 1;
    ++n;
  }
  cfg.attrs = attr; cfg.numAttrs = n;
  KGE_CUDA_OK(cudaLaunchKernelEx(&cfg, step_maps_kernel, a));
  return 0;
}
