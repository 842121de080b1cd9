// Page copies and pool compaction: pages of the paged K/V pools (and an INT8
// pool's scales) moved inside the pools, in every layer by one launch.
//
// Bound: each copied byte is read and written once, so the floor is twice the
// pages' bytes of HBM.  Whole pages are copied with eight 16-byte loads in
// flight per thread: 256 pages x 16 layers (bf16, 32 KB) in 89.5 us (0.92 of
// the measured copy rate), 93.7 us with four; 1900 moves of a compaction 151 us
// against 157.  Two CTAs of 256 threads an SM are enough and more are worse
// (four: 94.9 and 185 us).  Pages in rows take four loads and four CTAs.
#include "page_copy.cuh"

namespace pa {
namespace {

constexpr int kBatch = 128;  // pairs a CTA checks at once
constexpr int kTable = 256;  // hash slots of a batch's targets

// Pair j takes part when its ids are in range, differ, and it copies a slot.
__device__ __forceinline__ bool pair_active(int s, int d, int slots, const PageParams& g) {
  return s != d && s >= 0 && s < g.num_blocks && d >= 0 && d < g.num_blocks && slots > 0 && slots <= g.block_size;
}

__device__ __forceinline__ int hash_find(const int* key, int id) {
  int h = (id * 0x9E3779B1u) >> 24;
  while (key[h] != id && key[h] != -1) h = (h + 1) & (kTable - 1);
  return key[h] == id ? h : -1;
}

// A CTA owns a contiguous range of (pair, layer, K or V, part) items.  Two
// pairs with one target, or a target that another pair reads, would race: of
// pairs with the same target the first is copied, and a pair whose target is
// another's source is not; both report PA_STATUS_COPY_OVERLAP.  Each CTA
// checks its own pairs against the whole list.
template <int LOADS>
__global__ void __launch_bounds__(kCopyThreads, LOADS == 8 ? 1 : 4) copy_blocks_kernel(const PageParams g, const int* src, const int* dst,
                                                                   const int* num_slots, int pairs, int* status) {
  pdl_enter();
  __shared__ int key[kTable], first[kTable], read[kTable];
  __shared__ bool ok[kBatch];
  const int per_pair = g.layers * 2 * g.parts;
  const long long items = static_cast<long long>(pairs) * per_pair;
  long long item = items * blockIdx.x / gridDim.x;
  const long long end = items * (blockIdx.x + 1) / gridDim.x;
  while (item < end) {
    const int p0 = static_cast<int>(item / per_pair);
    const int p1 = min(static_cast<int>((end - 1) / per_pair) + 1, p0 + kBatch);
    for (int i = threadIdx.x; i < kTable; i += kCopyThreads) {
      key[i] = -1;
      first[i] = 0x7fffffff;
      read[i] = 0;
    }
    __syncthreads();
    for (int i = p0 + threadIdx.x; i < p1; i += kCopyThreads) {
      const int s = src[i], d = dst[i], n = num_slots ? num_slots[i] : g.block_size;
      if (pair_active(s, d, n, g)) {
        int h = (d * 0x9E3779B1u) >> 24;
        for (;;) {
          const int was = atomicCAS(&key[h], -1, d);
          if (was == -1 || was == d) break;
          h = (h + 1) & (kTable - 1);
        }
      } else if (s != d && n != 0) {
        set_status(status, n < 0 || n > g.block_size ? ST_BAD_POSITION : ST_BAD_BLOCK_ID);
      }
    }
    __syncthreads();
    for (int j = threadIdx.x; j < pairs; j += kCopyThreads) {
      const int s = src[j], d = dst[j], n = num_slots ? num_slots[j] : g.block_size;
      if (!pair_active(s, d, n, g)) continue;
      int h = hash_find(key, d);
      if (h >= 0) atomicMin(&first[h], j);
      h = hash_find(key, s);
      if (h >= 0) read[h] = 1;
    }
    __syncthreads();
    for (int i = p0 + threadIdx.x; i < p1; i += kCopyThreads) {
      const int d = dst[i], n = num_slots ? num_slots[i] : g.block_size;
      bool good = pair_active(src[i], d, n, g);
      if (good) {
        const int h = hash_find(key, d);
        good = first[h] == i && !read[h];
        if (!good) set_status(status, ST_COPY_OVERLAP);
      }
      ok[i - p0] = good;
    }
    __syncthreads();
    const long long stop = min(end, static_cast<long long>(p1) * per_pair);
    for (; item < stop; ++item) {
      const int pair = static_cast<int>(item / per_pair);
      if (!ok[pair - p0]) continue;
      int r = static_cast<int>(item - static_cast<long long>(pair) * per_pair);
      const int part = r % g.parts;
      r /= g.parts;
      copy_page<LOADS>(g, r >> 1, r & 1, src[pair], dst[pair], num_slots ? num_slots[pair] : g.block_size, part);
    }
    __syncthreads();
  }
}

// ---- compaction -----------------------------------------------------------------
// Scratch words: [2] pages to move, [3] live pages, [4] 1 when the pool was
// refused; after the bitmap of freed blocks map[NB] (new id of a moved page, else -1), src[NB], dst[NB].
constexpr int kPlanThreads = 1024;
constexpr int kPlanIds = 4;  // ids of a thread per round

__device__ __forceinline__ int block_prefix(int mine, int* warp_sum, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int inc = mine;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(0xffffffffu, inc, o);
    if (lane >= o) inc += v;
  }
  if (lane == 31) warp_sum[warp] = inc;
  __syncthreads();
  if (warp == 0) {
    int w = lane < static_cast<int>(blockDim.x >> 5) ? warp_sum[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, w, o);
      if (lane >= o) w += v;
    }
    warp_sum[lane] = w;
  }
  __syncthreads();
  const int before = (warp ? warp_sum[warp - 1] : 0) + inc - mine;
  *total = warp_sum[31];
  __syncthreads();
  return before;
}

// One CTA: planning 8192 blocks takes 8 us of a compaction's 168.  A single launch
// in which every resident CTA planned for itself (a bitmap of live blocks, moves
// by rank) took 182 us: its copies have no later CTAs to even out the SMs.
// Live pages are counted, then the holes below that count and the live pages
// at or above it are listed in ascending order: page src[i] moves to dst[i].
__global__ void __launch_bounds__(kPlanThreads) compact_plan_kernel(const PoolParams p, const ShareParams s, int after,
                                                                    int* live_out, int* status) {
  pdl_enter();
  __shared__ int warp_sum[32];
  int* map = s.scratch + kShareHead + (p.num_blocks + 31) / 32;
  int* src = map + p.num_blocks;
  int* dst = src + p.num_blocks;
  int mine = 0, live;
  for (int i = threadIdx.x; i < p.num_blocks; i += kPlanThreads) mine += s.ref[i] > 0;
  block_prefix(mine, warp_sum, &live);
  int moves = 0, holes = 0;
  if (live <= after) {
    for (int base = 0; base < p.num_blocks; base += kPlanThreads * kPlanIds) {
      const int id0 = base + threadIdx.x * kPlanIds;
      unsigned hole = 0, move = 0;
#pragma unroll
      for (int e = 0; e < kPlanIds; ++e) {
        const int id = id0 + e;
        if (id < p.num_blocks) {
          const bool used = s.ref[id] > 0;
          map[id] = -1;
          if (!used && id < live) hole |= 1u << e;
          if (used && id >= live) move |= 1u << e;
        }
      }
      // a thread's ids hold at most kPlanIds of each, a round far fewer than 2^16: both counts in one word
      int total;
      const int at = block_prefix(__popc(hole) | (__popc(move) << 16), warp_sum, &total);
      int h = holes + (at & 0xffff), m = moves + (at >> 16);
#pragma unroll
      for (int e = 0; e < kPlanIds; ++e) {
        if (hole >> e & 1) dst[h++] = id0 + e;
        if (move >> e & 1) src[m++] = id0 + e;
      }
      holes += total & 0xffff;
      moves += total >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < moves; i += kPlanThreads) map[src[i]] = dst[i];
  }
  if (threadIdx.x == 0) {
    s.scratch[2] = moves;
    s.scratch[3] = live;
    s.scratch[4] = live > after;
    if (live_out) *live_out = live;
    if (live > after) set_status(status, ST_BAD_POOL);
  }
}

// The planned moves.  `first`: the tables too (later launches carry further
// layers).  A moved page's holes and sources are disjoint, so nothing waits.
template <int LOADS>
__global__ void __launch_bounds__(kCopyThreads, LOADS == 8 ? 1 : 4) compact_move_kernel(const PoolParams p, const ShareParams s, int after,
                                                                    const PageParams g, int* status, bool first) {
  pdl_enter();
  const int* map = s.scratch + kShareHead + (p.num_blocks + 31) / 32;
  const int* src = map + p.num_blocks;
  const int* dst = src + p.num_blocks;
  const int moves = s.scratch[2], live = s.scratch[3];
  if (s.scratch[4]) return;
  if (first) {
    for (int row = blockIdx.x; row < p.max_seqs; row += gridDim.x) {
      const int c = min(p.count[row], p.max_blocks_per_seq);
      int* ids = p.table + row * p.table_stride;
      for (int j = threadIdx.x; j < c; j += kCopyThreads) {
        const int id = ids[j];
        if (id < 0 || id >= p.num_blocks) set_status(status, ST_BAD_BLOCK_ID);
        else if (id >= live && map[id] < 0) set_status(status, ST_BAD_POOL);  // held by a row, but not counted
        else if (id >= live) ids[j] = map[id];
      }
    }
    const int at = blockIdx.x * kCopyThreads + threadIdx.x, step = gridDim.x * kCopyThreads;
    for (int i = at; i < moves; i += step) {
      s.ref[dst[i]] = s.ref[src[i]];
      s.ref[src[i]] = 0;
    }
    // the lowest free id is handed out first
    for (int i = at; i < after - live; i += step) p.free_stack[i] = after - 1 - i;
    if (at == 0) *p.free_top = after - live;
  }
  const int per_page = g.layers * 2 * g.parts;
  const long long items = static_cast<long long>(moves) * per_page;
  for (long long item = blockIdx.x; item < items; item += gridDim.x) {
    const int i = static_cast<int>(item / per_page);
    int r = static_cast<int>(item - static_cast<long long>(i) * per_page);
    const int part = r % g.parts;
    r /= g.parts;
    copy_page<LOADS>(g, r >> 1, r & 1, src[i], dst[i], g.block_size, part);
  }
}

}  // namespace

cudaError_t launch_copy_blocks(const PageParams& g, const int* src, const int* dst, const int* num_slots, int pairs,
                               int* status, cudaStream_t stream) {
  const long long items = static_cast<long long>(pairs) * g.layers * 2 * g.parts;
  if (items <= 0) return cudaSuccess;
  const long long most = 8LL * device_sm_count();
  const bool run = page_is_run(g, num_slots == nullptr);
  cudaError_t e = launch_pdl(run ? copy_blocks_kernel<8> : copy_blocks_kernel<4>, dim3(static_cast<unsigned>(items < most ? items : most)),
                             dim3(kCopyThreads), 0, stream, g, src, dst, num_slots, pairs, status);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_block_pool_compact(const PoolParams& p, const ShareParams& s, int num_blocks_after, int* live,
                                      const PageParams& g, int* status, cudaStream_t stream, bool first) {
  if (first) {
    cudaError_t e = launch_pdl(compact_plan_kernel, dim3(1), dim3(kPlanThreads), 0, stream, p, s, num_blocks_after,
                               live, status);
    if (e != cudaSuccess) return e;
  }
  cudaError_t e = launch_pdl(page_is_run(g, true) ? compact_move_kernel<8> : compact_move_kernel<4>, dim3(8 * device_sm_count()), dim3(kCopyThreads), 0, stream, p, s,
                             num_blocks_after, g, status, first);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace pa
