// Copying pages inside the paged pools: the address arithmetic shared by the
// page-copy, beam-reorder and compaction kernels.
#pragma once

#include "pa_common.cuh"

namespace pa {

constexpr int kCopyThreads = 256;

// Whether what is copied of every page is one run of memory.
inline bool page_is_run(const PageParams& g, bool whole) {
  return (g.side[0].linear && g.side[1].linear) || (whole && g.side[0].dense && g.side[1].dense);
}

// Byte offset of 16-byte vector `v` of a page's first `slots` slots.
__device__ __forceinline__ long long page_vec(const PageParams& g, const PageSide& s, int v, int slots) {
  const int row = v >> g.row_vecs_log2;
  int slot, head;
  if (s.slot_fast) {
    head = row / slots;
    slot = row - head * slots;
  } else {
    slot = row / g.heads;
    head = row - slot * g.heads;
  }
  return slot * s.slot + head * s.head + 16LL * (v & ((1 << g.row_vecs_log2) - 1));
}

// N vectors in flight per thread, from vector v0 on.
template <int N, typename At>
__device__ __forceinline__ void copy_vecs(const char* from, char* to, int v0, int end, At&& at) {
  uint4 w[N];
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int v = v0 + i * kCopyThreads;
    if (v < end) w[i] = *reinterpret_cast<const uint4*>(from + at(v));
  }
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int v = v0 + i * kCopyThreads;
    if (v < end) *reinterpret_cast<uint4*>(to + at(v)) = w[i];
  }
}

// The first N vectors per thread that copy_page will read of page src, into L2.
template <int N>
__device__ __forceinline__ void prefetch_page(const PageParams& g, int layer, int kv, int src, int slots, int part) {
  const PageSide& s = g.side[kv];
  const char* from = g.page[kv][layer] + src * s.blk;
  const int vecs = (slots * g.heads) << g.row_vecs_log2;
  const int per = (vecs + g.parts - 1) / g.parts;
  const int begin = part * per + threadIdx.x, end = min(vecs, (part + 1) * per);
  const bool run = s.linear || (s.dense && slots == g.block_size);
#pragma unroll
  for (int i = 0; i < N; ++i) {
    const int v = begin + i * kCopyThreads;
    if (v < end) asm volatile("prefetch.global.L2 [%0];" ::"l"(from + (run ? 16LL * v : page_vec(g, s, v, slots))));
  }
}

// Part `part` of the copy of the first `slots` slots of page src to page dst,
// of layer `layer`'s K (kv 0) or V (kv 1) pool, by all threads of the CTA.
// Part 0 takes the page's scales too; a scale per block goes with any slot.
// LOADS: 16-byte loads in flight per thread; with 8 the page is known to be one
// run of memory (page_is_run).
template <int LOADS>
__device__ __forceinline__ void copy_page(const PageParams& g, int layer, int kv, int src, int dst, int slots, int part) {
  const PageSide& s = g.side[kv];
  const char* from = g.page[kv][layer] + src * s.blk;
  char* to = g.page[kv][layer] + dst * s.blk;
  const int vecs = (slots * g.heads) << g.row_vecs_log2;
  const int per = (vecs + g.parts - 1) / g.parts;
  const int begin = part * per + threadIdx.x, end = min(vecs, (part + 1) * per);
  if (LOADS == 8 || s.linear || (s.dense && slots == g.block_size)) {
    for (int v = begin; v < end; v += kCopyThreads * LOADS)
      copy_vecs<LOADS>(from, to, v, end, [](int u) { return 16LL * u; });
  } else {
    for (int v = begin; v < end; v += kCopyThreads * LOADS)
      copy_vecs<LOADS>(from, to, v, end, [&](int u) { return page_vec(g, s, u, slots); });
  }
  if (g.scale[kv][layer] && part == 0 && slots > 0) {
    const char* sf = g.scale[kv][layer] + src * s.sblk;
    char* st = g.scale[kv][layer] + dst * s.sblk;
    const int n = (s.sslot ? slots : 1) * g.heads;
    for (int i = threadIdx.x; i < n; i += kCopyThreads) {
      const int slot = i / g.heads, head = i - slot * g.heads;
      const long long o = slot * s.sslot + head * s.shead;
      if (g.scale_bytes == 4) *reinterpret_cast<uint32_t*>(st + o) = *reinterpret_cast<const uint32_t*>(sf + o);
      else *reinterpret_cast<uint16_t*>(st + o) = *reinterpret_cast<const uint16_t*>(sf + o);
    }
  }
}

}  // namespace pa
