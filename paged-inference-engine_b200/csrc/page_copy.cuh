// Copying pages inside the paged pools: the address arithmetic shared by the
// page-copy, beam-reorder and compaction kernels.
#pragma once

#include "pa_common.cuh"

namespace pa {

constexpr int kCopyThreads = 256;
constexpr int kCopyLoads = 4;  // 16-byte loads in flight per thread

// Byte offset of 16-byte vector `v` of a page's first `slots` slots.
__device__ __forceinline__ long long page_vec(const PageParams& g, const PageSide& s, int v, int slots, bool linear) {
  if (linear) return 16LL * v;
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

// Part `part` of the copy of the first `slots` slots of page src to page dst,
// of layer `layer`'s K (kv 0) or V (kv 1) pool, by all threads of the CTA.
// Part 0 takes the page's scales too; a scale per block goes with any slot.
__device__ __forceinline__ void copy_page(const PageParams& g, int layer, int kv, int src, int dst, int slots, int part) {
  const PageSide& s = g.side[kv];
  const char* from = g.page[kv][layer] + src * s.blk;
  char* to = g.page[kv][layer] + dst * s.blk;
  const int vecs = (slots * g.heads) << g.row_vecs_log2;
  const int per = (((g.block_size * g.heads) << g.row_vecs_log2) + g.parts - 1) / g.parts;
  const int end = min(vecs, (part + 1) * per);
  const bool linear = s.linear || (s.dense && slots == g.block_size);
  for (int v0 = part * per + threadIdx.x; v0 < end; v0 += kCopyThreads * kCopyLoads) {
    uint4 w[kCopyLoads];
    long long at[kCopyLoads];
#pragma unroll
    for (int i = 0; i < kCopyLoads; ++i) {
      const int v = v0 + i * kCopyThreads;
      at[i] = page_vec(g, s, v, slots, linear);
      if (v < end) w[i] = *reinterpret_cast<const uint4*>(from + at[i]);
    }
#pragma unroll
    for (int i = 0; i < kCopyLoads; ++i)
      if (v0 + i * kCopyThreads < end) *reinterpret_cast<uint4*>(to + at[i]) = w[i];
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
