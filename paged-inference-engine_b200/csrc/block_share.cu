// Sharing of pool blocks between sequences: reference counts beside the block
// pool, forks that share full blocks, and the reordering of beams.
//
// A block is written only while one sequence holds it: a fork shares the
// blocks its tokens fill and copies a partly filled last block, so no later
// append meets a shared block.  The reference's allocator has no sharing
// (core/block_manager.py:19-68: every id belongs to one sequence).
//
// Integer work on a few kilobytes; the page copies of a reorder are the only
// large traffic (both bytes of each copied token, once).  64 groups of 8 beams
// with 4 forks each, 4 layers of 64 KB pages: 28 us for 130 MB (20 us of HBM);
// one group: 6 us, a chain of seven dependent accesses.
#include "page_copy.cuh"

namespace pa {
namespace {

constexpr int kApplyThreads = 256;
constexpr int kColumns = 1024;  // table columns of one CTA

// Exclusive prefix of a flag over the CTA's kApplyThreads threads.
__device__ __forceinline__ int flag_prefix(bool flag, int* warp_sum, int* total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const unsigned mask = __ballot_sync(0xffffffffu, flag);
  if (lane == 0) warp_sum[warp] = __popc(mask);
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kApplyThreads / 32; ++w) {
    if (w < warp) before += warp_sum[w];
    all += warp_sum[w];
  }
  __syncthreads();
  *total = all;
  return before + __popc(mask & ((1u << lane) - 1));
}

__global__ void share_init_kernel(int* ref, int num_blocks, int* scratch, long long words) {
  pdl_enter();
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i < num_blocks) ref[i] = 0;
  if (i < words) scratch[i] = 0;
}

// ops[4 i + {0..3}] = (kind, slot, n, parent), in order:
//   ALLOCATE  n new blocks, each with one holder
//   RELEASE   one holder less for each of the slot's blocks; those without any
//             are pushed in list order
//   FORK      slot (without an entry) gets the first n tokens of `parent`: the
//             full blocks shared, and for a partly filled last one a new block
//             and the copy (copy_src[i], copy_dst[i], copy_slots[i])
// Operations without a copy leave a pair of equal ids.
__global__ void __launch_bounds__(kApplyThreads) apply_shared_kernel(const PoolParams p, const ShareParams s,
                                                                     const int* ops, int n_ops, int block_size,
                                                                     int* results, int* copy_src, int* copy_dst,
                                                                     int* copy_slots) {
  pdl_enter();
  __shared__ int s_top, warp_sum[kApplyThreads / 32];
  if (threadIdx.x == 0) s_top = *p.free_top;
  __syncthreads();
  for (int i = 0; i < n_ops; ++i) {
    const int kind = ops[4 * i], slot = ops[4 * i + 1], n = ops[4 * i + 2], parent = ops[4 * i + 3];
    const int top = s_top;
    int res = POOL_INVALID, new_top = top, new_count = 0;
    int from = 0, to = 0, part = 0;
    const bool known = (kind == POOL_ALLOC || kind == POOL_RELEASE || kind == POOL_FORK) && slot >= 0 &&
                       slot < p.max_seqs && n >= 0 && top >= 0 && top <= p.num_blocks;
    if (known) {
      int* row = p.table + static_cast<long long>(slot) * p.table_stride;
      const int c = p.count[slot];
      if (kind == POOL_ALLOC) {
        const int base = c < 0 ? 0 : c;
        if (top < n) {
          res = POOL_INSUFFICIENT_SPACE;
        } else if (static_cast<long long>(base) + n > p.max_blocks_per_seq) {
          res = POOL_ROW_FULL;
        } else {
          for (int j = threadIdx.x; j < n; j += kApplyThreads) {
            const int id = p.free_stack[top - 1 - j];
            row[base + j] = id;
            if (id >= 0 && id < p.num_blocks) s.ref[id] = 1;
          }
          res = POOL_SUCCESS;
          new_top = top - n;
          new_count = base + n;
        }
      } else if (kind == POOL_RELEASE) {
        if (c < 0) {
          res = POOL_FAILURE;
        } else if (c <= p.max_blocks_per_seq) {
          for (int j0 = 0; j0 < c; j0 += kApplyThreads) {
            const int j = j0 + threadIdx.x;
            const int id = j < c ? row[j] : -1;
            bool last = false;
            if (id >= 0 && id < p.num_blocks) last = --s.ref[id] == 0;  // a row holds an id once
            int freed;
            const int at = new_top + flag_prefix(last, warp_sum, &freed);
            if (last && at < p.num_blocks) p.free_stack[at] = id;
            new_top = min(new_top + freed, p.num_blocks);
          }
          res = POOL_SUCCESS;
          new_count = -1;
        }
      } else {
        const int pc = parent >= 0 && parent < p.max_seqs ? p.count[parent] : -1;
        const int full = n / block_size, tail = n - full * block_size;
        const int have = full + (tail > 0);
        if (pc < 0 || c >= 0) {
          res = POOL_FAILURE;
        } else if (have > pc || have > p.max_blocks_per_seq) {
          res = POOL_ROW_FULL;
        } else if (tail && top < 1) {
          res = POOL_INSUFFICIENT_SPACE;
        } else {
          const int* old = p.table + static_cast<long long>(parent) * p.table_stride;
          for (int j = threadIdx.x; j < full; j += kApplyThreads) {
            const int id = old[j];
            row[j] = id;
            if (id >= 0 && id < p.num_blocks) s.ref[id] += 1;
          }
          if (tail) {
            from = old[full];
            to = p.free_stack[top - 1];
            part = tail;
            if (threadIdx.x == 0) {
              row[full] = to;
              if (to >= 0 && to < p.num_blocks) s.ref[to] = 1;
            }
          }
          res = POOL_SUCCESS;
          new_top = top - (tail > 0);
          new_count = have;
        }
      }
      __syncthreads();  // every thread has read count / the stack before they change
      if (res == POOL_SUCCESS && threadIdx.x == 0) {
        p.count[slot] = new_count;
        s_top = new_top;
      }
    }
    if (threadIdx.x == 0) {
      if (results) results[i] = res;
      if (copy_src) {
        copy_src[i] = from;
        copy_dst[i] = to;
        copy_slots[i] = part;
      }
    }
    __syncthreads();  // the next operation sees this one's stack, counts and rows
  }
  if (threadIdx.x == 0) *p.free_top = s_top;
}

// ---- beams ------------------------------------------------------------------------
// Beam j of group g continues beam parents[g][j].  The first child of a
// parent keeps the parent's pool row; the other children take the rows of the
// beams without children, both in ascending order of beam.  Rows of parents
// therefore never change, and a child's row changes only against its donor's.
struct Forks {
  int child[kMaxBeams], donor[kMaxBeams];  // pool rows of the n forks
  int src[kMaxBeams], dst[kMaxBeams];      // their partly filled blocks
  int n, full, tail;                       // full blocks and tokens of the last one
};

// By warp 0; lane j stands for beam j: its row afterwards, and the holders of its row's partly filled block, which its
// copy and the next token write, so that a group with any other than 1 is left as it is too (ST_BAD_POOL).  That count
// is not waited for here: a CTA that copies has its first loads under way meanwhile.  Returns a status, 0 if the group's
// arguments hold.
__device__ __forceinline__ int plan_group(const PoolParams& p, const ShareParams& s, const ReorderParams& r, int log2BS,
                                          int g, Forks& f, int& row, int& holders) {
  const int lane = threadIdx.x & 31, K = r.beams;
  const bool on = lane < K;
  const int slot = on ? r.slots[g * K + lane] : -1 - lane;
  const int parent = on ? r.parents[g * K + lane] : -1 - lane;
  const int tokens = r.num_tokens[g];
  const int bs = 1 << log2BS;
  const bool in_range = !on || (slot >= 0 && slot < p.max_seqs && parent >= 0 && parent < K);
  const bool alone = __match_any_sync(0xffffffffu, slot) == (1u << lane);
  const bool named = __all_sync(0xffffffffu, in_range && alone);
  int bad = named ? 0 : ST_BAD_SEQ_INDEX;
  const int full = tokens >> log2BS;
  int last = 0;  // the row's partly filled block
  if (named) {
    if (on && tokens > 0 && full < p.max_blocks_per_seq) last = p.table[slot * p.table_stride + full];
    const int c = on ? p.count[slot] : 0;
    const int c0 = __shfl_sync(0xffffffffu, c, 0);
    const long long need = tokens < 0 ? -1 : (static_cast<long long>(tokens) + bs - 1) >> log2BS;
    if (!__all_sync(0xffffffffu, !on || c == c0) || need < 0 || need > c0 || c0 > p.max_blocks_per_seq)
      bad = ST_BAD_POSITION;
  }
  if (bad) return bad;
  const int tail = tokens & (bs - 1);
  const bool counted = on && tail && last >= 0 && last < p.num_blocks;
  holders = counted ? __ldcg(&s.ref[last]) : 1;
  const unsigned same = __match_any_sync(0xffffffffu, parent);
  const bool again = on && (same & ((1u << lane) - 1));
  const unsigned forks = __ballot_sync(0xffffffffu, again);
  const unsigned alive = __reduce_or_sync(0xffffffffu, on ? 1u << parent : 0u);
  const unsigned spare = ~alive & (K == 32 ? 0xffffffffu : (1u << K) - 1);
  const int nth = __popc(forks & ((1u << lane) - 1));
  const int donor = __shfl_sync(0xffffffffu, slot, on ? parent : 0);
  const int taken = again ? __fns(spare, 0, nth + 1) : 0;
  const int child = __shfl_sync(0xffffffffu, slot, taken & 31);
  const int src = __shfl_sync(0xffffffffu, last, on ? parent : 0);
  const int dst = __shfl_sync(0xffffffffu, last, taken & 31);
  if (again) {
    f.child[nth] = child;
    f.donor[nth] = donor;
    f.src[nth] = src;
    f.dst[nth] = dst;
  }
  if (lane == 0) {
    f.n = __popc(forks);
    f.full = full;
    f.tail = tail;
  }
  row = again ? child : donor;
  return 0;
}

// The first groups * chunks CTAs share full blocks (a CTA for kColumns table
// columns of a group, a thread for whole columns: a block stands in the same
// column of every row that holds it, so all changes of its count within a
// group come from one thread); the others copy the forks' last blocks, which
// no table change touches.  Freed blocks are marked in a bitmap, and the last
// table CTA pushes them in ascending order, so the stack does not depend on
// the order in which CTAs run.
__global__ void __launch_bounds__(kCopyThreads, 5) reorder_kernel(const PoolParams p, const ShareParams s,
                                                               const ReorderParams r, const PageParams g, int log2BS,
                                                               int chunks, int shares) {
  pdl_enter();
  __shared__ Forks f;
  __shared__ bool ok, writable, last;
  __shared__ int warp_sum[kApplyThreads / 32];
  const int tables = r.groups * chunks;
  int row, holders;
  if (static_cast<int>(blockIdx.x) >= tables) {
    const int cta = blockIdx.x - tables, share = cta % shares, fork = cta / shares;
    const int nth = fork / r.groups, group = fork - nth * r.groups;  // groups' first forks first: few groups have K - 1
    if (threadIdx.x < 32) {
      const int bad = plan_group(p, s, r, log2BS, group, f, row, holders);
      if (threadIdx.x == 0) ok = bad == 0;
    }
    __syncthreads();
    if (!ok || nth >= f.n || f.tail == 0) return;
    const int src = f.src[nth], dst = f.dst[nth];
    if (src < 0 || src >= g.num_blocks || dst < 0 || dst >= g.num_blocks) {
      if (threadIdx.x == 0) set_status(r.status, ST_BAD_BLOCK_ID);
      return;
    }
    const int items = g.layers * 2 * g.parts, begin = items * share / shares;
    prefetch_page<4>(g, begin / g.parts >> 1, begin / g.parts & 1, src, f.tail, begin % g.parts);
    if (threadIdx.x < 32) {
      const bool sole = __all_sync(0xffffffffu, holders == 1);
      if (threadIdx.x == 0) writable = sole;
    }
    __syncthreads();
    if (!writable) return;
    for (int i = begin; i < items * (share + 1) / shares; ++i)
      copy_page<4>(g, i / g.parts >> 1, i / g.parts & 1, src, dst, f.tail, i % g.parts);
    return;
  }

  const int group = blockIdx.x / chunks, chunk = blockIdx.x - group * chunks;
  unsigned* bitmap = reinterpret_cast<unsigned*>(s.scratch + kShareHead);
  if (threadIdx.x < 32) {
    int bad = plan_group(p, s, r, log2BS, group, f, row, holders);
    if (!bad && !__all_sync(0xffffffffu, holders == 1)) bad = ST_BAD_POOL;
    const int at = group * r.beams + threadIdx.x;
    if (chunk == 0 && static_cast<int>(threadIdx.x) < r.beams) r.slots_out[at] = bad ? r.slots[at] : row;
    if (chunk == 0 && threadIdx.x == 0 && bad) set_status(r.status, bad);
    if (threadIdx.x == 0) ok = bad == 0;
  }
  __syncthreads();
  if (ok) {
    const int end = min(f.full, (chunk + 1) * kColumns);
    for (int c = chunk * kColumns + threadIdx.x; c < end; c += kCopyThreads) {
      for (int i = 0; i < f.n; ++i) {
        int* mine = p.table + f.child[i] * p.table_stride + c;
        const int was = *mine, now = p.table[f.donor[i] * p.table_stride + c];
        if (was == now) continue;
        if (was < 0 || was >= p.num_blocks || now < 0 || now >= p.num_blocks) {
          set_status(r.status, ST_BAD_BLOCK_ID);
          continue;
        }
        *mine = now;
        atomicAdd(&s.ref[now], 1);
        if (atomicSub(&s.ref[was], 1) == 1) {
          atomicOr(&bitmap[was >> 5], 1u << (was & 31));
          atomicAdd(&s.scratch[1], 1);
        }
      }
    }
  }
  __threadfence();
  __syncthreads();
  if (threadIdx.x == 0) last = atomicAdd(&s.scratch[0], 1) == tables - 1;
  __syncthreads();
  if (!last) return;
  __threadfence();
  const int freed = *const_cast<volatile int*>(&s.scratch[1]);
  if (freed > 0) {
    int top = *p.free_top;
    const int words = (p.num_blocks + 31) / 32;
    for (int w0 = 0; w0 < words; w0 += kCopyThreads) {
      const int w = w0 + threadIdx.x;
      const unsigned bits = w < words ? __ldcg(&bitmap[w]) : 0;
      // the words' bit counts, one bit of the count at a time
      int before = 0, total = 0;
#pragma unroll
      for (int b = 0; b < 6; ++b) {
        int t;
        const int at = flag_prefix(__popc(bits) >> b & 1, warp_sum, &t);
        before += at << b;
        total += t << b;
      }
      if (total == 0) continue;
      int at = top + before;
      for (unsigned m = bits; m; m &= m - 1, ++at)
        if (at >= 0 && at < p.num_blocks) p.free_stack[at] = 32 * w + __ffs(m) - 1;
      if (bits) bitmap[w] = 0;
      top += total;
    }
    if (threadIdx.x == 0) *p.free_top = min(top, p.num_blocks);
  }
  if (threadIdx.x == 0) {
    s.scratch[0] = 0;
    s.scratch[1] = 0;
  }
}

}  // namespace

cudaError_t launch_block_pool_init_shared(const PoolParams& p, const ShareParams& s, long long scratch_words,
                                          cudaStream_t stream) {
  const long long n = scratch_words > p.num_blocks ? scratch_words : p.num_blocks;
  cudaError_t e = launch_block_pool_init(p, stream);
  if (e != cudaSuccess) return e;
  e = launch_pdl(share_init_kernel, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, stream, s.ref,
                 p.num_blocks, s.scratch, scratch_words);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_block_pool_apply_shared(const PoolParams& p, const ShareParams& s, const int* ops, int n_ops,
                                           int block_size, int* results, int* copy_src, int* copy_dst, int* copy_slots,
                                           cudaStream_t stream) {
  if (n_ops <= 0) return cudaSuccess;
  cudaError_t e = launch_pdl(apply_shared_kernel, dim3(1), dim3(kApplyThreads), 0, stream, p, s, ops, n_ops, block_size,
                             results, copy_src, copy_dst, copy_slots);
  return e != cudaSuccess ? e : cudaGetLastError();
}

cudaError_t launch_block_pool_reorder(const PoolParams& p, const ShareParams& s, const ReorderParams& r,
                                      const PageParams& g, cudaStream_t stream, bool first) {
  const int chunks = !first ? 0 : p.max_blocks_per_seq > kColumns ? (p.max_blocks_per_seq + kColumns - 1) / kColumns : 1;
  // A fork's copies are shared by so many CTAs that all forks together, half of
  // the beams perhaps, fill every SM twice: planning a group costs a CTA more than
  // 1 us, and partly filled blocks differ in size.  With 4, 8, 16 and 32 CTAs an SM:
  // 64 groups of 8 beams, 4 layers of 64 KB pages 32.0, 30.5, 29.9 and 33.7 us; 16
  // layers of 32 KB 55.9, 49.5, 49.3 and 50.4; 16 x 6, 4 x 4, 64 x 4 and 1 x 4
  // within 0.1 us of one another.
  const long long items = g.layers * 2LL * g.parts, forks = static_cast<long long>(r.groups) * (r.beams - 1);
  long long shares = forks ? (16LL * device_sm_count() + forks - 1) / forks : 1;
  shares = shares < items ? shares : items;
  const long long ctas = static_cast<long long>(r.groups) * chunks + forks * shares;
  if (ctas <= 0) return cudaSuccess;
  int log2BS = 0;
  while ((1 << log2BS) < g.block_size) ++log2BS;
  cudaError_t e = launch_pdl(reorder_kernel, dim3(static_cast<unsigned>(ctas)), dim3(kCopyThreads), 0, stream, p, s, r,
                             g, log2BS, chunks, static_cast<int>(shares));
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace pa
