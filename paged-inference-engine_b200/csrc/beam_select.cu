// Beam selection: the best `num_out` continuations of each sequence's beams
// over the vocabulary.
//
// For sequence b, beam k and token v
//   score(b, k, v) = beam_score[b, k] + x[b, k, v] - log sum_u exp(x[b, k, u])
// and the outputs are the num_out largest, ordered by score, then lower beam,
// then larger logit, then lower token.  A finished beam's row counts as
// log-probability 0 at eos_id and -inf elsewhere and is not read.  NaN logits
// count as -inf, +inf as the largest float.
//
// Measured (B200): 64 x 8 rows of 131072 bf16 logits in 36 us (134 MB, 20.6 us of
// HBM), 6 x 16 rows of 65536 fp16 in 14.7, one sequence of 4 rows of 32000 in 7.3
// in a captured graph and 12 through the op.  Rows with fewer finite logits than
// T needs in a part (masks) take a second, slower look: 294 us for the first of
// these with 50 tokens a row allowed.
//
// Bound: every logit is read once, so the floor is rows * vocab * size bytes
// of HBM; next comes the one exponential per logit (16 a clock and SM: 0.77 of
// the HBM time for 16-bit logits).  Two launches: `beam_rows_kernel` streams a
// part of a row through registers, each thread with its own running maximum
// and sum, and no barrier until the part's end; `beam_merge_kernel` joins the
// parts and the beams of one sequence.
//
// The best logits come from the maxima that the softmax needs anyway.  The
// threads' maxima are joined in groups; with T the num_out-th largest of the
// groups' maxima, num_out logits are at least T, so the best are among the
// logits that are, and only the threads whose maximum reaches T have their
// logits looked at again (for 16 of 32768 independent logits: 22 threads of
// 256; each remembers the maxima of 8 spans, so it reads one of them, from L2).
// Selection compares (logit, token) as one 64-bit integer, so it is exact
// whatever the order of the threads; the sum's order depends on the logits'
// places in the row alone, not on its address, so equal rows have equal sums.
#include "pa_common.cuh"

#include <cfloat>
#include <cmath>
#include <type_traits>

namespace pa {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowCtas = 5;            // resident on an SM
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kLaneRuns = 4;            // runs of 16 bytes of a lane per chunk
constexpr int kLogLaneRuns = 2;
constexpr int kChunkRuns = 32 * kLaneRuns;
constexpr int kUnitRuns = kRowWarps * kChunkRuns;  // a chunk of every warp: the grain in which rows are split
constexpr int kStages = 2;             // chunks of a warp in shared memory
constexpr int kPartUnits = 32;         // units of a part at most: a thread's sum is rounded, and perhaps rescaled, once a unit
constexpr int kSpans = 8;              // a thread's units are remembered in so many spans, by their maxima
constexpr int kHits = kRowWarps * kMaxBeamOut;  // logits at T that a part may have; with more its warps keep sorted lists
constexpr int kMergeThreads = 512;
constexpr int kMergeWarps = kMergeThreads / 32;
constexpr int kNoGroup = static_cast<int>(0x80000000u);  // below every float in this order
constexpr int kMergeKeys = 8192;        // candidates that the merge holds in shared memory (20 bytes each)
constexpr float kLog2e = 1.4426950408889634f;

template <int DT>
constexpr int logit_bytes() {
  return DT == PA_DTYPE_F32 ? 4 : 2;
}

__device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -INFINITY), FLT_MAX) + 0.f; }  // NaN, +inf, -0

// (logit, token) as one integer: larger logit first, then the lower token.  0 is below every candidate.
__device__ __forceinline__ unsigned long long make_key(float x, unsigned token) {
  const unsigned u = __float_as_uint(clean(x));
  const unsigned o = u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u);
  return (static_cast<unsigned long long>(o) << 32) | (0xffffffffu - token);
}
__device__ __forceinline__ float key_logit(unsigned long long k) {
  const unsigned o = static_cast<unsigned>(k >> 32);
  return __uint_as_float(o ^ ((o >> 31) ? 0x80000000u : 0xffffffffu));
}
__device__ __forceinline__ int key_token(unsigned long long k) {
  return static_cast<int>(0xffffffffu - static_cast<unsigned>(k));
}

// The logits of a 4-byte word: one in fp32 (the second counts as -inf), two in 16 bits.
template <int DT>
__device__ __forceinline__ float2 word_logits(uint32_t w) {
  if constexpr (DT == PA_DTYPE_F32) return make_float2(__uint_as_float(w), -INFINITY);
  else if constexpr (DT == PA_DTYPE_BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  else return __half22float2(*reinterpret_cast<const __half2*>(&w));
}
template <int DT>
__device__ __forceinline__ uint32_t word_max(uint32_t a, uint32_t b) {  // NaN gives way
  if constexpr (DT == PA_DTYPE_F32) {
    return __float_as_uint(fmaxf(__uint_as_float(a), __uint_as_float(b)));
  } else if constexpr (DT == PA_DTYPE_BF16) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  } else {
    const __half2 m = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
    return *reinterpret_cast<const uint32_t*>(&m);
  }
}
template <int DT>
constexpr uint32_t word_lowest() {  // -inf
  return DT == PA_DTYPE_F32 ? 0xff800000u : DT == PA_DTYPE_BF16 ? 0xff80ff80u : 0xfc00fc00u;
}

// 32 values, one per lane, from large to small.
__device__ __forceinline__ float sort_lanes(float v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
    for (int step = size >> 1; step > 0; step >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, step);
      v = (((lane & size) == 0) == ((lane & step) == 0)) ? fmaxf(v, o) : fminf(v, o);
    }
  }
  return v;
}

struct RowShared {
  unsigned long long hit[kHits];
  float peak[kRowWarps][32], sum[kRowWarps];  // peak: the threads' maxima
  float top, limit;
  int count;                                  // of hit
};

// The n-th largest of 64 groups' values, two (a, b) in each lane; for n <= 16 of
// the 32 lanes' larger ones, which is enough (the n-th of n groups would be
// their smallest, and four times n values reach it).  `top`: the largest.
__device__ __forceinline__ float nth_group(float a, float b, int n, float& top) {
  const int lane = threadIdx.x & 31;
  float v;
  if (n <= 16) {
    v = sort_lanes(fmaxf(a, b));
  } else {
    v = fmaxf(sort_lanes(a), __shfl_sync(0xffffffffu, sort_lanes(b), 31 - lane));  // the 32 largest, falling and rising
#pragma unroll
    for (int step = 16; step > 0; step >>= 1) {
      const float o = __shfl_xor_sync(0xffffffffu, v, step);
      v = (lane & step) == 0 ? fmaxf(v, o) : fminf(v, o);
    }
  }
  top = __shfl_sync(0xffffffffu, v, 0);
  return __shfl_sync(0xffffffffu, v, n - 1);
}

// Run j of a row is its 16 bytes with logits [j PER, (j + 1) PER).  `base` is the
// row's start rounded down to 16 bytes and `lead` (in bytes) what that left
// off: run j lies in the aligned pieces j and j + 1 of base.
__device__ __forceinline__ uint4 shift_run(const uint4& a, const uint4& b, int lead) {
  uint32_t x[8] = {a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w};
#pragma unroll
  for (int i = 0; i < 6; ++i) x[i] = lead & 8 ? x[i + 2] : x[i];
#pragma unroll
  for (int i = 0; i < 5; ++i) x[i] = lead & 4 ? x[i + 1] : x[i];
  const unsigned pick = lead & 2 ? 0x5432 : 0x3210;
  return make_uint4(__byte_perm(x[0], x[1], pick), __byte_perm(x[1], x[2], pick), __byte_perm(x[2], x[3], pick),
                    __byte_perm(x[3], x[4], pick));
}

template <int DT>
struct Row {
  static constexpr int SZ = logit_bytes<DT>();
  static constexpr int PER = 16 / SZ;
  const char* first;
  const uint4* base;
  int lead, vocab;
  int safe0, safe1;  // runs [safe0, safe1) lie in pieces that belong to the row entirely

  __device__ __forceinline__ Row(const BeamParams& p, int row) {
    const int b = row / p.beams;
    first = static_cast<const char*>(p.logits) +
            (b * p.stride_seq + static_cast<long long>(row - b * p.beams) * p.stride_beam) * SZ;
    lead = static_cast<int>(reinterpret_cast<uintptr_t>(first) & 15);
    base = reinterpret_cast<const uint4*>(first - lead);
    vocab = p.vocab;
    safe0 = lead ? 1 : 0;
    safe1 = (vocab + lead / SZ) / PER - safe0;
  }
  __device__ __forceinline__ float one(int i) const {
    if constexpr (DT == PA_DTYPE_F32) return reinterpret_cast<const float*>(first)[i];
    else if constexpr (DT == PA_DTYPE_BF16) return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(first)[i]);
    else return __half2float(reinterpret_cast<const __half*>(first)[i]);
  }
  // Run j, with -inf past the row's end.
  __device__ __forceinline__ uint4 run(int j) const {
    if (j >= safe0 && j < safe1) return lead ? shift_run(__ldg(base + j), __ldg(base + j + 1), lead) : __ldg(base + j);
    uint32_t w[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      if constexpr (SZ == 4) {
        const int i = j * PER + k;
        w[k] = i < vocab ? reinterpret_cast<const uint32_t*>(first)[i] : word_lowest<DT>();
      } else {
        const int i = j * PER + 2 * k;
        const uint16_t* r = reinterpret_cast<const uint16_t*>(first);
        const uint32_t low = word_lowest<DT>() & 0xffffu;
        w[k] = (i < vocab ? r[i] : low) | (i + 1 < vocab ? r[i + 1] : low) << 16;
      }
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// N runs into a thread's maximum m and its sum s of exp(x - m); returns their maximum.
template <int DT, int N>
__device__ __forceinline__ float take_runs(const uint4 (&u)[N], float& m, float& s) {
  uint32_t a = word_max<DT>(u[0].x, u[0].y), b = word_max<DT>(u[0].z, u[0].w);
#pragma unroll
  for (int i = 1; i < N; ++i) {
    a = word_max<DT>(word_max<DT>(a, u[i].x), u[i].y);
    b = word_max<DT>(word_max<DT>(b, u[i].z), u[i].w);
  }
  const float2 f = word_logits<DT>(word_max<DT>(a, b));
  const float top = fminf(fmaxf(fmaxf(f.x, f.y), -INFINITY), FLT_MAX);  // both NaN: -inf
  if (top > m) {
    s *= ex2((m - top) * kLog2e);
    m = top;
  }
  const float ref = fmaxf(m, -FLT_MAX);
  auto all = [&](auto&& term) {  // term: of two logits, as a pair
    uint64_t part[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const uint32_t w[4] = {u[i].x, u[i].y, u[i].z, u[i].w};
      if constexpr (DT == PA_DTYPE_F32) {
        part[0] = f2_add(part[0], term(__uint_as_float(w[0]), __uint_as_float(w[1])));
        part[1] = f2_add(part[1], term(__uint_as_float(w[2]), __uint_as_float(w[3])));
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const float2 g = word_logits<DT>(w[k]);
          part[k & 1] = f2_add(part[k & 1], term(g.x, g.y));
        }
      }
    }
    float a, b;
    f2_unpack(f2_add(part[0], part[1]), a, b);
    return a + b;
  };
  // exp(x - ref) = 2^(x L + c) 2^e with c = -ref L rounded and e what that left off: at most 2^-11 for these ref, so
  // that 1 + e ln 2 is 2^e to 2^-24
  const float c = -ref * kLog2e, e = fmaf(-ref, kLog2e, -c);
  float sum = NAN;
  if (fabsf(ref) < 8192.f) {
    const uint64_t scale = f2_pack(kLog2e, kLog2e), shift = f2_pack(c, c);
    sum = all([&](float x, float y) {
      float a, b;
      f2_unpack(f2_fma(f2_pack(x, y), scale, shift), a, b);
      return f2_pack(ex2(a), ex2(b));
    });
    sum = fmaf(sum, e * 0.6931472f, sum);
  }
  if (!(sum <= FLT_MAX)) {  // NaN, +inf, or a larger maximum: the difference first
    sum = all([&](float x, float y) { return f2_pack(ex2((clean(x) - ref) * kLog2e), ex2((clean(y) - ref) * kLog2e)); });
  }
  s += sum;
  return top;
}

// The warp's list (lane i: the i-th largest key) takes the lanes' keys above its n-th.
__device__ __forceinline__ void insert_keys(unsigned long long& list, int n, bool hit, unsigned long long key) {
  const int lane = threadIdx.x & 31;
  unsigned long long last = __shfl_sync(0xffffffffu, list, n - 1);
  unsigned todo = __ballot_sync(0xffffffffu, hit && key > last);
  while (todo) {
    const int from = __ffs(todo) - 1;
    const unsigned long long k = __shfl_sync(0xffffffffu, key, from);
    const int place = __popc(__ballot_sync(0xffffffffu, list > k));
    const unsigned long long up = __shfl_up_sync(0xffffffffu, list, 1);
    if (lane == place) list = k;
    else if (lane > place) list = up;
    last = __shfl_sync(0xffffffffu, list, n - 1);
    todo = __ballot_sync(0xffffffffu, hit && key > last) & ~((2u << from) - 1);
  }
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads, kRowCtas) beam_rows_kernel(const BeamParams p) {
  pdl_enter();
  constexpr int PER = Row<DT>::PER, SZ = Row<DT>::SZ;
  extern __shared__ uint4 ring[];  // [warp][stage][kChunkRuns + 1] pieces, then spans' maxima [span][thread]
  __shared__ RowShared sh;
  const int n = p.num_out;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int runs = (p.vocab + PER - 1) / PER;
  uint4* const mine = ring + warp * kStages * (kChunkRuns + 1);
  const int row = blockIdx.x, out = row * p.parts + blockIdx.y;
  if (p.finished && p.finished[row]) return;
  const Row<DT> r(p, row);
  const int u0 = blockIdx.y * p.part_units, u1 = min(p.row_units, u0 + p.part_units);
  if (tid == 0) sh.count = 0;
  // ---- maximum and sum over the units [u0, u1) of the row, in each a chunk for
  // every warp.  Chunks whose pieces all belong to the row come through the
  // warp's own ring of asynchronous copies; the row's ends are read run by run.
  __nv_bfloat16* const peaks = reinterpret_cast<__nv_bfloat16*>(ring + kRowWarps * kStages * (kChunkRuns + 1));
  float m = -INFINITY, s = 0.f, span = -INFINITY;
  auto start = [&](int u) { return u * kUnitRuns + warp * kChunkRuns; };
  auto ringed = [&](int u) { return start(u) >= r.safe0 && start(u) + kChunkRuns <= r.safe1; };
  auto stream = [&](auto shifts) {  // shifts: the row starts off a 16-byte boundary
    auto fetch = [&](int u, int stage) {  // one commit group, empty where there is nothing to fetch
      if (u < u1 && ringed(u)) {
        const uint4* src = r.base + start(u) + lane;
        const uint32_t dst = smem_u32(mine + stage * (kChunkRuns + 1) + lane);
#pragma unroll
        for (int k = 0; k < kLaneRuns; ++k) cp_async_16(dst + 512 * k, src + 32 * k, 16);
        if (shifts && lane == 0) cp_async_16(dst + 512 * kLaneRuns, src + kChunkRuns, 16);
      }
      cp_async_commit();
    };
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) fetch(u0 + i, i);
    int stage = 0;
    for (int u = u0; u < u1; ++u) {
      __syncwarp();  // the stage before this one has been read
      fetch(u + kStages - 1, stage == 0 ? kStages - 1 : stage - 1);
      cp_async_wait<kStages - 1>();
      __syncwarp();
      uint4 x[kLaneRuns];
      if (ringed(u)) {
        const uint4* src = mine + stage * (kChunkRuns + 1) + lane;
#pragma unroll
        for (int k = 0; k < kLaneRuns; ++k) x[k] = src[32 * k];
        if (shifts) {
#pragma unroll
          for (int k = 0; k < kLaneRuns; ++k) x[k] = shift_run(x[k], src[32 * k + 1], r.lead);
        }
      } else {
#pragma unroll
        for (int k = 0; k < kLaneRuns; ++k) x[k] = r.run(start(u) + 32 * k + lane);
      }
      const float top = take_runs<DT, kLaneRuns>(x, m, s);
      span = ((u - u0) & ((1 << p.log_span) - 1)) == 0 ? top : fmaxf(span, top);
      peaks[((u - u0) >> p.log_span) * kRowThreads + tid] = __float2bfloat16_ru(span);
      stage = stage + 1 == kStages ? 0 : stage + 1;
    }
  };
  if (r.lead) stream(std::true_type());
  else stream(std::false_type());
  sh.peak[warp][lane] = m;
  __syncthreads();
  if (warp == 0) {
    // a group for each lane, of the even and of the odd warps: a part that leaves warps without logits has every group
    float a = sh.peak[0][lane], b = sh.peak[1][lane], top;
#pragma unroll
    for (int w = 2; w < kRowWarps; w += 2) {
      a = fmaxf(a, sh.peak[w][lane]);
      b = fmaxf(b, sh.peak[w + 1][lane]);
    }
    const float limit = nth_group(a, b, n, top);
    if (lane == 0) {
      sh.top = fminf(top, FLT_MAX);
      sh.limit = limit;
    }
  }
  __syncthreads();
  // ---- the spans whose maximum reaches T, of this warp's threads whose own does
  const float top = sh.top, limit = sh.limit;
  unsigned short* const list = reinterpret_cast<unsigned short*>(mine);  // the warp is through with its ring
  const int spans = ((u1 - u0 - 1) >> p.log_span) + 1;
  int listed = 0;
  for (unsigned todo = __ballot_sync(0xffffffffu, m >= limit); todo; todo &= todo - 1) {
    const int t = __ffs(todo) - 1;
    const bool in = lane < spans && __bfloat162float(peaks[lane * kRowThreads + warp * 32 + t]) >= limit;
    const unsigned some = __ballot_sync(0xffffffffu, in);
    if (in) list[listed + __popc(some & ((1u << lane) - 1))] = static_cast<unsigned short>(lane * 32 + t);
    listed += __popc(some);
  }
  __syncwarp();
  // ---- their runs once more, a lane for each; few hold a logit at T
  const int log_each = p.log_span + kLogLaneRuns, items = listed << log_each;
  auto run_of = [&](int i) {  // of item i; past every row where there is none
    if (i >= items) return runs;
    const int entry = list[i >> log_each], e = i & ((1 << log_each) - 1);
    const int u = u0 + (entry / 32 << p.log_span) + (e >> kLogLaneRuns);
    return u < u1 ? start(u) + e % kLaneRuns * 32 + entry % 32 : runs;
  };
  int j = run_of(lane);
  uint4 x = make_uint4(0, 0, 0, 0);
  if (j < runs) x = r.run(j);
  s *= ex2((m - fmaxf(top, -FLT_MAX)) * kLog2e);  // the part's sum, while that comes
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) sh.sum[warp] = s;
  for (int i0 = 0; i0 < items; i0 += 32) {
    if (i0) {
      j = run_of(i0 + lane);
      if (j < runs) x = r.run(j);
    }
    const float2 f = word_logits<DT>(word_max<DT>(word_max<DT>(x.x, x.y), word_max<DT>(x.z, x.w)));
    if (j >= runs || fmaxf(f.x, f.y) < limit) continue;
    const uint32_t w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int e = 0; e < PER; ++e) {
      const float2 g = word_logits<DT>(w[e * SZ / 4]);
      const float v = SZ == 2 && (e & 1) ? g.y : g.x;
      if ((v >= limit || limit == -INFINITY) && j * PER + e < p.vocab) {
        const int at = atomicAdd(&sh.count, 1);
        if (at < kHits) sh.hit[at] = make_key(v, j * PER + e);
      }
    }
  }
  __syncthreads();
  int count = sh.count;
  if (count > kHits) {  // many equal logits: each warp keeps its n best
    unsigned long long best = 0;
    for (int i0 = 0; i0 < items; i0 += 32 / PER) {  // a lane for each logit of 32 / PER runs
      const int j = run_of(i0 + lane / PER);
      const int i = j < runs ? j * PER + lane % PER : p.vocab;
      const float v = i < p.vocab ? r.one(i) : 0.f;
      insert_keys(best, n, i < p.vocab && (v >= limit || limit == -INFINITY), make_key(v, i));
    }
    __syncthreads();
    if (lane < n) sh.hit[warp * n + lane] = best;
    count = kRowWarps * n;
    __syncthreads();
  }
  if (tid == 0) {
    float total = 0.f;
    for (int w = 0; w < kRowWarps; ++w) total += sh.sum[w];
    p.part_max[out] = top;
    p.part_sum[out] = total;
  }
  // ---- a key's place is the number of keys above it, counted by eight lanes
  unsigned long long* keys = p.part_key + static_cast<long long>(out) * n;
  if (tid < n && tid >= count) keys[tid] = 0;
  for (int i0 = warp * 4; i0 < count; i0 += kRowThreads / 8) {
    const int i = i0 + (lane >> 3);
    const unsigned long long key = i < count ? sh.hit[i] : 0;
    int place = 0;
    for (int q = lane & 7; q < count; q += 8) place += sh.hit[q] > key || (sh.hit[q] == key && q < i);
#pragma unroll
    for (int o = 4; o; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
    if (i < count && place < n && (lane & 7) == 0) keys[place] = key;
  }
}

// One CTA per sequence: the n best of its beams' parts.  Scores are compared in
// 64 bits: candidates of different beams lie as near as their logits' rounding,
// and -50 + x - lse in 32 bits would swap them.  Only candidates that may be
// among the n best get there: as in the rows, T is the n-th largest of groups'
// maxima, here of scores in fp32 and less their rounding.  A part's list is
// sorted, so the groups mix ranks and lists.
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamParams p) {
  extern __shared__ unsigned long long dyn[];
  const int b = blockIdx.x, K = p.beams, S = p.parts, n = p.num_out;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = S * n, total = K * per;
  unsigned long long* keys = dyn;                             // every candidate's
  double* score = reinterpret_cast<double*>(keys + total);    // of the candidates at T
  int* which = reinterpret_cast<int*>(score + total);
  __shared__ double top[kMaxBeams], logsum[kMaxBeams];  // apart: beside a maximum of 1e30 the logarithm would vanish
  __shared__ float ftop[kMaxBeams], offset[kMaxBeams];
  __shared__ int group[64], count;
  __shared__ float limit_of_all, largest_offset;
  const int row0 = b * K;
  if (tid < 64) group[tid] = kNoGroup;
  if (tid == 0) count = 0;
  pdl_enter();
  // rows and lists of candidate i, by multiplication (total < 2^14: exact)
  const unsigned per_inv = (1u << 28) / per + 1, n_inv = (1u << 28) / n + 1;
  auto over = [](int i, unsigned inv) { return static_cast<int>((static_cast<unsigned long long>(i) * inv) >> 28); };
  auto load_key = [&](int i) -> unsigned long long {
    const int k = over(i, per_inv), r = i - k * per;
    if (!(p.finished && p.finished[row0 + k])) return p.part_key[static_cast<long long>(row0) * per + i];
    if (r >= n || r >= p.vocab) return 0;
    return make_key(r == 0 ? 0.f : -INFINITY, r == 0 ? p.eos : r - 1 + (r - 1 >= p.eos));  // eos, then the others at -inf
  };
  constexpr int kFirst = 4;  // keys on their way while the sums are joined
  unsigned long long first[kFirst];
#pragma unroll
  for (int q = 0; q < kFirst; ++q) {
    const int i = tid + q * kMergeThreads;
    first[q] = i < total ? load_key(i) : 0;
  }
  for (int k = warp; k < K; k += kMergeWarps) {
    const bool fin = p.finished && p.finished[row0 + k];
    const int parts = fin ? 0 : S, at = (row0 + k) * S;
    float m = lane < parts ? p.part_max[at + lane] : -INFINITY;
    float t = lane < parts ? p.part_sum[at + lane] : 0.f;
    const float base = p.scores[row0 + k];
    float M = m;
    for (int i = lane + 32; i < parts; i += 32) M = fmaxf(M, p.part_max[at + i]);
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    double sum = t > 0.f ? t * exp(static_cast<double>(m) - static_cast<double>(M)) : 0.0;
    for (int i = lane + 32; i < parts; i += 32) {
      t = p.part_sum[at + i];
      if (t > 0.f) sum += t * exp(static_cast<double>(p.part_max[at + i]) - static_cast<double>(M));
    }
    if (S > 1) {
#pragma unroll
      for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    }
    if (lane == 0) {
      // a row of -inf has no sum: all its scores are -inf; a finished beam's are 0 and -inf
      const double log_sum = sum > 0.0 ? log(sum) : 0.0;
      top[k] = sum > 0.0 ? M : 0.0;
      ftop[k] = sum > 0.0 ? M : 0.f;
      logsum[k] = log_sum;
      offset[k] = static_cast<float>(base - log_sum);
    }
  }
#pragma unroll
  for (int q = 0; q < kFirst; ++q) {
    const int i = tid + q * kMergeThreads;
    if (i < total) keys[i] = first[q];
  }
  for (int i = tid + kFirst * kMergeThreads; i < total; i += kMergeThreads) keys[i] = load_key(i);
  __syncthreads();
  auto rough = [&](int i, int k) {
    const float v = (key_logit(keys[i]) - ftop[k]) + offset[k];
    return v == v ? v : -INFINITY;
  };
  for (int i = tid; i < total; i += kMergeThreads) {
    if (!keys[i]) continue;
    const int list = over(i, n_inv), r = i - list * n;
    const int f = __float_as_int(rough(i, over(i, per_inv)) + 0.f);
    atomicMax(&group[(r + 11 * list) & 63], f >= 0 ? f : f ^ 0x7fffffff);  // floats in their order
  }
  __syncthreads();
  if (warp == 0) {
    auto value = [](int g) { return g == kNoGroup ? -INFINITY : __int_as_float(g >= 0 ? g : g ^ 0x7fffffff); };
    float largest;
    const float v = nth_group(value(group[lane]), value(group[32 + lane]), n, largest);
    if (lane == 0) limit_of_all = v;
  }
  if (warp == 1) {  // the largest finite |offset|; floats of no sign lie in the order of their bits
    const float o = lane < K ? fabsf(offset[lane]) : 0.f;
    const unsigned most = __reduce_max_sync(0xffffffffu, o <= FLT_MAX ? __float_as_uint(o) : 0u);
    if (lane == 0) largest_offset = __uint_as_float(most);
  }
  __syncthreads();
  const float limit = limit_of_all, coarse = fabsf(limit) + largest_offset;
  for (int i = tid; i < total; i += kMergeThreads) {
    const unsigned long long key = keys[i];
    const int k = over(i, per_inv);
    bool hit = key != 0;
    if (hit) {
      const float v = rough(i, k);
      // offset, x - top and their sum are rounded here, and in the n candidates at the limit, of any beam:
      // each time by at most 2^-24 of |offset| + |sum|, and no sum is larger than its offset
      const float slack = 4.f * 1.2e-7f * (coarse + fabsf(v));
      hit = v >= limit || (v > -INFINITY && !(limit - v > slack));
    }
    if (!hit) continue;
    const int at = atomicAdd(&count, 1);
    const double v = static_cast<double>(p.scores[row0 + k]) + ((static_cast<double>(key_logit(key)) - top[k]) - logsum[k]);
    score[at] = v == v ? v : -INFINITY;  // NaN counts as -inf
    which[at] = i;
  }
  __syncthreads();
  // a candidate's place is the number of candidates before it, counted by eight lanes
  const int have = count;
  for (int i0 = warp * 4; i0 < have; i0 += kMergeThreads / 8) {
    const int i = i0 + (lane >> 3);
    const bool in = i < have;
    const double v = in ? score[i] : 0.0;
    const int c = in ? which[i] : 0, k = over(c, per_inv);
    int place = 0;
    for (int q = lane & 7; q < have; q += 8) {
      const double o = score[q];
      if (o > v) ++place;
      if (o == v) {
        const int d = which[q], l = over(d, per_inv);
        place += l < k || (l == k && keys[d] > keys[c]);
      }
    }
#pragma unroll
    for (int o = 4; o; o >>= 1) place += __shfl_xor_sync(0xffffffffu, place, o);
    if (in && place < n && (lane & 7) == 0) {
      const long long o = static_cast<long long>(b) * n + place;
      p.out_scores[o] = static_cast<float>(v);
      p.out_tokens[o] = key_token(keys[c]);
      p.out_parents[o] = k;
    }
  }
}

}  // namespace

// Parts of a row: the number that leaves the fewest SMs idle at the rows
// kernel's end, with a unit's time added to each part for its selection; the
// merge's shared memory bounds it, and the sums' accuracy asks for enough.  With U
// units a thread's sum is rounded U + 23 times (10 in a unit, 13 where threads
// and warps are joined) by 2^-24 of its size and rescaled U + 1 times with 2^-22
// more; exponentials and their arguments add 113 times 2^-24.  6 U + 141 of
// those are 2e-5 for U = 32.
long long beam_vocab_limit(int beams, int num_out, int dtype) {
  const int per = dtype == PA_DTYPE_F32 ? 4 : 8;
  const long long most = (kMergeKeys / (static_cast<long long>(beams) * num_out)) * kPartUnits * kUnitRuns * per;
  return most < 1 << 30 ? most : 1 << 30;
}

void beam_plan(BeamParams& p, int dtype) {
  const int per = dtype == PA_DTYPE_F32 ? 4 : 8;
  const long long rows = static_cast<long long>(p.seqs) * p.beams;
  const long long runs = (static_cast<long long>(p.vocab) + per - 1) / per;
  const long long units = (runs + kUnitRuns - 1) / kUnitRuns;
  const long long slots = static_cast<long long>(kRowCtas) * device_sm_count();
  const long long fit = kMergeKeys / (static_cast<long long>(p.beams) * p.num_out);
  long long least = 0;
  const long long fewest = (units + kPartUnits - 1) / kPartUnits;
  for (long long parts = fewest; parts <= units && parts <= fit; ++parts) {
    const long long share = (units + parts - 1) / parts, used = (units + share - 1) / share;
    const long long cost = (rows * used + slots - 1) / slots * (share + 1);
    if (parts == fewest || cost < least) {
      least = cost;
      p.part_units = static_cast<int>(share);
      p.parts = static_cast<int>(used);
    }
  }
  p.row_units = static_cast<int>(units);
  p.log_span = 0;
  while ((p.part_units - 1) >> p.log_span >= kSpans) ++p.log_span;
}

template <int DT>
cudaError_t launch_rows(const BeamParams& p, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  const int ring = kRowWarps * kStages * (kChunkRuns + 1) * 16;
  const int smem = ring + (((p.part_units - 1) >> p.log_span) + 1) * kRowThreads * 2;
  cudaError_t e = allow_smem(beam_rows_kernel<DT>, ring + kSpans * kRowThreads * 2, done);
  if (e != cudaSuccess) return e;
  return launch_pdl(beam_rows_kernel<DT>, dim3(p.seqs * p.beams, p.parts), dim3(kRowThreads), smem, stream, p);
}

cudaError_t launch_beam_select(const BeamParams& p, int dtype, cudaStream_t stream) {
  static std::atomic<unsigned long long> done{0};
  cudaError_t e = allow_smem(beam_merge_kernel, kMergeKeys * 20 + 8, done);
  if (e != cudaSuccess) return e;
  e = dtype == PA_DTYPE_F32    ? launch_rows<PA_DTYPE_F32>(p, stream)
      : dtype == PA_DTYPE_BF16 ? launch_rows<PA_DTYPE_BF16>(p, stream)
                               : launch_rows<PA_DTYPE_F16>(p, stream);
  if (e != cudaSuccess) return e;
  const size_t smem = static_cast<size_t>(p.beams) * p.parts * p.num_out * 20 + 8;
  e = launch_pdl(beam_merge_kernel, dim3(p.seqs), dim3(kMergeThreads), smem, stream, p);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace pa
