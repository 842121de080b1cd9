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
// Bound: every logit is read once, so the floor is rows * vocab * size bytes
// of HBM.  Two launches: `beam_rows_kernel` streams each row in S splits, with
// the running maximum, the sum of exponentials and the best num_out logits of
// its split kept on chip; `beam_merge_kernel` joins the splits and the beams of
// one sequence.  Row selection compares (logit, token) as one 64-bit integer,
// so it is exact whatever the order of the threads.
#include "pa_common.cuh"

#include <cfloat>
#include <cmath>

namespace pa {
namespace {

constexpr int kRowThreads = 256;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kVec = 4;             // 16-byte loads a thread has in flight per tile
constexpr int kMergeThreads = 512;
constexpr int kMaxSplits = 32;      // one lane per split when sums are joined
constexpr float kLog2e = 1.4426950408889634f;

template <int DT>
struct Logit {
  static constexpr int kBytes = DT == PA_DTYPE_F32 ? 4 : 2;
  static constexpr int kPer = 16 / kBytes;      // logits of a 16-byte load
  static constexpr int kMine = kVec * kPer;     // logits of a thread per tile
};

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

template <int DT>
__device__ __forceinline__ float load_one(const void* row, long long i) {
  if constexpr (DT == PA_DTYPE_F32) return static_cast<const float*>(row)[i];
  else if constexpr (DT == PA_DTYPE_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(row)[i]);
  else return __half2float(static_cast<const __half*>(row)[i]);
}

template <int DT>
__device__ __forceinline__ void unpack(const uint4& w, float* f) {
  const uint32_t a[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (DT == PA_DTYPE_F32) {
      f[i] = __uint_as_float(a[i]);
    } else if constexpr (DT == PA_DTYPE_BF16) {
      f[2 * i] = __uint_as_float(a[i] << 16);
      f[2 * i + 1] = __uint_as_float(a[i] & 0xffff0000u);
    } else {
      const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&a[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

// Position of `key` in a list sorted from large to small: entries above it.
__device__ __forceinline__ int count_above(const unsigned long long* list, int n, unsigned long long key) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (list[mid] > key) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

struct RowShared {
  unsigned long long sorted[kRowWarps][32];
  unsigned long long buf[(kMaxBeamOut + 1) * 33];  // at most kMaxBeamOut threads' logits and the list
  unsigned long long top[kMaxBeamOut];
  unsigned long long limit;
  float m[kRowWarps], s[kRowWarps];
  int count;
};

// Vector `vec` of a row whose first logit is number `lead` of its 16-byte
// aligned vector 0.  A vector that reaches over an end of the row or of the
// split is left to loads of single logits (`edge`).
template <int DT>
__device__ __forceinline__ void load_vec(const char* base, int vec, int vend, int lead, int vocab, uint4& raw, bool& edge) {
  constexpr int PER = Logit<DT>::kPer;
  const int first = vec * PER - lead;
  edge = vec >= vend || first < 0 || first + PER > vocab;
  if (!edge) raw = __ldcs(reinterpret_cast<const uint4*>(base) + vec);
}

template <int DT>
__global__ void __launch_bounds__(kRowThreads, 4) beam_rows_kernel(const BeamParams p) {
  pdl_enter();
  using L = Logit<DT>;
  __shared__ RowShared sh;
  const int row = blockIdx.x, split = blockIdx.y;
  if (p.finished && p.finished[row]) return;
  const int b = row / p.beams;
  const long long at = b * p.stride_seq + static_cast<long long>(row - b * p.beams) * p.stride_beam;
  const char* first = static_cast<const char*>(p.logits) + at * L::kBytes;
  const int lead = static_cast<int>((reinterpret_cast<uintptr_t>(first) & 15) / L::kBytes);
  const char* base = first - lead * L::kBytes;
  const int vecs = static_cast<int>((static_cast<long long>(lead) + p.vocab + L::kPer - 1) / L::kPer);
  const int v0 = split * p.split_vecs;
  const int vend = min(vecs, v0 + p.split_vecs);
  const int n = p.num_out;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int out = row * p.splits + split;

  if (tid == 0) sh.limit = 0;
  for (int i = tid; i < n; i += kRowThreads) sh.top[i] = 0;
  float m = -INFINITY, s = 0.f;  // this thread's maximum and sum of exp(x - m)
  __syncthreads();

  for (int t0 = v0; t0 < vend; t0 += kRowThreads * kVec) {
    float x[L::kMine];
    uint4 raw[kVec];
    bool edge[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) load_vec<DT>(base, t0 + j * kRowThreads + tid, vend, lead, p.vocab, raw[j], edge[j]);
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      if (!edge[j]) {
        unpack<DT>(raw[j], x + j * L::kPer);
      } else {
        const int vec = t0 + j * kRowThreads + tid;
#pragma unroll
        for (int e = 0; e < L::kPer; ++e) {
          const int i = vec * L::kPer - lead + e;
          x[j * L::kPer + e] = (vec < vend && i >= 0 && i < p.vocab) ? load_one<DT>(first, i) : -INFINITY;
        }
      }
    }
    // ---- sum of exponentials -------------------------------------------------
    float tmax = x[0];
#pragma unroll
    for (int e = 1; e < L::kMine; ++e) tmax = fmaxf(tmax, x[e]);  // fmaxf drops NaN
    tmax = fminf(fmaxf(tmax, -INFINITY), FLT_MAX);
    if (tmax > m) {
      s *= ex2((m - tmax) * kLog2e);  // m = -inf gives 0
      m = tmax;
    }
    const float ref = fmaxf(m, -FLT_MAX);
    float part[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int e = 0; e < L::kMine; ++e) part[e & 3] += ex2((x[e] - ref) * kLog2e);
    float sum = (part[0] + part[1]) + (part[2] + part[3]);
    if (!(sum <= FLT_MAX)) {  // a NaN or +inf among them
      sum = 0.f;
#pragma unroll
      for (int e = 0; e < L::kMine; ++e) sum += ex2((clean(x[e]) - ref) * kLog2e);
    }
    s += sum;
    // ---- the best n logits so far ----------------------------------------------
    const unsigned long long limit = sh.limit;
    const int token0 = (t0 + tid) * L::kPer - lead;
    auto token_of = [&](int j, int e) { return token0 + j * kRowThreads * L::kPer + e; };
    auto valid = [&](int j, int tok) { return t0 + j * kRowThreads + tid < vend && tok >= 0 && tok < p.vocab; };
    unsigned long long best = 0;  // this thread's largest key, where it may pass the limit
    if (limit == 0 || tmax >= key_logit(limit)) {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
#pragma unroll
        for (int e = 0; e < L::kPer; ++e) {
          const int tok = token_of(j, e);
          const float v = x[j * L::kPer + e];
          if ((v >= tmax || tmax == -INFINITY) && valid(j, tok)) {  // a NaN counts as -inf
            const unsigned long long k = make_key(v, tok);
            best = k > best ? k : best;
          }
        }
    }
    if (!__syncthreads_or(best > limit)) continue;
    // The n-th largest of the threads' best keys bounds the candidates from
    // below, and only the n threads at or above it can hold any.
    {
      unsigned long long k = best;
#pragma unroll
      for (int size = 2; size <= 32; size <<= 1) {
#pragma unroll
        for (int step = size >> 1; step > 0; step >>= 1) {
          const unsigned long long o = __shfl_xor_sync(0xffffffffu, k, step);
          const bool larger = ((lane & size) == 0) == ((lane & step) == 0);
          k = (larger == (o > k)) ? o : k;
        }
      }
      sh.sorted[warp][lane] = k;
      if (tid == 0) sh.count = 0;
      __syncthreads();
      int rank = lane;
#pragma unroll
      for (int w = 0; w < kRowWarps; ++w)
        if (w != warp) {
          int a = count_above(sh.sorted[w], 32, k);
          if (k == 0 && w < warp) a = 32;  // zeros stand for absent keys: any order among them
          rank += a;
        }
      if (rank == n - 1) sh.limit = k > limit ? k : limit;
      for (int i = tid; i < n; i += kRowThreads) {
        const unsigned long long k0 = sh.top[i];
        if (k0) sh.buf[atomicAdd(&sh.count, 1)] = k0;
      }
      __syncthreads();
    }
    const unsigned long long low = sh.limit;
    if (best && best >= low) {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
#pragma unroll
        for (int e = 0; e < L::kPer; ++e) {
          const int tok = token_of(j, e);
          if (valid(j, tok)) {
            const unsigned long long k = make_key(x[j * L::kPer + e], tok);
            if (k >= low && k > limit) sh.buf[atomicAdd(&sh.count, 1)] = k;
          }
        }
    }
    __syncthreads();
    const int have = sh.count;
    for (int i = tid; i < have; i += kRowThreads) {
      const unsigned long long k = sh.buf[i];
      int r = 0;
      for (int q = 0; q < have; ++q) r += sh.buf[q] > k;
      if (r < n) sh.top[r] = k;
    }
    __syncthreads();
    if (tid == 0) sh.limit = sh.top[n - 1];
    __syncthreads();
  }

  // ---- join the threads' sums ---------------------------------------------------
  float mm = m;
#pragma unroll
  for (int o = 16; o; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(0xffffffffu, mm, o));
  s *= ex2((m - fmaxf(mm, -FLT_MAX)) * kLog2e);
#pragma unroll
  for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
  if (lane == 0) {
    sh.m[warp] = mm;
    sh.s[warp] = s;
  }
  __syncthreads();
  if (tid == 0) {
    float M = sh.m[0], S = 0.f;
    for (int w = 1; w < kRowWarps; ++w) M = fmaxf(M, sh.m[w]);
    for (int w = 0; w < kRowWarps; ++w) S += sh.s[w] * ex2((sh.m[w] - fmaxf(M, -FLT_MAX)) * kLog2e);
    p.part_max[out] = M;
    p.part_sum[out] = S;
  }
  for (int i = tid; i < n; i += kRowThreads) p.part_key[static_cast<long long>(out) * n + i] = sh.top[i];
}

// One CTA per sequence: the splits' lists of each beam, then the beams.  An
// entry's place is the number of entries above it, found by binary search in
// the other sorted lists.  Scores are formed in 64 bits: candidates of
// different beams lie as near as their logits' rounding, and -50 + x - lse in
// 32 bits would swap them.
__global__ void __launch_bounds__(kMergeThreads) beam_merge_kernel(const BeamParams p) {
  pdl_enter();
  extern __shared__ unsigned long long dyn[];
  const int b = blockIdx.x, K = p.beams, S = p.splits, n = p.num_out;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  unsigned long long* keys = dyn;                                // [K][S][n]
  unsigned long long* rows = keys + K * S * n;                   // [K][n]
  double* score = reinterpret_cast<double*>(rows + K * n);       // [K][n]
  __shared__ double lse[kMaxBeams];
  __shared__ unsigned char done[kMaxBeams];
  const int row0 = b * K;
  for (int i = tid; i < K * S * n; i += kMergeThreads) {
    const int k = i / (S * n);
    const bool fin = p.finished && p.finished[row0 + k];
    keys[i] = fin ? 0 : p.part_key[static_cast<long long>(row0) * S * n + i];
  }
  for (int i = tid; i < K * n; i += kMergeThreads) rows[i] = 0;
  for (int k = warp; k < K; k += kMergeThreads / 32) {
    const bool fin = p.finished && p.finished[row0 + k];
    float m = -INFINITY, s = 0.f;
    if (!fin && lane < S) {
      m = p.part_max[(row0 + k) * S + lane];
      s = p.part_sum[(row0 + k) * S + lane];
    }
    float M = m;
#pragma unroll
    for (int o = 16; o; o >>= 1) M = fmaxf(M, __shfl_xor_sync(0xffffffffu, M, o));
    double sum = s > 0.f ? static_cast<double>(s) * exp(static_cast<double>(m) - static_cast<double>(M)) : 0.0;
#pragma unroll
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) {
      lse[k] = sum > 0.0 ? static_cast<double>(M) + log(sum) : 0.0;  // a row of -inf: every score is -inf
      done[k] = fin;
    }
  }
  __syncthreads();
  for (int i = tid; i < K * S * n; i += kMergeThreads) {
    const unsigned long long key = keys[i];
    if (!key) continue;
    const int list = i / n, k = list / S;
    int rank = i - list * n;
    for (int q = k * S; q < (k + 1) * S && rank < n; ++q)
      if (q != list) rank += count_above(keys + q * n, n, key);
    if (rank < n) rows[k * n + rank] = key;
  }
  __syncthreads();
  for (int i = tid; i < K * n; i += kMergeThreads) {
    const int k = i / n, r = i - k * n;
    const float base = p.scores[row0 + k];
    double v = -INFINITY;
    if (done[k]) {
      const int tok = r == 0 ? p.eos : r - 1 + (r - 1 >= p.eos);
      if (r < p.vocab) {
        rows[i] = make_key(r == 0 ? 0.f : -INFINITY, tok);
        if (r == 0) v = base;
      }
    } else if (rows[i]) {
      v = static_cast<double>(base) + (static_cast<double>(key_logit(rows[i])) - lse[k]);
    }
    score[i] = v == v ? v : -INFINITY;  // NaN counts as -inf
  }
  __syncthreads();
  const int width = min(n, p.vocab);  // entries of a beam's list
  for (int i = tid; i < K * n; i += kMergeThreads) {
    const int k = i / n, r = i - k * n;
    if (r >= width) continue;
    const double v = score[i];
    int rank = r;
    for (int q = 0; q < K && rank < n; ++q) {
      if (q == k) continue;
      int lo = 0, hi = width;
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        const double o = score[q * n + mid];
        if (o > v || (o == v && q < k)) lo = mid + 1;
        else hi = mid;
      }
      rank += lo;
    }
    if (rank < n) {
      const long long o = static_cast<long long>(b) * n + rank;
      p.out_scores[o] = static_cast<float>(v);
      p.out_tokens[o] = key_token(rows[i]);
      p.out_parents[o] = k;
    }
  }
}

}  // namespace

// Splits of a row: enough CTAs for two rounds of the four that fit an SM, at
// least one tile each, no more than the merge joins with a lane each and its
// shared memory (64 KB of keys) holds.
int beam_splits(int rows, int beams, int num_out, int vocab, int dtype, int aligned, int* split_vecs) {
  const int per = dtype == PA_DTYPE_F32 ? 4 : 8;
  const long long vecs = (static_cast<long long>(vocab) + per - 1) / per + (aligned ? 0 : 1);  // a row may start inside its first vector
  const long long tile = kRowThreads * kVec;
  long long s = (2LL * 4 * device_sm_count() + rows - 1) / rows;
  const long long most[3] = {(vecs + tile - 1) / tile, kMaxSplits, 8192 / (static_cast<long long>(beams) * num_out)};
  for (long long m : most) s = s < m ? s : m;
  if (s < 1) s = 1;
  *split_vecs = static_cast<int>((vecs + s - 1) / s);
  return static_cast<int>((vecs + *split_vecs - 1) / *split_vecs);
}

cudaError_t launch_beam_select(const BeamParams& p, int dtype, cudaStream_t stream) {
  const dim3 grid(p.seqs * p.beams, p.splits);
  cudaError_t e;
  if (dtype == PA_DTYPE_F32) e = launch_pdl(beam_rows_kernel<PA_DTYPE_F32>, grid, dim3(kRowThreads), 0, stream, p);
  else if (dtype == PA_DTYPE_BF16) e = launch_pdl(beam_rows_kernel<PA_DTYPE_BF16>, grid, dim3(kRowThreads), 0, stream, p);
  else e = launch_pdl(beam_rows_kernel<PA_DTYPE_F16>, grid, dim3(kRowThreads), 0, stream, p);
  if (e != cudaSuccess) return e;
  const size_t smem = (static_cast<size_t>(p.beams) * p.splits + 2 * p.beams) * p.num_out * 8;
  if (smem > 48 * 1024) {
    e = cudaFuncSetAttribute(beam_merge_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  e = launch_pdl(beam_merge_kernel, dim3(p.seqs), dim3(kMergeThreads), smem, stream, p);
  return e != cudaSuccess ? e : cudaGetLastError();
}

}  // namespace pa
