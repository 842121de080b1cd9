// Penalties for repeated tokens, biases and grammar masks on logits, in one pass.
//
// For logit x of token v in row r, with n the times v was generated in the row
//   x' = v seen (prompt or generated) ? (x > 0 ? x / rep : x * rep) : x
//   x' = (x' - freq * n) - pres * [n > 0]
//   x' = x' + bias[bias_row[r]][v]
//   x' = -inf where mask[mask_row[r]] has v's bit clear
// in fp32, each operation rounded by itself, and once to the output's type.  The
// reference samples from plain logits (core/model_runner.py:28-159).
//
// A logit is read and written once; HBM is at 38 % in the largest case below, the first stall is a load: a CTA goes through its
// row's tokens before its first piece.  A CTA asks for its span of a row to be brought into
// L2 whole, then applies biases and masks to every column, chunk by chunk.  The few seen columns are done behind that
// stream: while the span is on its way the CTA sets a bit for each, counts how often it was generated (whole numbers: the
// order of the atomics does not show) and lists the bits; a stream that works in place leaves those logits as they are;
// then every listed column's logit is read again, from L2, and its result written.
// 512 rows of 131072 bf16 logits, 750-1500 tokens each, a bias and a mask: 70-79 us (42 without any
// of them, as a plain copy).  The stream with the penalties inside took 137 (nearly every warp went through eight divisions for one
// column), results worked out before the stream 117, a register double buffer at a third of the occupancy 97.
#include <atomic>

#include "pa_common.cuh"

namespace pa {
namespace {

template <int T>
struct Elem;
template <>
struct Elem<PA_DTYPE_F32> {
  using type = float;
  static __device__ __forceinline__ float get(float v) { return v; }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <>
struct Elem<PA_DTYPE_F16> {
  using type = __half;
  static __device__ __forceinline__ float get(__half v) { return __half2float(v); }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <>
struct Elem<PA_DTYPE_BF16> {
  using type = __nv_bfloat16;
  static __device__ __forceinline__ float get(__nv_bfloat16 v) { return __bfloat162float(v); }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

// Asks for [a, b) to be brought into L2, in whole units of 16 bytes.
__device__ __forceinline__ void prefetch_l2(const void* a, const void* b) {
  const uintptr_t lo = (reinterpret_cast<uintptr_t>(a) + 15) & ~uintptr_t(15), hi = reinterpret_cast<uintptr_t>(b) & ~uintptr_t(15);
  if (lo < hi) asm volatile("cp.async.bulk.prefetch.L2.global [%0], %1;" ::"l"(lo), "r"(static_cast<uint32_t>(hi - lo)));
}

// Elements of type T in 16 bytes, and the values of one such piece.
template <int T>
__device__ __forceinline__ void load16(const uint4& w, float* f) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (T == PA_DTYPE_F32) {
      f[i] = __uint_as_float(x[i]);
    } else {
      float2 v;
      if constexpr (T == PA_DTYPE_BF16) v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[i]));
      else v = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

constexpr int LA_THREADS = 512;
constexpr int LA_EARLY = 4;  // tokens of a thread that are asked for before the row's length is known

// NV: 16-byte pieces a thread takes of a chunk.  Piece j of a row starts at column j * EPL - off, with off the elements
// between the last 16-byte boundary and the row's start: every inner piece is one aligned load.  splits: spans of a row;
// per_span: chunks of a span; pair: two counts a word (no row has 65536 tokens).
template <int IN, int OUT, int NV>
__global__ void __launch_bounds__(LA_THREADS, 3) logits_adjust_kernel(const LogitsParams p, int splits, int per_span, int pair) {
  pdl_enter();
  using EI = Elem<IN>;
  using EO = Elem<OUT>;
  using TI = typename EI::type;
  using TO = typename EO::type;
  constexpr int EPL = 16 / static_cast<int>(sizeof(TI));
  constexpr int COLS = LA_THREADS * NV * EPL;
  static_assert(COLS % 32 == 0, "whole words of bits");
  const int words = per_span * (COLS / 32);
  extern __shared__ __align__(16) uint32_t la_smem[];
  uint32_t* bits = la_smem;           // [words] seen columns
  uint32_t* times = la_smem + words;  // [columns, or half as many] times generated; set for seen columns alone
  uint16_t* list = reinterpret_cast<uint16_t*>(times + (per_span * COLS >> pair));  // the seen columns
  __shared__ uint32_t listed;
  const int r = static_cast<int>(blockIdx.x / splits);
  const int tid = threadIdx.x;
  const TI* x = static_cast<const TI*>(p.x) + r * p.x_stride;
  TO* out = static_cast<TO*>(p.out) + r * p.out_stride;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(TI));
  const int s0 = static_cast<int>(blockIdx.x % splits) * per_span * COLS - off;  // first column, maybe before the row
  if (s0 >= p.vocab) return;
  const int s1 = min(s0 + per_span * COLS, p.vocab);

  auto whole = [&](int c) { return c >= 0 && c + EPL <= p.vocab; };
  if (tid == 0) prefetch_l2(x + max(s0, 0), x + s1);
  // what the row's penalties, bias and mask are, and its first tokens, all asked for at once
  const bool history = p.max_tokens > 0;
  const int* tok = p.tokens + r * p.tokens_stride;
  int early[LA_EARLY];
#pragma unroll
  for (int k = 0; k < LA_EARLY; ++k) early[k] = k * LA_THREADS + tid < p.max_tokens ? tok[k * LA_THREADS + tid] : -1;
  const int b = p.bias ? (p.bias_row ? p.bias_row[r] : p.bias_rows == 1 ? 0 : r) : -1;
  const int m = p.mask ? (p.mask_row ? p.mask_row[r] : p.mask_rows == 1 ? 0 : r) : -1;
  float rep = p.rep_v, pres = p.pres_v, freq = p.freq_v;
  int n = p.max_tokens, prompt = 0;
  if (history) {
    if (p.rep) rep = p.rep[r];
    if (p.pres) pres = p.pres[r];
    if (p.freq) freq = p.freq[r];
    if (p.num_tokens) n = min(p.num_tokens[r], p.max_tokens);
    if (p.prompt_len) prompt = p.prompt_len[r];
  }
  if ((b < -1 || b >= p.bias_rows || m < -1 || m >= p.mask_rows) && tid == 0) set_status(p.status, ST_BAD_SEQ_INDEX);
  const float* bias = b >= 0 && b < p.bias_rows ? p.bias + b * p.bias_stride : nullptr;
  const uint32_t* mask = m >= 0 && m < p.mask_rows ? reinterpret_cast<const uint32_t*>(p.mask) + m * p.mask_stride : nullptr;
  if (tid == 32 && mask) prefetch_l2(mask + (max(s0, 0) >> 5), mask + (s1 >> 5));
  if (tid == 64 && bias) prefetch_l2(bias + max(s0, 0), bias + s1);
  // every token of the span, with its place in the row
  auto tokens = [&](auto&& f) {
    const int lo = max(s0, 0);
#pragma unroll
    for (int k = 0; k < LA_EARLY; ++k)
      if (k * LA_THREADS + tid < n && early[k] >= lo && early[k] < s1) f(early[k] - s0, k * LA_THREADS + tid);
    for (int i = LA_EARLY * LA_THREADS + tid; i < n; i += LA_THREADS) {
      const int v = tok[i];
      if (v >= lo && v < s1) f(v - s0, i);
    }
  };
  if (history) {
    for (int i = tid; i < words; i += LA_THREADS) bits[i] = 0;
    if (tid == 0) listed = 0;
    __syncthreads();
    tokens([&](int at, int) {
      atomicOr(&bits[at >> 5], 1u << (at & 31));
      times[at >> pair] = 0;
    });
    __syncthreads();
    tokens([&](int at, int i) {
      if (i >= prompt) atomicAdd(&times[at >> pair], pair && (at & 1) ? 0x10000u : 1u);
    });
    for (int w = tid; w < words; w += LA_THREADS) {
      uint32_t left = bits[w];
      uint32_t k = left ? atomicAdd(&listed, __popc(left)) : 0u;
      for (; left; left &= left - 1) list[k++] = static_cast<uint16_t>(32 * w + __ffs(left) - 1);
    }
  }
  const bool in_place = history && static_cast<const void*>(p.x) == static_cast<const void*>(p.out);

  // Biases are read around a piece by aligned loads, `sh` columns too early (alike in every lane and chunk: pieces start on a
  // 16-byte boundary of the logits, not of the biases).
  const int sh = bias ? static_cast<int>((reinterpret_cast<uintptr_t>(bias + (s0 + COLS)) >> 2) & 3) : 0;
  const bool out_vec = ((reinterpret_cast<uintptr_t>(out) - off * sizeof(TO)) & 15) == 0;
  for (int c0 = s0; c0 < s1; c0 += COLS) {
    uint4 raw[NV];
    uint32_t allowed[NV];  // a piece's mask bits
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = c0 + (i * LA_THREADS + tid) * EPL;
      raw[i] = whole(c) ? *reinterpret_cast<const uint4*>(x + c) : make_uint4(0, 0, 0, 0);
    }
    if (mask) {
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        const int c = c0 + (i * LA_THREADS + tid) * EPL;
        allowed[i] = 0;
        if (whole(c)) {
          allowed[i] = mask[c >> 5] >> (c & 31);
          if ((c & 31) > 32 - EPL) allowed[i] |= mask[(c >> 5) + 1] << (32 - (c & 31));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const int c = c0 + (i * LA_THREADS + tid) * EPL;
      if (c + EPL <= 0 || c >= p.vocab) continue;
      const int at = c - s0;
      const uint32_t seen = in_place ? (bits[at >> 5] >> (at & 31)) & ((1u << EPL) - 1u) : 0u;
      if (!whole(c)) {
        for (int e = 0; e < EPL; ++e) {
          const int col = c + e;
          if (col < 0 || col >= p.vocab) continue;
          float v = EI::get(x[col]);
          if (bias) v = __fadd_rn(v, bias[col]);
          if (mask && !((mask[col >> 5] >> (col & 31)) & 1u)) v = -INFINITY;
          if (!((seen >> e) & 1u)) out[col] = EO::put(v);
        }
        continue;
      }
      float f[EPL];
      load16<IN>(raw[i], f);
      if (bias) {
        if (sh == 0) {
#pragma unroll
          for (int q = 0; q < EPL / 4; ++q) {
            const float4 w = __ldg(reinterpret_cast<const float4*>(bias + c) + q);
            f[4 * q] = __fadd_rn(f[4 * q], w.x);
            f[4 * q + 1] = __fadd_rn(f[4 * q + 1], w.y);
            f[4 * q + 2] = __fadd_rn(f[4 * q + 2], w.z);
            f[4 * q + 3] = __fadd_rn(f[4 * q + 3], w.w);
          }
        } else if (c >= sh && c - sh + EPL + 4 <= p.vocab) {
          float g[EPL + 4];
#pragma unroll
          for (int q = 0; q < EPL / 4 + 1; ++q) {
            const float4 w = __ldg(reinterpret_cast<const float4*>(bias + c - sh) + q);
            g[4 * q] = w.x, g[4 * q + 1] = w.y, g[4 * q + 2] = w.z, g[4 * q + 3] = w.w;
          }
#pragma unroll
          for (int e = 0; e < EPL; ++e) f[e] = __fadd_rn(f[e], sh == 1 ? g[e + 1] : sh == 2 ? g[e + 2] : g[e + 3]);
        } else {  // that would leave the row
#pragma unroll
          for (int e = 0; e < EPL; ++e) f[e] = __fadd_rn(f[e], __ldg(bias + c + e));
        }
      }
      if (mask) {
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          if (!((allowed[i] >> e) & 1u)) f[e] = -INFINITY;
      }
      if (seen) {
        float g[EPL];
        load16<IN>(raw[i], g);
#pragma unroll
        for (int e = 0; e < EPL; ++e)
          if ((seen >> e) & 1u) f[e] = g[e];
      }
      TO o[EPL];
#pragma unroll
      for (int e = 0; e < EPL; ++e) o[e] = EO::put(f[e]);
      if (out_vec) {
#pragma unroll
        for (int q = 0; q < static_cast<int>(EPL * sizeof(TO) / 16); ++q)
          reinterpret_cast<uint4*>(out + c)[q] = reinterpret_cast<const uint4*>(o)[q];
      } else {
#pragma unroll
        for (int e = 0; e < EPL; ++e) out[c + e] = o[e];
      }
    }
  }

  if (!history) return;
  __syncthreads();  // the span is written, the counts and the list are complete
  for (uint32_t i = tid; i < listed; i += LA_THREADS) {
    const int at = list[i], col = s0 + at;
    uint32_t c = times[at >> pair];
    if (pair) c = at & 1 ? c >> 16 : c & 0xffffu;
    const float add = bias ? bias[col] : 0.f;
    const bool ok = !mask || ((mask[col >> 5] >> (col & 31)) & 1u);
    float v = EI::get(x[col]);
    v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
    v = __fsub_rn(v, __fmul_rn(freq, static_cast<float>(c)));
    if (c) v = __fsub_rn(v, pres);
    if (bias) v = __fadd_rn(v, add);
    out[col] = EO::put(ok ? v : -INFINITY);
  }
}

template <int IN, int OUT, int NV>
cudaError_t launch_nv(const LogitsParams& p, cudaStream_t stream) {
  constexpr int EPL = IN == PA_DTYPE_F32 ? 4 : 8;
  constexpr int COLS = LA_THREADS * NV * EPL;
  // a row may start up to EPL - 1 elements behind a 16-byte boundary
  const long long chunks = (p.vocab + EPL - 1LL + COLS - 1) / COLS;
  // Every span goes through its row's tokens, so spans are as long as a wave of three CTAs an SM allows, and as their
  // counts leave room for three (512 rows of 131072: 79 us with spans of 16384 columns, 74 with 32768).
  const int pair = p.max_tokens < 65536;
  constexpr long long most = 32768 / COLS;
  const long long wave = 3LL * device_sm_count();
  long long per_span = (chunks * p.rows + wave - 1) / wave;
  per_span = per_span < 1 ? 1 : per_span > (pair ? most : most / 2) ? (pair ? most : most / 2) : per_span;
  const long long splits = (chunks + per_span - 1) / per_span;
  per_span = (chunks + splits - 1) / splits;
  if (splits * p.rows > 0x7fffffffLL) return cudaErrorInvalidValue;
  const size_t columns = static_cast<size_t>(per_span * COLS);
  const size_t room = ((static_cast<size_t>(p.max_tokens) < columns ? p.max_tokens : columns) + 1) & ~size_t{1};
  const size_t smem = p.max_tokens > 0 ? columns / 8 + (columns * 4 >> pair) + 2 * room : 0;
  auto kern = logits_adjust_kernel<IN, OUT, NV>;
  if (smem > 48 * 1024) {  // at most 4 + 64 + 64 KB; allowed once per device
    static std::atomic<unsigned long long> done{0};
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess && !(dev < 64 && (done.load(std::memory_order_acquire) >> dev & 1))) {
      e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 132 * 1024);
      if (e == cudaSuccess && dev < 64) done.fetch_or(1ull << dev, std::memory_order_release);
    }
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(kern, dim3(static_cast<unsigned>(splits * p.rows)), dim3(LA_THREADS), smem, stream, p,
                    static_cast<int>(splits), static_cast<int>(per_span), pair);
}

template <int IN, int OUT>
cudaError_t launch_la(const LogitsParams& p, cudaStream_t stream) {
  // few columns in all: a piece a thread, so that more SMs take part (16 rows of 32000 bf16 logits: 4.1 against 4.6 us,
  // 64 rows of 32000 alike, 16 of 128256 7.2 both ways)
  if (static_cast<long long>(p.rows) * p.vocab < device_sm_count() * 16384LL) return launch_nv<IN, OUT, 1>(p, stream);
  return launch_nv<IN, OUT, 2>(p, stream);
}

}  // namespace

cudaError_t launch_logits_adjust(const LogitsParams& p, int dtype, int out_dtype, cudaStream_t stream) {
  if (p.rows == 0) return cudaSuccess;
  const bool wide = out_dtype == PA_DTYPE_F32;
  switch (dtype) {
    case PA_DTYPE_F32:
      return launch_la<PA_DTYPE_F32, PA_DTYPE_F32>(p, stream);
    case PA_DTYPE_BF16:
      return wide ? launch_la<PA_DTYPE_BF16, PA_DTYPE_F32>(p, stream) : launch_la<PA_DTYPE_BF16, PA_DTYPE_BF16>(p, stream);
    default:
      return wide ? launch_la<PA_DTYPE_F16, PA_DTYPE_F32>(p, stream) : launch_la<PA_DTYPE_F16, PA_DTYPE_F16>(p, stream);
  }
}

}  // namespace pa
