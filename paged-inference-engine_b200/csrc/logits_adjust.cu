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
// Bound by HBM: a logit is read and written once.  A CTA takes CTA_COLS columns of a
// row: it loads them into registers, and while those loads are in flight goes
// over the row's tokens for the ones in its columns.  A bit per column says which were
// seen, a word per column counts the generated ones; the words are cleared only where a
// bit is set, so nothing is spent on the columns that no token names, and a lane looks at
// the words only if one of its columns' bits is set.  Counts are whole numbers: the order
// of the atomics does not show.
#include "pa_common.cuh"

namespace pa {
namespace {

constexpr int LA_THREADS = 256;

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

// NV: 16-byte pieces a thread takes.  Piece j of a row starts at column j * EPL - off, with off the elements
// between the last 16-byte boundary and the row's start: every inner piece is one aligned load.
template <int IN, int OUT, int NV>
__global__ void __launch_bounds__(LA_THREADS) logits_adjust_kernel(const LogitsParams p, int chunks) {
  pdl_enter();
  using EI = Elem<IN>;
  using EO = Elem<OUT>;
  using TI = typename EI::type;
  using TO = typename EO::type;
  constexpr int EPL = 16 / static_cast<int>(sizeof(TI));
  constexpr int CTA_COLS = LA_THREADS * NV * EPL;
  extern __shared__ uint32_t la_smem[];
  uint32_t* bits = la_smem;                    // [CTA_COLS / 32]
  uint32_t* times = la_smem + CTA_COLS / 32;   // [CTA_COLS]
  const int r = static_cast<int>(blockIdx.x / chunks);
  const int tid = threadIdx.x;
  const TI* x = static_cast<const TI*>(p.x) + r * p.x_stride;
  TO* out = static_cast<TO*>(p.out) + r * p.out_stride;
  const int off = static_cast<int>((reinterpret_cast<uintptr_t>(x) & 15) / sizeof(TI));
  const int c0 = static_cast<int>(blockIdx.x % chunks) * CTA_COLS - off;  // first column, maybe before the row
  if (c0 >= p.vocab) return;

  // ---- this thread's logits --------------------------------------------------
  uint4 raw[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int c = c0 + (i * LA_THREADS + tid) * EPL;
    raw[i] = make_uint4(0, 0, 0, 0);
    if (c >= 0 && c + EPL <= p.vocab) raw[i] = *reinterpret_cast<const uint4*>(x + c);
  }

  // ---- the row's tokens in these columns --------------------------------------
  const bool history = p.max_tokens > 0;
  float rep = p.rep_v, pres = p.pres_v, freq = p.freq_v;
  if (history) {
    if (p.rep) rep = p.rep[r];
    if (p.pres) pres = p.pres[r];
    if (p.freq) freq = p.freq[r];
    const int* tok = p.tokens + r * p.tokens_stride;
    const int n = p.num_tokens ? min(p.num_tokens[r], p.max_tokens) : p.max_tokens;
    const int prompt = p.prompt_len ? p.prompt_len[r] : 0;
    for (int i = tid; i < CTA_COLS / 32; i += LA_THREADS) bits[i] = 0;
    __syncthreads();
    const int hi = min(c0 + CTA_COLS, p.vocab), lo = max(c0, 0);
    for (int i = tid; i < n; i += LA_THREADS) {
      const int v = tok[i];
      if (v < lo || v >= hi) continue;
      const int k = v - c0;
      times[k] = 0;
      atomicOr(&bits[k >> 5], 1u << (k & 31));
    }
    __syncthreads();
    for (int i = max(prompt, 0) + tid; i < n; i += LA_THREADS) {
      const int v = tok[i];
      if (v >= lo && v < hi) atomicAdd(&times[v - c0], 1u);
    }
    __syncthreads();
  }
  const float* bias = nullptr;
  if (p.bias) {
    const int b = p.bias_row ? p.bias_row[r] : p.bias_rows == 1 ? 0 : r;
    if (b >= 0 && b < p.bias_rows) bias = p.bias + b * p.bias_stride;
    else if (b != -1 && tid == 0) set_status(p.status, ST_BAD_SEQ_INDEX);
  }
  const uint32_t* mask = nullptr;
  if (p.mask) {
    const int m = p.mask_row ? p.mask_row[r] : p.mask_rows == 1 ? 0 : r;
    if (m >= 0 && m < p.mask_rows) mask = reinterpret_cast<const uint32_t*>(p.mask) + m * p.mask_stride;
    else if (m != -1 && tid == 0) set_status(p.status, ST_BAD_SEQ_INDEX);
  }

  auto rule = [&](float v, int k, bool seen) {  // history, for the column at place k of the CTA's
    if (seen) {
      v = v > 0.f ? __fdiv_rn(v, rep) : __fmul_rn(v, rep);
      const uint32_t n = times[k];
      v = __fsub_rn(v, __fmul_rn(freq, static_cast<float>(n)));
      if (n) v = __fsub_rn(v, pres);
    }
    return v;
  };

  const bool out_vec = ((reinterpret_cast<uintptr_t>(out) - off * sizeof(TO)) & 15) == 0;

#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int k0 = (i * LA_THREADS + tid) * EPL;
    const int c = c0 + k0;
    if (c + EPL <= 0 || c >= p.vocab) continue;
    const uint32_t seen = history ? (bits[k0 >> 5] >> (k0 & 31)) & ((1u << EPL) - 1u) : 0u;
    if (c < 0 || c + EPL > p.vocab) {
      for (int e = 0; e < EPL; ++e) {
        const int col = c + e;
        if (col < 0 || col >= p.vocab) continue;
        float v = rule(EI::get(x[col]), k0 + e, (seen >> e) & 1u);
        if (bias) v = __fadd_rn(v, bias[col]);
        if (mask && !((mask[col >> 5] >> (col & 31)) & 1u)) v = -INFINITY;
        out[col] = EO::put(v);
      }
      continue;
    }
    float f[EPL];
    load16<IN>(raw[i], f);
    if (seen) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) f[e] = rule(f[e], k0 + e, (seen >> e) & 1u);
    }
    if (bias) {
#pragma unroll
      for (int e = 0; e < EPL; ++e) f[e] = __fadd_rn(f[e], __ldg(bias + c + e));
    }
    if (mask) {
      const uint32_t m = __funnelshift_r(mask[c >> 5], mask[(c + EPL - 1) >> 5], c & 31);
#pragma unroll
      for (int e = 0; e < EPL; ++e)
        if (!((m >> e) & 1u)) f[e] = -INFINITY;
    }
    TO o[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) o[e] = EO::put(f[e]);
    if (out_vec) {
#pragma unroll
      for (int b = 0; b < static_cast<int>(EPL * sizeof(TO) / 16); ++b)
        reinterpret_cast<uint4*>(out + c)[b] = reinterpret_cast<const uint4*>(o)[b];
    } else {
#pragma unroll
      for (int e = 0; e < EPL; ++e) out[c + e] = o[e];
    }
  }
}

template <int IN, int OUT, int NV>
cudaError_t launch_nv(const LogitsParams& p, cudaStream_t stream) {
  constexpr int EPL = IN == PA_DTYPE_F32 ? 4 : 8;
  constexpr int COLS = LA_THREADS * NV * EPL;
  // a row may start up to EPL - 1 elements behind a 16-byte boundary
  const long long chunks = (p.vocab + EPL - 1LL + COLS - 1) / COLS;
  if (chunks * p.rows > 0x7fffffffLL) return cudaErrorInvalidValue;
  const size_t smem = p.max_tokens > 0 ? COLS / 8 + COLS * 4 : 0;
  auto kern = logits_adjust_kernel<IN, OUT, NV>;
  return launch_pdl(kern, dim3(static_cast<unsigned>(chunks * p.rows)), dim3(LA_THREADS), smem, stream, p,
                    static_cast<int>(chunks));
}

template <int IN, int OUT>
cudaError_t launch_la(const LogitsParams& p, cudaStream_t stream) {
  return launch_nv<IN, OUT, IN == PA_DTYPE_F32 ? 8 : 4>(p, stream);
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
