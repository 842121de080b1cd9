// Rotary position embedding with the write of new K/V rows into the paged pool.
//
// For a token at position p and a pair (a, b) of a query or key row's dims
//   a' = a cos - b sin,  b' = b cos + a sin   (cos, sin: row p of the table)
// with pairs (i, i + R/2) of the first R dims, or neighbours (2i, 2i + 1).  The
// rotated keys and the values then go where csrc/kv_write.cu puts rows, by the
// same rule (INT8: one absmax scale per (token, head); else rounded once).  The
// reference has no position embedding in its attention layer; its cache write
// is transformer/model.py:85-122.
//
// Every product and sum of the rotation is rounded to fp32 by itself (no fused
// multiply-add), so that the rows, and with them the INT8 codes, are those that
// the same four elementary fp32 operations give anywhere else.
//
// Bound by HBM for prompts (each row is read and written once), by latency for a
// decode step's few rows.  One warp per (token, unit): a unit is the K and V rows of HG
// kv heads, or NL * RPI query rows, all loaded before the first is used; the
// table row is loaded once a warp and serves all of the unit's rows, which is
// why a unit does not cross tokens.  The partner dims of the halves form lie
// R/2 dims away in the same row, that is in another lane of the same warp: they come by
// shuffles of packed words instead of a second load.
#include "pa_common.cuh"
#include "quant.cuh"

namespace pa {
namespace {

constexpr int ROT_THREADS = 256;

template <int IN, int D>
struct RCfg {
  static constexpr int ESZ = IN == PA_DTYPE_F32 ? 4 : 2;
  static constexpr int EPL = 16 / ESZ;  // elements per lane and load
  static constexpr int LPR = D / EPL;   // lanes per row
  static constexpr int RPI = 32 / LPR;  // rows per load instruction
  static constexpr int NL = 4;          // loads per lane in flight
  static constexpr int ROWS = NL * RPI;
  static constexpr int HG = ROWS / 2;   // kv heads of a unit (K and V rows)
  static_assert(LPR <= 32 && 32 % LPR == 0 && ROWS % 2 == 0, "a row maps onto whole lanes");
};

template <int IN, int EPL>
__device__ __forceinline__ void unpack_words(const uint4& w, float (&f)[EPL]) {
  const uint32_t x[4] = {w.x, w.y, w.z, w.w};
  if constexpr (IN == PA_DTYPE_F32) {
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(x[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float2 v;
      if constexpr (IN == PA_DTYPE_BF16) v = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&x[i]));
      else v = __half22float2(*reinterpret_cast<const __half2*>(&x[i]));
      f[2 * i] = v.x;
      f[2 * i + 1] = v.y;
    }
  }
}

template <int IN, int EPL>
__device__ __forceinline__ uint4 pack_words(const float (&f)[EPL]) {
  if constexpr (IN == PA_DTYPE_F32) {
    return make_uint4(__float_as_uint(f[0]), __float_as_uint(f[1]), __float_as_uint(f[2]), __float_as_uint(f[3]));
  } else {
    constexpr bool BF = IN == PA_DTYPE_BF16;
    return make_uint4(pack2<BF>(f[0], f[1]), pack2<BF>(f[2], f[3]), pack2<BF>(f[4], f[5]), pack2<BF>(f[6], f[7]));
  }
}

// This lane's part of a table row: its dims' cos and sin.  HALVES: one each per
// dim, the sin with the sign that the partner's product carries; pairs: one per pair.
template <bool PAIRS, int EPL>
struct Turn {
  static constexpr int N = PAIRS ? EPL / 2 : EPL;
  float c[N], s[N];
  int src;   // lane that holds the partner dims
  bool on;   // dims below rot_dim

  __device__ __forceinline__ void load(const float* row, int rot, int part, int lane) {
    const int d = part * EPL, half = rot >> 1;
    on = d < rot;
    src = lane;
    if (!on) return;
    float sign = 1.f;
    int at = d >> 1;
    if constexpr (!PAIRS) {
      const bool low = d < half;  // half is a multiple of EPL: a lane's dims lie on one side
      sign = low ? -1.f : 1.f;
      src = low ? lane + half / EPL : lane - half / EPL;
      at = low ? d : d - half;
    }
#pragma unroll
    for (int i = 0; i < N; i += N < 4 ? N : 4) {
      if constexpr (N >= 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(row + at + i));
        const float4 b = __ldg(reinterpret_cast<const float4*>(row + half + at + i));
        c[i] = a.x, c[i + 1] = a.y, c[i + 2] = a.z, c[i + 3] = a.w;
        s[i] = b.x * sign, s[i + 1] = b.y * sign, s[i + 2] = b.z * sign, s[i + 3] = b.w * sign;
      } else {
        const float2 a = __ldg(reinterpret_cast<const float2*>(row + at));
        const float2 b = __ldg(reinterpret_cast<const float2*>(row + half + at));
        c[0] = a.x, c[1] = a.y;
        s[0] = b.x, s[1] = b.y;
      }
    }
  }

  // f: this lane's dims of a row, raw: the same as loaded (for the partner).  Every lane of the warp calls it.
  template <int IN>
  __device__ __forceinline__ void apply(const uint4& raw, float (&f)[EPL]) const {
    unpack_words<IN, EPL>(raw, f);
    if constexpr (PAIRS) {
      if (on) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
          const float a = f[2 * i], b = f[2 * i + 1];
          f[2 * i] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
          f[2 * i + 1] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
        }
      }
    } else {
      uint4 o;
      o.x = __shfl_sync(0xffffffffu, raw.x, src);
      o.y = __shfl_sync(0xffffffffu, raw.y, src);
      o.z = __shfl_sync(0xffffffffu, raw.z, src);
      o.w = __shfl_sync(0xffffffffu, raw.w, src);
      float g[EPL];
      unpack_words<IN, EPL>(o, g);
      if (on) {
#pragma unroll
        for (int i = 0; i < EPL; ++i) f[i] = __fadd_rn(__fmul_rn(f[i], c[i]), __fmul_rn(g[i], s[i]));
      }
    }
  }
};

template <int IN, int D, bool PAIRS>
__global__ void __launch_bounds__(ROT_THREADS) kv_rotate_kernel(const WriteParams p, const RotateParams r) {
  pdl_enter();
  using C = RCfg<IN, D>;
  constexpr int EPL = C::EPL;
  const int lane = threadIdx.x & 31;
  const int kv_units = (p.Hkv + C::HG - 1) / C::HG;
  const int units = kv_units + (r.Hq + C::ROWS - 1) / C::ROWS;
  const long long wid = (static_cast<long long>(blockIdx.x) * ROT_THREADS + threadIdx.x) >> 5;
  if (wid >= static_cast<long long>(p.T) * units) return;
  const int t = static_cast<int>(wid / units);
  const int u = static_cast<int>(wid - static_cast<long long>(t) * units);
  const int part = lane % C::LPR;
  const int sub = lane / C::LPR;
  const bool isq = u >= kv_units;
  const int h0 = isq ? (u - kv_units) * C::ROWS : u * C::HG;

  // ---- source rows: row j of a kv unit is head h0 + j / 2, K for even j -------
  uint4 raw[C::NL];
#pragma unroll
  for (int it = 0; it < C::NL; ++it) {
    const int j = it * C::RPI + sub;
    raw[it] = make_uint4(0, 0, 0, 0);
    if (isq) {
      if (h0 + j < r.Hq)
        raw[it] = *(reinterpret_cast<const uint4*>(static_cast<const char*>(r.q) +
                                                   (t * r.q_st + (h0 + j) * r.q_sh) * C::ESZ) + part);
    } else if (h0 + (j >> 1) < p.Hkv) {
      const int h = h0 + (j >> 1);
      const char* src = (j & 1) ? static_cast<const char*>(p.v_new) + (t * p.vn_st + h * p.vn_sh) * C::ESZ
                                : static_cast<const char*>(p.k_new) + (t * p.kn_st + h * p.kn_sh) * C::ESZ;
      raw[it] = __ldg(reinterpret_cast<const uint4*>(src) + part);
    }
  }
  const int pos = p.pos[t];
  if (pos < 0 || pos >= r.num_pos) {
    if (lane == 0) set_status(p.status, ST_BAD_POSITION);
    return;
  }
  Turn<PAIRS, EPL> turn;
  turn.load(r.table + pos * r.table_stride, r.rot, part, lane);

  if (isq) {
#pragma unroll
    for (int it = 0; it < C::NL; ++it) {
      const int h = h0 + it * C::RPI + sub;
      float f[EPL];
      turn.template apply<IN>(raw[it], f);
      if (h < r.Hq)
        *(reinterpret_cast<uint4*>(static_cast<char*>(r.q_out) + (t * r.qo_st + h * r.qo_sh) * C::ESZ) + part) =
            pack_words<IN, EPL>(f);
    }
    return;
  }

  // ---- destination block / slot (as kv_write_kernel) --------------------------
  const int s = p.seq_idx[t];
  if (s < 0 || s >= p.num_seqs) {
    if (lane == 0) set_status(p.status, ST_BAD_SEQ_INDEX);
    return;
  }
  const int bi = pos >> p.log2BS;
  if (bi >= p.bt_cols) {
    if (lane == 0) set_status(p.status, ST_BAD_POSITION);
    return;
  }
  const int blk = p.bt[s * p.bt_ss + bi * p.bt_sc];
  if (blk < 0 || blk >= p.NB) {
    if (lane == 0) set_status(p.status, ST_BAD_BLOCK_ID);
    return;
  }
  const int slot = pos & (p.BS - 1);
  const long long kb = blk * p.k_sblk + slot * p.k_sslot, vb = blk * p.v_sblk + slot * p.v_sslot;
  const long long ksb = blk * p.ks_sblk + slot * p.ks_sslot, vsb = blk * p.vs_sblk + slot * p.vs_sslot;
  const bool i8 = p.cache_dtype == PA_DTYPE_I8;
  const bool f32 = p.cache_dtype == PA_DTYPE_F32;
  const bool bf = p.cache_dtype == PA_DTYPE_BF16;

  // rows stay in registers; the phases of an INT8 pool run over all of them, so that their shuffles overlap
  float f[C::NL][EPL], am[C::NL];
#pragma unroll
  for (int it = 0; it < C::NL; ++it) {
    const int j = it * C::RPI + sub;
    turn.template apply<IN>(raw[it], f[it]);
    if (j & 1) unpack_words<IN, EPL>(raw[it], f[it]);  // values are not rotated
  }
  if (i8) {
#pragma unroll
    for (int it = 0; it < C::NL; ++it) {
      am[it] = fabsf(f[it][0]);
#pragma unroll
      for (int i = 1; i < EPL; ++i) am[it] = fmaxf(am[it], fabsf(f[it][i]));
    }
#pragma unroll
    for (int o = C::LPR / 2; o >= 1; o >>= 1)
#pragma unroll
      for (int it = 0; it < C::NL; ++it) am[it] = fmaxf(am[it], __shfl_xor_sync(0xffffffffu, am[it], o));
  }
#pragma unroll
  for (int it = 0; it < C::NL; ++it) {
    const int j = it * C::RPI + sub;
    const int h = h0 + (j >> 1);
    const bool isv = j & 1;
    const long long at = (isv ? vb + h * p.v_shead : kb + h * p.k_shead) + part * EPL;
    void* base = isv ? p.v : p.k;
    if (i8) {
      const float sc = am[it] == 0.f ? 1.0f : div127_rn(am[it]);
      uint32_t w[EPL / 4];
      // the reciprocal of a scale below 2^-126 is not finite: such rows, too, take the division
      const bool near = quant_row_fast<EPL>(f[it], rcp_approx(sc), w) || sc < 1.2e-38f;
      if (__any_sync(0xffffffffu, near)) quant_row_exact<EPL>(f[it], sc, w);
      if (h >= p.Hkv) continue;
      int8_t* dst = static_cast<int8_t*>(base) + at;
      if constexpr (EPL == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
      else *reinterpret_cast<uint32_t*>(dst) = w[0];
      if (part == 0) {
        const long long so = isv ? vsb + h * p.vs_shead : ksb + h * p.ks_shead;
        void* sp = isv ? p.vs : p.ks;
        if (p.scale_f32) static_cast<float*>(sp)[so] = sc;
        else static_cast<__half*>(sp)[so] = __float2half_rn(sc);
      }
      continue;
    }
    if (h >= p.Hkv) continue;
    if (f32) {
      float4* dst = reinterpret_cast<float4*>(static_cast<float*>(base) + at);
#pragma unroll
      for (int i = 0; i < EPL / 4; ++i) dst[i] = make_float4(f[it][4 * i], f[it][4 * i + 1], f[it][4 * i + 2], f[it][4 * i + 3]);
      continue;
    }
    uint16_t* dst = static_cast<uint16_t*>(base) + at;
    if constexpr (IN != PA_DTYPE_F32) {
      if (isv && (IN == PA_DTYPE_BF16) == bf) {  // the same 16-bit type: the bits as they are
        *reinterpret_cast<uint4*>(dst) = raw[it];
        continue;
      }
    }
    uint32_t w[EPL / 2];
#pragma unroll
    for (int i = 0; i < EPL / 2; ++i)
      w[i] = bf ? pack2<true>(f[it][2 * i], f[it][2 * i + 1]) : pack2<false>(f[it][2 * i], f[it][2 * i + 1]);
    if constexpr (EPL == 8) *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
    else *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  }
}

template <int IN, int D>
cudaError_t launch_rot(const WriteParams& p, const RotateParams& r, cudaStream_t stream) {
  using C = RCfg<IN, D>;
  const long long units = (p.Hkv + C::HG - 1) / C::HG + (r.Hq + C::ROWS - 1) / C::ROWS;
  const long long blocks = (p.T * units * 32 + ROT_THREADS - 1) / ROT_THREADS;
  auto kern = r.pairs ? kv_rotate_kernel<IN, D, true> : kv_rotate_kernel<IN, D, false>;
  return launch_pdl(kern, dim3(static_cast<unsigned>(blocks)), dim3(ROT_THREADS), 0, stream, p, r);
}

template <int IN>
cudaError_t launch_rot_in(const WriteParams& p, const RotateParams& r, cudaStream_t stream) {
  return p.D == 64 ? launch_rot<IN, 64>(p, r, stream) : launch_rot<IN, 128>(p, r, stream);
}

}  // namespace

cudaError_t launch_kv_rotate(const WriteParams& p, const RotateParams& r, cudaStream_t stream) {
  if (p.T == 0) return cudaSuccess;
  switch (p.in_dtype) {
    case PA_DTYPE_F32:
      return launch_rot_in<PA_DTYPE_F32>(p, r, stream);
    case PA_DTYPE_BF16:
      return launch_rot_in<PA_DTYPE_BF16>(p, r, stream);
    default:
      return launch_rot_in<PA_DTYPE_F16>(p, r, stream);
  }
}

}  // namespace pa
