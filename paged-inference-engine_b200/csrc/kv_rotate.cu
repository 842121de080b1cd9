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
// Bound by latency: for prompts of the loads (long scoreboard is the first stall, 36-42 % of the warps' places are
// filled, 37-56 % of the issue slots, 16-47 % of DRAM), for a decode step's few rows of one launch.  One warp per (token, unit): a
// unit is up to ROWS query rows, key rows or value rows of one token, all loaded before the first is
// used; the table row is loaded once a warp and serves all of the unit's rows, which is why a unit does not cross tokens.
// Where whole heads are rotated by halves (FULL), a lane takes the same few dims of both halves, so both of a pair are
// its own and a cos and a sin serve two dims.  With fewer dims rotated, the partner lies
// in another lane of the same warp and comes by shuffles of packed words.  16384 tokens of 32 + 8 + 8 heads, INT8
// pool: 87 us (120 with shuffles for all, K and V rows in one warp and arithmetic a value at a time); 3001 tokens into a bf16
// pool 17 us, 64 into INT8 3.6, one 2.4.
#include "pa_common.cuh"
#include "quant.cuh"

namespace pa {
namespace {

constexpr int ROT_THREADS = 256;
enum : int { ROT_HALVES = 0, ROT_PAIRS = 1, ROT_FULL = 2 };

template <int IN, int D>
struct RCfg {
  static constexpr int ESZ = IN == PA_DTYPE_F32 ? 4 : 2;
  static constexpr int EPL = 16 / ESZ;  // elements of a lane
  static constexpr int LPR = D / EPL;   // lanes per row
  static constexpr int RPI = 32 / LPR;  // rows per load instruction
  static constexpr int NL = 4;          // rows of a lane, in flight together
  static constexpr int ROWS = NL * RPI;
  static_assert(LPR <= 32 && 32 % LPR == 0, "a row maps onto whole lanes");
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

// A lane's elements of a row: EPL neighbours, or (SPLIT) EPL / 2 neighbours of either half of the row.
template <int D, int EPL, bool SPLIT>
__device__ __forceinline__ int run_start(int part, int run) {
  return SPLIT ? run * (D / 2) + part * (EPL / 2) : part * EPL + run * (EPL / 2);
}
template <int ESZ, int D, int EPL, bool SPLIT>
__device__ __forceinline__ uint4 load_row(const char* row, int part) {
  if constexpr (SPLIT) {
    const uint2 a = *reinterpret_cast<const uint2*>(row + run_start<D, EPL, true>(part, 0) * ESZ);
    const uint2 b = *reinterpret_cast<const uint2*>(row + run_start<D, EPL, true>(part, 1) * ESZ);
    return make_uint4(a.x, a.y, b.x, b.y);
  } else {
    return *reinterpret_cast<const uint4*>(row + part * EPL * ESZ);
  }
}
// N bytes (2, 4, 8 or 16) of packed words.
template <int N>
__device__ __forceinline__ void store_bytes(char* at, const uint32_t* w) {
  if constexpr (N == 2) *reinterpret_cast<uint16_t*>(at) = static_cast<uint16_t>(w[0]);
  else if constexpr (N == 4) *reinterpret_cast<uint32_t*>(at) = w[0];
  else if constexpr (N == 8) *reinterpret_cast<uint2*>(at) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint4*>(at) = make_uint4(w[0], w[1], w[2], w[3]);
}
// The lane's EPL elements as OSZ-byte values in the words w, to its one or two places in `row`.
template <int OSZ, int D, int EPL, bool SPLIT>
__device__ __forceinline__ void store_row(char* row, int part, const uint32_t* w) {
  constexpr int RUN = EPL / 2 * OSZ;  // bytes of a run
  if constexpr (SPLIT || RUN * 2 > 16) {
    store_bytes<RUN>(row + run_start<D, EPL, SPLIT>(part, 0) * OSZ, w);
    const uint32_t half = w[0] >> 16;  // (runs of two bytes: both in the first word)
    store_bytes<RUN>(row + run_start<D, EPL, SPLIT>(part, 1) * OSZ, RUN == 2 ? &half : w + RUN / 4);
  } else {
    store_bytes<2 * RUN>(row + part * EPL * OSZ, w);
  }
}

// This lane's part of a table row.  HALVES: a cos and a sin per dim, the sin with the sign that the partner's
// product carries; PAIRS and FULL: one of each per pair.  (Scalar arithmetic: packed products, .rn or not, were found
// contracted with the additions behind them.)
template <int MODE, int EPL>
struct Turn {
  static constexpr int N = MODE == ROT_HALVES ? EPL : EPL / 2;
  float c[N], s[N];
  int src;   // HALVES: lane that holds the partner dims
  bool on;   // dims below rot_dim

  __device__ __forceinline__ void load(const float* row, int rot, int part, int lane) {
    const int half = rot >> 1;
    const int d = part * EPL;
    on = MODE == ROT_FULL || d < rot;
    src = lane;
    if (!on) return;
    float sign = 1.f;
    int at = part * (EPL / 2);
    if constexpr (MODE == ROT_HALVES) {
      const bool low = d < half;  // half is a multiple of EPL: a lane's dims lie on one side
      sign = low ? -1.f : 1.f;
      src = low ? lane + half / EPL : lane - half / EPL;
      at = low ? d : d - half;
    }
#pragma unroll
    for (int i = 0; i < N; i += N < 4 ? 2 : 4) {
      if constexpr (N >= 4) {
        const float4 a = __ldg(reinterpret_cast<const float4*>(row + at + i));
        const float4 b = __ldg(reinterpret_cast<const float4*>(row + half + at + i));
        c[i] = a.x, c[i + 1] = a.y, c[i + 2] = a.z, c[i + 3] = a.w;
        s[i] = b.x * sign, s[i + 1] = b.y * sign, s[i + 2] = b.z * sign, s[i + 3] = b.w * sign;
      } else {
        const float2 a = __ldg(reinterpret_cast<const float2*>(row + at));
        const float2 b = __ldg(reinterpret_cast<const float2*>(row + half + at));
        c[0] = a.x, c[1] = a.y;
        s[0] = b.x * sign, s[1] = b.y * sign;
      }
    }
  }

  // f: the rotated elements of a row, from those loaded.  Every lane of the warp calls it.
  template <int IN>
  __device__ __forceinline__ void apply(const uint4& raw, float (&f)[EPL]) const {
    unpack_words<IN, EPL>(raw, f);
    if constexpr (MODE == ROT_HALVES) {
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
    } else if (on) {
#pragma unroll
      for (int i = 0; i < EPL / 2; ++i) {
        const int x = MODE == ROT_FULL ? i : 2 * i, y = MODE == ROT_FULL ? i + EPL / 2 : 2 * i + 1;
        const float a = f[x], b = f[y];
        f[x] = __fsub_rn(__fmul_rn(a, c[i]), __fmul_rn(b, s[i]));
        f[y] = __fadd_rn(__fmul_rn(b, c[i]), __fmul_rn(a, s[i]));
      }
    }
  }
};

// quant_row_fast on pairs of values: the codes' words, and whether a quotient lies near a rounding boundary.
template <int EPL>
__device__ __forceinline__ bool quant_pairs(const float (&f)[EPL], float inv, uint32_t* w) {
  const uint64_t k = f2_pack(inv, inv), up = f2_pack(RNE_MAGIC, RNE_MAGIC), down = f2_pack(-RNE_MAGIC, -RNE_MAGIC);
  const uint64_t minus = f2_pack(-1.f, -1.f);
  float far = 0.f;
  uint32_t b[EPL];
#pragma unroll
  for (int i = 0; i < EPL; i += 2) {
    const uint64_t y = f2_fma(f2_pack(f[i], f[i + 1]), k, f2_pack(-0.f, -0.f));  // the product (near checks cover its rounding)
    const uint64_t t = f2_add(y, up);
    float d0, d1, t0, t1;
    f2_unpack(f2_fma(f2_add(t, down), minus, y), d0, d1);  // y - rint(y)
    f2_unpack(t, t0, t1);
    far = fmaxf(far, fmaxf(fabsf(d0), fabsf(d1)));
    b[i] = __float_as_uint(t0);
    b[i + 1] = __float_as_uint(t1);
  }
#pragma unroll
  for (int i = 0; i < EPL / 4; ++i) w[i] = pack_bytes(b[4 * i], b[4 * i + 1], b[4 * i + 2], b[4 * i + 3]);
  return far > NEAR_HALF;
}

// One row of K or V into the pool: this lane's elements f (raw: as loaded), its row at element offset `at`, scale at `so`.
template <int IN, int D, bool SPLIT>
__device__ __forceinline__ void write_row(const WriteParams& p, const float (&f)[RCfg<IN, D>::EPL], const uint4& raw, bool same,
                                          bool live, void* base, long long at, void* sbase, long long so, int part) {
  using C = RCfg<IN, D>;
  constexpr int EPL = C::EPL;
  if (p.cache_dtype == PA_DTYPE_I8) {
    float am = fmaxf(fabsf(f[0]), fabsf(f[1]));
#pragma unroll
    for (int i = 2; i < EPL; i += 2) am = fmax3f(am, fabsf(f[i]), fabsf(f[i + 1]));
#pragma unroll
    for (int o = C::LPR / 2; o >= 1; o >>= 1) am = fmaxf(am, __shfl_xor_sync(0xffffffffu, am, o));
    const float sc = am == 0.f ? 1.0f : div127_rn(am);
    uint32_t w[EPL / 4];
    // the reciprocal of a scale below 2^-126 is not finite: such rows, too, take the division
    const bool near = quant_pairs<EPL>(f, rcp_approx(sc), w) || sc < 1.2e-38f;
    if (__any_sync(0xffffffffu, near)) quant_row_exact<EPL>(f, sc, w);
    if (!live) return;
    store_row<1, D, EPL, SPLIT>(static_cast<char*>(base) + at, part, w);
    if (part == 0) {
      if (p.scale_f32) static_cast<float*>(sbase)[so] = sc;
      else static_cast<__half*>(sbase)[so] = __float2half_rn(sc);
    }
    return;
  }
  if (!live) return;
  if (p.cache_dtype == PA_DTYPE_F32) {
    store_row<4, D, EPL, SPLIT>(static_cast<char*>(base) + at * 4, part, reinterpret_cast<const uint32_t*>(f));
    return;
  }
  const bool bf = p.cache_dtype == PA_DTYPE_BF16;
  uint32_t w[EPL / 2];
#pragma unroll
  for (int i = 0; i < EPL / 2; ++i) w[i] = bf ? pack2<true>(f[2 * i], f[2 * i + 1]) : pack2<false>(f[2 * i], f[2 * i + 1]);
  if constexpr (IN != PA_DTYPE_F32) {
    if (same) {  // values of the pool's own type: the bits as they are
      w[0] = raw.x, w[1] = raw.y, w[2] = raw.z, w[3] = raw.w;
    }
  }
  store_row<2, D, EPL, SPLIT>(static_cast<char*>(base) + at * 2, part, w);
}

template <int IN, int D, int MODE>
__global__ void __launch_bounds__(ROT_THREADS, 4) kv_rotate_kernel(const WriteParams p, const RotateParams r) {
  pdl_enter();
  using C = RCfg<IN, D>;
  constexpr int EPL = C::EPL;
  constexpr bool SPLIT = MODE == ROT_FULL;
  const int lane = threadIdx.x & 31;
  const int kv_units = (p.Hkv + C::ROWS - 1) / C::ROWS;
  const int q_units = (r.Hq + C::ROWS - 1) / C::ROWS;
  const int units = q_units + 2 * kv_units;
  const long long wid = (static_cast<long long>(blockIdx.x) * ROT_THREADS + threadIdx.x) >> 5;
  if (wid >= static_cast<long long>(p.T) * units) return;
  const int t = static_cast<int>(wid / units);
  int u = static_cast<int>(wid - static_cast<long long>(t) * units);
  const int part = lane % C::LPR;
  const int sub = lane / C::LPR;
  const int kind = u < q_units ? 0 : u < q_units + kv_units ? 1 : 2;  // queries, keys, values
  u -= kind == 0 ? 0 : kind == 1 ? q_units : q_units + kv_units;
  const int h0 = u * C::ROWS;
  const int H = kind == 0 ? r.Hq : p.Hkv;
  const char* src = static_cast<const char*>(kind == 0 ? r.q : kind == 1 ? p.k_new : p.v_new);
  const long long src_t = kind == 0 ? r.q_st : kind == 1 ? p.kn_st : p.vn_st;
  const long long src_h = kind == 0 ? r.q_sh : kind == 1 ? p.kn_sh : p.vn_sh;

  uint4 raw[C::NL];
#pragma unroll
  for (int it = 0; it < C::NL; ++it) {
    const int h = h0 + it * C::RPI + sub;
    raw[it] = make_uint4(0, 0, 0, 0);
    if (h < H) {
      const char* row = src + (t * src_t + h * src_h) * C::ESZ;
      raw[it] = kind < 2 ? load_row<C::ESZ, D, EPL, SPLIT>(row, part) : load_row<C::ESZ, D, EPL, false>(row, part);
    }
  }
  const int pos = p.pos[t];
  const int s = kind == 0 ? 0 : p.seq_idx[t];
  if (pos < 0 || pos >= r.num_pos) {
    if (lane == 0) set_status(p.status, ST_BAD_POSITION);
    return;
  }
  // the block and the angles at once: one more round of latency, not two
  const int bi = pos >> p.log2BS;
  const bool placed = s >= 0 && s < p.num_seqs && bi < p.bt_cols;
  int blk = -1;
  if (kind > 0 && placed) blk = p.bt[s * p.bt_ss + bi * p.bt_sc];
  Turn<MODE, EPL> turn;
  if (kind < 2) turn.load(r.table + pos * r.table_stride, r.rot, part, lane);

  if (kind == 0) {
#pragma unroll
    for (int it = 0; it < C::NL; ++it) {
      const int h = h0 + it * C::RPI + sub;
      float f[EPL];
      turn.template apply<IN>(raw[it], f);
      if (h < H) {
        const uint4 w = pack_words<IN, EPL>(f);
        const uint32_t x[4] = {w.x, w.y, w.z, w.w};
        store_row<C::ESZ, D, EPL, SPLIT>(static_cast<char*>(r.q_out) + (t * r.qo_st + h * r.qo_sh) * C::ESZ, part, x);
      }
    }
    return;
  }
  // ---- K and V rows, where kv_write_kernel puts them --------------------------
  if (blk < 0 || blk >= p.NB) {
    if (lane == 0)
      set_status(p.status, placed ? ST_BAD_BLOCK_ID : (s < 0 || s >= p.num_seqs) ? ST_BAD_SEQ_INDEX : ST_BAD_POSITION);
    return;
  }
  const int slot = pos & (p.BS - 1);
  const bool same = kind == 2 && IN == p.cache_dtype;
  const long long at0 = kind == 1 ? blk * p.k_sblk + slot * p.k_sslot : blk * p.v_sblk + slot * p.v_sslot;
  const long long so0 = kind == 1 ? blk * p.ks_sblk + slot * p.ks_sslot : blk * p.vs_sblk + slot * p.vs_sslot;
  if (kind == 1) {
#pragma unroll
    for (int it = 0; it < C::NL; ++it) {
      const int h = h0 + it * C::RPI + sub;
      float f[EPL];
      turn.template apply<IN>(raw[it], f);
      write_row<IN, D, SPLIT>(p, f, raw[it], false, h < H, p.k, at0 + h * p.k_shead, p.ks, so0 + h * p.ks_shead, part);
    }
  } else {
#pragma unroll
    for (int it = 0; it < C::NL; ++it) {
      const int h = h0 + it * C::RPI + sub;
      float f[EPL];
      unpack_words<IN, EPL>(raw[it], f);
      write_row<IN, D, false>(p, f, raw[it], same, h < H, p.v, at0 + h * p.v_shead, p.vs, so0 + h * p.vs_shead, part);
    }
  }
}

template <int IN, int D>
cudaError_t launch_rot(const WriteParams& p, const RotateParams& r, cudaStream_t stream) {
  using C = RCfg<IN, D>;
  const long long units = 2 * ((p.Hkv + C::ROWS - 1) / C::ROWS) + (r.Hq + C::ROWS - 1) / C::ROWS;
  const long long blocks = (p.T * units * 32 + ROT_THREADS - 1) / ROT_THREADS;
  auto kern = r.pairs ? kv_rotate_kernel<IN, D, ROT_PAIRS>
              : r.rot == D ? kv_rotate_kernel<IN, D, ROT_FULL> : kv_rotate_kernel<IN, D, ROT_HALVES>;
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
