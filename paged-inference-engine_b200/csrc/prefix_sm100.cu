// Attention of many query rows over a shared prefix on the 5th-generation
// tensor cores (tcgen05 + TMEM).
//
// A group's rows over one kv head (sequences x query rows x group heads) are cut into tiles of
// 128, its shared keys into tiles of 128.  A work unit is one of each; units lie in the
// order (group, kv head, row tile, key tile), and every CTA of a persistent grid takes an equal
// run of them.  A run's part within one (group, kv head, row tile) is a piece: its 128 rows'
// statistics and unnormalised sums go to the workspace, where prefix_merge_kernel
// joins them (csrc/prefix_plan.cu).  Every row sees every shared key (the plan sees to it), so
// the only mask is the end of the last tile.
//
// The two softmax groups of a CTA take the key tiles of a piece in turn, each with its own logits,
// maximum and sum in TMEM (S0 S1 O0 O1): while one turns its logits into
// probabilities, the tensor core works for the other, as with the two heads of
// csrc/prefill_sm100.cu, but with one row tile, so that few rows do not leave half of the CTA idle.
// At the end of a piece the two results are joined in registers and written once.
//
//   warps 0-7    softmax: a thread per row (TMEM lane) and stream (w >> 2); they also load and convert Q
//   warp 8       producer: K and V boxes gathered through the block table by TMA
//   warp 9       MMA issuer
//   warps 10-13  INT8 pools: raw tiles -> fp16 operand tiles, q * scale in fp32 rounded once, as
//                csrc/kv_dequant.cu does for prompts; the raw bytes cross HBM once and the
//                fp16 tile never leaves the SM
//
// Bound by HBM up to about 256 rows a kv head (16-bit pools), by the softmax chain beyond.
#include <atomic>

#include "pa_common.cuh"

namespace pa {
namespace {

constexpr int W_HALF = 128 * 128;  // 64 columns (128 bytes) of a 128-row tile
constexpr uint32_t W_TMEM = 512;
constexpr uint32_t W_OCOL = 256;
constexpr float W_THRESHOLD = 8.0f;  // growth of the maximum (log2) that rescales
constexpr int W_SOFTMAX = 8;         // warps
constexpr int W_PRODUCER = 8, W_MMA = 9, W_CONVERT = 10;

template <int D, bool I8>
struct WideCfg {
  static constexpr int TILE = (D / 64) * W_HALF;      // fp16 / bf16 operand tile of 128 rows
  static constexpr int RAW = 128 * D;                 // int8 tile
  static constexpr int ST = I8 ? 2 : (D == 128 ? 3 : 6);  // K stages, and V stages
  static constexpr int RST = I8 ? (D == 128 ? 4 : 8) : 0;  // raw tiles in flight, K and V alternating
  static constexpr int K0 = TILE;
  static constexpr int V0 = K0 + ST * TILE;
  static constexpr int R0 = V0 + ST * TILE;
  static constexpr int BAR = R0 + RST * RAW;
  static constexpr int B_QREADY = 0, B_QEMPTY = 1, B_SFULL = 2, B_PFULL = 4, B_ODONE = 6, B_SLOT = 8, B_PLACE = 9,
                       B_KFULL = 11, B_KEMPTY = B_KFULL + ST, B_VFULL = B_KEMPTY + ST, B_VEMPTY = B_VFULL + ST,
                       B_RFULL = B_VEMPTY + ST, B_REMPTY = B_RFULL + RST, B_END = B_REMPTY + RST;
  static constexpr int XCH = BAR + 512 / (D == 128 ? 2 : 1);
  static constexpr int SMEM = XCH + 1024 + 1024;  // exchange of the two streams, alignment
  static constexpr int THREADS = 32 * (I8 ? W_CONVERT + 4 : W_CONVERT);
  static_assert(B_END * 8 <= XCH - BAR && SMEM <= 227 * 1024, "shared memory per CTA");
};

__device__ unsigned int g_wide_abort = 0;  // launch generation in which a wait gave up

__device__ __noinline__ void wide_wait_slow(const SharedParams& p, uint32_t bar, uint32_t parity) {
  for (int i = 0; i < (1 << 20); ++i) {
    if (mbar_try_wait(bar, parity)) return;
    if ((i & 1023) == 1023 && *reinterpret_cast<volatile unsigned int*>(&g_wide_abort) == p.abort_gen) return;
  }
  atomicExch(&g_wide_abort, p.abort_gen);
  set_status(p.status, ST_WAIT_TIMEOUT);
}
__device__ __forceinline__ void wide_wait(const SharedParams& p, uint32_t bar, uint32_t parity) {
  if (!mbar_try_wait(bar, parity)) wide_wait_slow(p, bar, parity);
}
__device__ __forceinline__ void wide_barrier(int id, int n) { asm volatile("bar.sync %0, %1;\n" ::"r"(id), "r"(n) : "memory"); }

// The pieces of a CTA's run of units, walked alike by every role.
struct Pieces {
  int left;                  // units of the run not walked yet
  int g, kvh, rt, t;         // group, kv head, row tile, first key tile
  int keys, first, n, lead;  // of the group
  int rows, RT, KT;

  __device__ __forceinline__ void group(const SharedParams& p) {
    const int4 v = p.grp[g];
    keys = v.x, first = v.y, n = v.z, lead = v.w;
    rows = n * p.maxq * p.G;
    RT = (rows + kWideRows - 1) / kWideRows;
    KT = (keys + kWideKeys - 1) / kWideKeys;
  }
  __device__ __forceinline__ void begin(const SharedParams& p, int u0, int u1, int g0) {
    left = u1 - u0;
    g = g0;
    if (left <= 0) return;
    group(p);
    const int u = u0 - p.unit0[g];
    t = u % KT;
    rt = u / KT % RT;
    kvh = u / KT / RT;
  }
  __device__ __forceinline__ int tiles() const { return min(KT - t, left); }  // of this piece
  __device__ __forceinline__ void next(const SharedParams& p) {
    left -= tiles();
    t = 0;
    if (++rt == RT) {
      rt = 0;
      if (++kvh == p.Hkv) {
        kvh = 0;
        if (left > 0) {
          do {
            ++g;
          } while (p.grp[g].x == 0);  // a group with units is still ahead
          group(p);
        }
      }
    }
  }
};

template <int D, bool MMA_BF16, bool QBF16, bool I8>
__global__ void __launch_bounds__(WideCfg<D, I8>::THREADS, 1)
    prefix_wide_kernel(const SharedParams p, const __grid_constant__ KvMaps maps) {
  pdl_enter();
  using C = WideCfg<D, I8>;
  constexpr int ST = C::ST, TILE = C::TILE;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* sm = smem_raw + (base - raw);
  auto bar = [&](int i) { return base + C::BAR + 8u * i; };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  const int units = p.unit0[p.groups];
  const int chunk = (units + p.wide_ctas - 1) / p.wide_ctas;
  const int u0 = static_cast<int>(blockIdx.x) * chunk, u1 = min(u0 + chunk, units);
  if (u0 >= u1) return;

  if (warp == 0) {
    // the group of unit u0: the last with unit0[g] <= u0, found 32 at a time
    int lo = 0, hi = p.groups;  // unit0[lo] <= u0 < unit0[hi]
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int at = lo + lane * step;
      const unsigned le = __ballot_sync(0xffffffffu, at < hi && p.unit0[min(at, hi)] <= u0);
      const int last = 31 - __clz(le);  // lane 0 always holds
      lo += last * step;
      hi = min(hi, lo + step);
    }
    if (lane == 0) *reinterpret_cast<volatile int*>(sm + C::BAR + 8 * C::B_PLACE) = lo;
  }
  if (tid == 32) {
    mbar_init(bar(C::B_QREADY), 32 * W_SOFTMAX);
    mbar_init(bar(C::B_QEMPTY), 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(bar(C::B_SFULL + x), 1);
      mbar_init(bar(C::B_PFULL + x), 16 * W_SOFTMAX);
      mbar_init(bar(C::B_ODONE + x), 1);
    }
    for (int s = 0; s < ST; ++s) {
      mbar_init(bar(C::B_KFULL + s), I8 ? 128 : 1);
      mbar_init(bar(C::B_KEMPTY + s), 1);
      mbar_init(bar(C::B_VFULL + s), I8 ? 128 : 1);
      mbar_init(bar(C::B_VEMPTY + s), 1);
    }
    for (int s = 0; s < C::RST; ++s) {
      mbar_init(bar(C::B_RFULL + s), 1);
      mbar_init(bar(C::B_REMPTY + s), 128);
    }
    fence_mbar_init();
  }
  if (warp == W_MMA) {
    tmem_alloc(bar(C::B_SLOT), W_TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + C::BAR + 8 * C::B_SLOT);
  Pieces it;
  it.begin(p, u0, u1, *reinterpret_cast<volatile int*>(sm + C::BAR + 8 * C::B_PLACE));

  if (warp == W_PRODUCER) {
    // ------------------------------------------------------------ producer
    // Lane i owns box i of every tile; the block ids of a tile are fetched one tile ahead.
    const int boxs = p.BS < 16 ? p.BS : 16;
    const int nbox = kWideKeys / boxs;  // <= 16 (block_size >= 8)
    int gt = 0;
    for (; it.left > 0; it.next(p)) {
      const int* bt_row = p.bt + static_cast<long long>(it.lead) * p.bt_ss;
      auto fetch = [&](int j) {
        const int key = (it.t + j) * kWideKeys + lane * boxs;
        int blk = p.NB;  // out of range: TMA fills the box with zeros
        if (lane < nbox && key < it.keys) {
          const int x = bt_row[static_cast<long long>(key >> p.log2BS) * p.bt_sc];
          if (x >= 0 && x < p.NB) blk = x;
          else set_status(p.status, ST_BAD_BLOCK_ID);
        }
        return blk;
      };
      const int n = it.tiles();
      int blk = fetch(0);
      for (int j = 0; j < n; ++j, ++gt) {
        const int blk_next = j + 1 < n ? fetch(j + 1) : p.NB;
        const int slot = blk < p.NB ? (it.t * kWideKeys + j * kWideKeys + lane * boxs) & (p.BS - 1) : 0;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
          uint32_t dst, full;
          if constexpr (I8) {
            const int i = 2 * gt + v, s = i % C::RST;
            full = bar(C::B_RFULL + s);
            dst = base + C::R0 + s * C::RAW + lane * boxs * D;
            if (lane == 0) {
              if (i >= C::RST) wide_wait(p, bar(C::B_REMPTY + s), (i / C::RST - 1) & 1);
              mbar_arrive_expect_tx(full, C::RAW);
            }
          } else {
            const int s = gt % ST;
            full = bar((v ? C::B_VFULL : C::B_KFULL) + s);
            dst = base + (v ? C::V0 : C::K0) + s * TILE + lane * boxs * 128;
            if (lane == 0) {
              if (gt >= ST) wide_wait(p, bar((v ? C::B_VEMPTY : C::B_KEMPTY) + s), (gt / ST - 1) & 1);
              mbar_arrive_expect_tx(full, TILE);
            }
          }
          __syncwarp();
          if (lane < nbox) {
            const CUtensorMap* m = v ? &maps.v : &maps.k;
            tma_load_4d(dst, m, full, 0, it.kvh, slot, blk);
            if constexpr (!I8 && D == 128) tma_load_4d(dst + W_HALF, m, full, 64, it.kvh, slot, blk);
          }
        }
        blk = blk_next;
      }
    }
  } else if (warp == W_MMA) {
    // ------------------------------------------------------------ MMA issuer
    if (lane == 0) {
      constexpr uint32_t IDESC_QK = instr_desc_f16(MMA_BF16, false, false, kWideRows, kWideKeys);
      constexpr uint32_t IDESC_PV = instr_desc_f16(MMA_BF16, false, true, kWideRows, D);
      int gt = 0, piece = 0;
      int px[2] = {0, 0};  // probabilities taken of each stream
      for (; it.left > 0; it.next(p), ++piece) {
        const int n = it.tiles();
        auto qk = [&](int j) {
          const int x = j & 1, s = (gt + j) % ST;
          wide_wait(p, bar(C::B_KFULL + s), ((gt + j) / ST) & 1);
          tc_fence_after();
          const uint64_t a = smem_desc(base, 16, 1024), b = smem_desc(base + C::K0 + s * TILE, 16, 1024);
          const uint32_t d = tmem + 128u * x;
          if constexpr (D == 128) {
            tc_mma_ss_k128<W_HALF / 16, W_HALF / 16>(d, a, b, IDESC_QK);
          } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) tc_mma_ss(d, a + 2 * k, b + 2 * k, IDESC_QK, k > 0);
          }
          tc_commit(bar(C::B_SFULL + x));
          tc_commit(bar(C::B_KEMPTY + s));
          if (j == n - 1) tc_commit(bar(C::B_QEMPTY));
        };
        wide_wait(p, bar(C::B_QREADY), piece & 1);
        tc_fence_after();
        qk(0);
        if (n > 1) qk(1);
        for (int j = 0; j < n; ++j) {
          const int x = j & 1, s = (gt + j) % ST;
          wide_wait(p, bar(C::B_VFULL + s), ((gt + j) / ST) & 1);
          wide_wait(p, bar(C::B_PFULL + x), px[x] & 1);
          ++px[x];
          tc_fence_after();
          tc_mma_ts_seq<8>(tmem + W_OCOL + 128u * x, tmem + 128u * x, smem_desc(base + C::V0 + s * TILE, W_HALF, 1024),
                           IDESC_PV, j >= 2 ? 1u : 0u);
          tc_commit(bar(C::B_VEMPTY + s));
          tc_commit(bar(C::B_ODONE + x));
          if (j + 2 < n) qk(j + 2);
        }
        gt += n;
      }
    }
  } else if (warp >= W_CONVERT) {
    // ------------------------------------------------------------ INT8 -> fp16 tiles
    if constexpr (I8) {
      // Warp c converts rows 32 c .. 32 c + 31 of every tile; lane l holds the scales of row 32 c + l.
      constexpr int CH = D / 16;        // 16-byte pieces of a raw row
      constexpr int RPI = 32 / CH;      // rows an iteration of a warp
      const int c = warp - W_CONVERT;
      const int ch = lane % CH;
      int gt = 0;
      for (; it.left > 0; it.next(p)) {
        const int* bt_row = p.bt + static_cast<long long>(it.lead) * p.bt_ss;
        const int n = it.tiles();
        auto block = [&](int j) {
          const int key = (it.t + j) * kWideKeys + 32 * c + lane;
          return j < n && key < it.keys ? bt_row[static_cast<long long>(key >> p.log2BS) * p.bt_sc] : -1;
        };
        auto scales = [&](int j, int blk, float& k, float& v) {
          k = v = 0.f;  // keys past the end, and of blocks outside the pool, are zeros
          if (blk < 0 || blk >= p.NB) return;
          const int slot = ((it.t + j) * kWideKeys + 32 * c + lane) & (p.BS - 1);
          k = load_scale(p.ks, blk * p.ks_sblk + slot * p.ks_sslot + it.kvh * p.ks_shead, p.scale_f32);
          v = load_scale(p.vs, blk * p.vs_sblk + slot * p.vs_sslot + it.kvh * p.vs_shead, p.scale_f32);
        };
        float sk, sv, sk1, sv1;
        scales(0, block(0), sk, sv);
        int blk1 = block(1);
        for (int j = 0; j < n; ++j, ++gt) {
          const int blk2 = block(j + 2);
          scales(j + 1, blk1, sk1, sv1);
          const int s = gt % ST;
#pragma unroll
          for (int v = 0; v < 2; ++v) {
            const int i = 2 * gt + v, rs = i % C::RST;
            const unsigned char* src = sm + C::R0 + rs * C::RAW;
            unsigned char* dst = sm + (v ? C::V0 : C::K0) + s * TILE;
            const float mine = v ? sv : sk;
            wide_wait(p, bar(C::B_RFULL + rs), (i / C::RST) & 1);
            if (gt >= ST) wide_wait(p, bar((v ? C::B_VEMPTY : C::B_KEMPTY) + s), (gt / ST - 1) & 1);
#pragma unroll 4
            for (int k = 0; k < 32 / RPI; ++k) {
              const int lr = k * RPI + lane / CH;  // row within the warp's 32
              const int r = 32 * c + lr;
              const float f = __shfl_sync(0xffffffffu, mine, lr);
              const int at = D == 128 ? r * 128 + ((ch ^ (r & 7)) << 4) : r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
              const uint4 w = *reinterpret_cast<const uint4*>(src + at);
              const uint32_t x[4] = {w.x, w.y, w.z, w.w};
              uint32_t o[8];
#pragma unroll
              for (int q = 0; q < 4; ++q) {
                uint32_t a, b;
                i8x4_to_f16x4(x[q], a, b);
                const float2 fa = __half22float2(*reinterpret_cast<__half2*>(&a));
                const float2 fb = __half22float2(*reinterpret_cast<__half2*>(&b));
                o[2 * q] = pack_f16(fa.x * f, fa.y * f);
                o[2 * q + 1] = pack_f16(fb.x * f, fb.y * f);
              }
              // dims 16 ch .. 16 ch + 15: two pieces of 64-column half ch / 4; the upper half's lanes store them the
              // other way round, so that a row's lanes meet every bank once
              const int half = ch >> 2, odd = half & 1;
              unsigned char* row = dst + half * W_HALF + r * 128;
              const int p0 = 2 * (ch & 3);
              const uint4 lo = make_uint4(o[0], o[1], o[2], o[3]), hi = make_uint4(o[4], o[5], o[6], o[7]);
              *reinterpret_cast<uint4*>(row + (((p0 + odd) ^ (r & 7)) << 4)) = odd ? hi : lo;
              *reinterpret_cast<uint4*>(row + (((p0 + 1 - odd) ^ (r & 7)) << 4)) = odd ? lo : hi;
            }
            fence_proxy_async_smem();
            mbar_arrive(bar((v ? C::B_VFULL : C::B_KFULL) + s));
            mbar_arrive(bar(C::B_REMPTY + rs));
          }
          sk = sk1, sv = sv1, blk1 = blk2;
        }
      }
    }
  } else {
    // ------------------------------------------------------------ softmax
    const int x = warp >> 2;
    const int r = tid & 127;  // row of the tile = TMEM lane
    const uint32_t trow = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16);
    const uint32_t scol = trow + 128u * x, ocol = trow + W_OCOL + 128u * x;
    float* xch = reinterpret_cast<float*>(sm + C::XCH);  // [2 streams][128 rows]
    const int per = p.maxq * p.G;
    int done[2] = {0, 0};  // tiles of each stream
    for (int piece = 0; it.left > 0; it.next(p), ++piece) {
      const int n = it.tiles();
      const int live = min(kWideRows, it.rows - it.rt * kWideRows);  // rows of this tile
      const bool busy = 32 * (warp & 3) < live;                      // this warp holds one
      // ---- Q: 16-byte pieces of the 128 rows, converted to the operand type, swizzled
      if (piece > 0) wide_wait(p, bar(C::B_QEMPTY), (piece - 1) & 1);
#pragma unroll 4
      for (int i = 0; i < 128 * (D / 8) / 256; ++i) {
        const int idx = i * 256 + tid;
        const int row = idx / (D / 8), c = idx % (D / 8);
        uint4 w = make_uint4(0, 0, 0, 0);
        if (row < live) {
          const int R = it.rt * kWideRows + row;
          const int m = R / per, rem = R - m * per;
          const int qi = rem / p.G, b = it.first + m;
          if (qi < seq_rows(p, b)) {
            w = *(reinterpret_cast<const uint4*>(static_cast<const unsigned short*>(p.q) + q_seq_base(p, b) +
                                                 (it.kvh * p.G + rem - qi * p.G) * p.q_sh + static_cast<long long>(qi) * p.q_sm) + c);
            w.x = cvt_pair<QBF16, MMA_BF16>(w.x);
            w.y = cvt_pair<QBF16, MMA_BF16>(w.y);
            w.z = cvt_pair<QBF16, MMA_BF16>(w.z);
            w.w = cvt_pair<QBF16, MMA_BF16>(w.w);
          }
        }
        *reinterpret_cast<uint4*>(sm + (c >> 3) * W_HALF + row * 128 + (((c & 7) ^ (row & 7)) << 4)) = w;
      }
      fence_proxy_async_smem();
      mbar_arrive(bar(C::B_QREADY));

      float m_ref = -INFINITY, l = 0.f;
      for (int j = x; j < n; j += 2) {
        wide_wait(p, bar(C::B_SFULL + x), (done[x] + (j >> 1)) & 1);
        tc_fence_after();
        if (busy) {
          const int left = it.keys - (it.t + j) * kWideKeys;  // keys of this tile, maybe more than 128
          // first look: the row's maximum.  The logits are read again below: 128 of them do not fit the registers
          // beside the rest, and a second read of TMEM is cheap
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            uint32_t r0[32], r1[32];
            tmem_ld32(scol + 64 * c, r0);
            tmem_ld32(scol + 64 * c + 32, r1);
            tmem_wait_ld();
            if (left < kWideKeys) {
#pragma unroll
              for (int i = 0; i < 32; ++i) {
                if (64 * c + i >= left) r0[i] = 0xff800000u;  // -inf
                if (64 * c + 32 + i >= left) r1[i] = 0xff800000u;
              }
            }
#pragma unroll
            for (int i = 0; i < 32; ++i) mx4[i & 3] = fmax3f(mx4[i & 3], __uint_as_float(r0[i]), __uint_as_float(r1[i]));
          }
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
          float alpha = 1.f;
          bool resc = false;
          if (mx > m_ref + W_THRESHOLD) {  // also the first finite maximum
            alpha = ex2(m_ref - mx);
            resc = j >= 2;  // O holds this stream's earlier tiles
            m_ref = mx;
          }
          const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
          const float c2 = p.scale_log2;
          uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
          // P of keys [32 c, 32 c + 32) takes TMEM columns [16 c, 16 c + 16): behind the logits still to be read
          uint32_t rr[2][32];
          tmem_ld32(scol, rr[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_wait_ld();
            if (c < 3) tmem_ld32(scol + 32 * (c + 1), rr[(c + 1) & 1]);
            const uint32_t* s = rr[c & 1];
            uint32_t pk[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
              float p0, p1;
              f2_unpack(f2_fma(f2_pack(__uint_as_float(s[2 * i]), __uint_as_float(s[2 * i + 1])), f2_pack(c2, c2),
                               f2_pack(neg_m, neg_m)),
                        p0, p1);
              p0 = ex2(p0);
              p1 = ex2(p1);
              if (left < kWideKeys) {
                if (32 * c + 2 * i >= left) p0 = 0.f;
                if (32 * c + 2 * i + 1 >= left) p1 = 0.f;
              }
              sum[i & 1] = f2_add(sum[i & 1], f2_pack(p0, p1));
              pk[i] = pack2<MMA_BF16>(p0, p1);
            }
            tmem_st16(scol + 16 * c, pk);
          }
          float a0, a1, b0, b1;
          f2_unpack(sum[0], a0, a1);
          f2_unpack(sum[1], b0, b1);
          l = l * alpha + ((a0 + a1) + (b0 + b1));
          // S of this tile was issued behind the stream's last P*V, so that product is complete
          if (__any_sync(0xffffffffu, resc)) {
            const float a = resc ? alpha : 1.f;
#pragma unroll 1
            for (int c = 0; c < D / 32; ++c) {
              uint32_t o[32];
              tmem_ld32(ocol + 32 * c, o);
              tmem_wait_ld();
#pragma unroll
              for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * a);
              tmem_st32(ocol + 32 * c, o);
            }
          }
          tmem_wait_st();
        }
        tc_fence_before();
        mbar_arrive(bar(C::B_PFULL + x));
      }
      done[0] += (n + 1) / 2;
      done[1] += n / 2;
      // ---- end of the piece: the two streams' results joined and written ----------
      const bool two = n > 1;
      float* mine = xch + x * 128 + r;
      const float* other = xch + (x ^ 1) * 128 + r;
      *mine = m_ref;
      wide_barrier(1, 256);
      const float m_o = *other;
      wide_barrier(1, 256);
      *mine = l;
      wide_barrier(1, 256);
      const float l_o = *other;
      const float M = fmaxf(m_ref, m_o);
      const float Mu = M == -INFINITY ? 0.f : M;
      const float fm = ex2(m_ref - Mu), fo = ex2(m_o - Mu);
      const float f0 = x ? fo : fm, f1 = x ? fm : fo;
      wide_wait(p, bar(C::B_ODONE), (done[0] - 1) & 1);  // every stream's last P*V
      if (two) wide_wait(p, bar(C::B_ODONE + 1), (done[1] - 1) & 1);
      tc_fence_after();
      const long long row0 = shared_wide_row(p, it.first, it.rows, it.kvh, it.rt, blockIdx.x);
      if (busy) {
        // this thread's stream names its half of the columns
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          const int col = (D / 2) * x + 32 * c;
          uint32_t a[32], b[32];
          tmem_ld32(trow + W_OCOL + col, a);
          if (two) tmem_ld32(trow + W_OCOL + 128 + col, b);
          tmem_wait_ld();
          uint4 ov[8];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float v = __uint_as_float(a[i]) * f0;
            if (two) v += __uint_as_float(b[i]) * f1;
            (&ov[i >> 2].x)[i & 3] = __float_as_uint(v);
          }
          // coalesced: the eight lanes of a group exchange their pieces, store k writes row 8 g + k
          transpose8_u4(ov, lane & 7);
          const int rb = (warp & 3) * 32 + (lane & ~7);
#pragma unroll
          for (int k = 0; k < 8; ++k)
            if (rb + k < live) *reinterpret_cast<uint4*>(p.part_o + (row0 + rb + k) * D + col + 4 * (lane & 7)) = ov[k];
        }
        if (x == 0 && r < live)
          *reinterpret_cast<float2*>(p.part_ml + (row0 + r) * 2) = make_float2(M, l * fm + (two ? l_o * fo : 0.f));
      }
      // both streams' sums are read by all before the next piece's products overwrite them
      tc_fence_before();
      wide_barrier(1, 256);
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == W_MMA) {
    __syncwarp();
    tc_fence_after();
    tmem_dealloc(tmem, W_TMEM);
  }
}

template <int D, bool MMA_BF16, bool QBF16, bool I8>
cudaError_t launch_wide(const SharedParams& p, const KvMaps& maps, cudaStream_t stream) {
  using C = WideCfg<D, I8>;
  auto kern = prefix_wide_kernel<D, MMA_BF16, QBF16, I8>;
  cudaError_t e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM);
  if (e != cudaSuccess) return e;
  return launch_pdl(kern, dim3(p.wide_ctas), dim3(C::THREADS), C::SMEM, stream, p, maps);
}

template <int D>
cudaError_t launch_wide_d(const SharedParams& p, const KvMaps& m, int kv, cudaStream_t s) {
  if (kv == KV_I8) return p.q_bf16 ? launch_wide<D, false, true, true>(p, m, s) : launch_wide<D, false, false, true>(p, m, s);
  if (kv == KV_BF16) return p.q_bf16 ? launch_wide<D, true, true, false>(p, m, s) : launch_wide<D, true, false, false>(p, m, s);
  return p.q_bf16 ? launch_wide<D, false, true, false>(p, m, s) : launch_wide<D, false, false, false>(p, m, s);
}

}  // namespace

bool prefix_wide_supported(int kv_kind, int D, int BS) {
  return (kv_kind == KV_F16 || kv_kind == KV_BF16 || kv_kind == KV_I8) && (D == 64 || D == 128) && BS >= 8;
}

cudaError_t launch_prefix_wide(const SharedParams& p_in, const KvMaps& maps, int kv_kind, int D, cudaStream_t stream) {
  static std::atomic<unsigned int> generation{0};
  SharedParams p = p_in;
  do {
    p.abort_gen = ++generation;
  } while (p.abort_gen == 0);
  return D == 64 ? launch_wide_d<64>(p, maps, kv_kind, stream) : launch_wide_d<128>(p, maps, kv_kind, stream);
}

}  // namespace pa
