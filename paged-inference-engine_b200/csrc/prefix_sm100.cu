// Attention of many query rows over a shared prefix on the 5th-generation
// tensor cores (tcgen05 + TMEM).
//
// A group's rows over one kv head (sequences x query rows x group heads) are cut into tiles of
// 128, its shared keys into tiles of 128.  The CTAs of a persistent grid form teams that walk the list
// of (group, kv head, key tiles), an equal run of it each; inside a team, every CTA has two row tiles of
// the group (WideShape).  So the row tiles of a group pass over the same keys at about the same time, and
// K and V come from HBM once: with the row tiles one after the other along the list, 128 sequences of 4 heads over 65536 bf16 keys
// read their 268 MB four times (231 us).  What a CTA makes of its part of a run within one (group, kv
// head) is a piece: its rows' statistics and unnormalised sums go to the workspace, where
// prefix_merge_kernel joins them (csrc/prefix_plan.cu).  Every row sees every shared key (the plan
// sees to it), so the only mask is the end of the last tile.
//
// A CTA runs two streams, each with its own logits, maximum and sum in TMEM (S0 S1 O0 O1): while one
// turns its logits into probabilities, the tensor core works for the other.  The streams are its two
// row tiles, which share each K/V tile; or, where there is one row tile, its even and odd key tiles, whose
// results are joined in registers at the end of the piece, so that few rows do not leave half of the CTA idle.
//
//   warps 0-7    softmax: a thread per row (TMEM lane) and stream (w >> 2); they also load and convert Q
//   warp 8       producer: K and V boxes gathered through the block table by TMA
//   warp 9       MMA issuer
//   warps 10-13  INT8 pools: raw tiles -> fp16 operand tiles, q * scale in fp32 rounded once, as
//                csrc/kv_dequant.cu does for prompts; the raw bytes cross HBM once and the
//                fp16 tile never leaves the SM
//
// Roundings to 16 bits, as in the library's other attention kernels: the operands of a product have one type, so the
// probabilities take the pool's (bf16: off by up to 2^-8, which leaves 1.7e-3 in the output over 65536 keys; fp16 and INT8 pools:
// fp16, 2^-11), Q too where it differs, and INT8 keys and values fp16 once they carry their scales. A second
// product with what the rounding left would halve the rate of a kernel that the products bound. Logits, maxima, sums (of the
// unrounded probabilities) and outputs stay in fp32 until the join.  INT8 keys may lie beyond fp16's range, and values up to
// 127 * 65536 (RANGE); it is the range of bf16 queries over fp16 and INT8 pools, as of the outputs.
//
// 16-bit pools with many rows: 128 keys of 128 rows take 1995 cycles, about 1000 of the products and 1000 of the exponentials, one
// after the other for most of it (128 sequences of 4 heads over 65536 bf16 keys: tensor pipe 49 %, the exponentials'
// unit 50 %, DRAM 24 %).  With few rows (64 sequences of 4 heads over 8192 fp16 keys: 20 %, 21 %, 14 %) by latency: the first tiles, and pieces
// of 256 rows that every CTA writes.
// INT8 pools: by the conversion of the tiles, 1100 cycles each (tensor pipe 21 %, issue slots 40 %); eight warps for
// it left 96 registers a thread and gained nothing.
#include <type_traits>

#include "bounded_wait.cuh"
#include "pa_common.cuh"

namespace pa {
namespace {

constexpr int W_HALF = 128 * 128;  // 64 columns (128 bytes) of a 128-row tile
constexpr uint32_t W_TMEM = 512;
constexpr uint32_t W_OCOL = 256;
constexpr float W_THRESHOLD = 8.0f;  // growth of the maximum (log2) that rescales
constexpr int W_SOFTMAX = 8;         // warps
constexpr int W_PRODUCER = 8, W_MMA = 9, W_CONVERT = 10;
constexpr int W_CONVERTERS = 4;      // warps, INT8

template <int D, bool I8>
struct WideCfg {
  static constexpr int TILE = (D / 64) * W_HALF;   // fp16 / bf16 operand tile of 128 rows
  static constexpr int RAW = 128 * D;              // int8 tile
  static constexpr int KST = D == 128 ? (I8 ? 2 : 3) : (I8 ? 3 : 5);  // K stages
  static constexpr int VST = D == 128 ? 2 : (I8 ? 3 : 5);               // V stages
  static constexpr int RST = I8 ? (D == 128 ? 2 : 8) : 0;  // raw tiles in flight, K and V alternating (4 and one V stage: 120 us where this took 115)
  static constexpr int K0 = 2 * TILE;
  static constexpr int V0 = K0 + KST * TILE;
  static constexpr int R0 = V0 + VST * TILE;
  static constexpr int BAR = R0 + RST * RAW;
  static constexpr int B_QREADY = 0, B_QEMPTY = 1, B_SFULL = 2, B_PFULL = 4, B_ODONE = 6, B_SLOT = 8, B_PLACE = 9,
                       B_LAST = 10, B_KFULL = 11, B_KEMPTY = B_KFULL + KST, B_VFULL = B_KEMPTY + KST, B_VEMPTY = B_VFULL + VST,
                       B_RFULL = B_VEMPTY + VST, B_REMPTY = B_RFULL + RST, B_END = B_REMPTY + RST;
  static constexpr int BARS = D == 128 ? 256 : 512;  // bytes of the barriers, and what a wait that gives up writes (16 bytes)
  static constexpr int RANGE = BAR + BARS;  // INT8: powers of two that keys and values were divided by
  // Tiles whose powers are held.  They are written with K of a tile and read with its logits.  Before K of tile t comes V of
  // t - 2, which waits until the stage that tile t - 2 - VST had is free: its products, and so its probabilities, are done.
  static constexpr int RANGES = I8 ? 8 : 0;
  static_assert(!I8 || RANGES >= VST + 2, "a tile's powers are read before they are written again");
  static constexpr int XCH = RANGE + RANGES * W_CONVERTERS * 8;
  static constexpr int SMEM = XCH + 1024 + 1024;  // exchange of the two streams, alignment
  static constexpr int THREADS = 32 * (I8 ? W_CONVERT + W_CONVERTERS : W_CONVERT);
  static_assert(B_END * 8 + 16 <= BARS && BAR % BARS == 0 && SMEM <= 227 * 1024, "shared memory per CTA");
};

// A scale's bits, where there is one: loaded without a branch or a conversion, so that nothing
// waits for it before its use (4 groups of 32 over 16384 keys: 116 us with a wait in every unit, 115 without).
__device__ __forceinline__ uint32_t scale_bits(const void* base, long long at, bool is, bool f32) {
  uint32_t v;
  const char* a = static_cast<const char*>(base) + (at << (f32 ? 2 : 1));
  asm volatile(
      "{\n.reg .pred p, q;\nsetp.ne.s32 p, %2, 0;\nsetp.ne.s32 q, %3, 0;\nmov.b32 %0, 0;\n"
      "@p ld.global.nc.u32 %0, [%1];\n@q ld.global.nc.u16 %0, [%1];\n}\n"
      : "=&r"(v)
      : "l"(a), "r"(static_cast<int>(is && f32)), "r"(static_cast<int>(is && !f32)));
  return v;
}

// A wait that fails gave up, by itself or since another wait of this launch did (the plan clears their word in the call's workspace
// on every run, a captured call's replays too).  A CTA then walks to its end without its results being good (the status
// word says so); the producer stops, and it and the issuer of the products wait for theirs before the CTA ends.
// The addresses of their word and of the status word lie at the end of the barriers' block, which a barrier's address gives: so
// a wait has no other arguments (with the parameters for one, 128 sequences of 4 heads over 65536 keys took 192 us, so 187).
template <int D>
struct WideGiveUp {
  uint32_t bar;
  __device__ __forceinline__ uint64_t address(int i) const {
    constexpr uint32_t BARS = WideCfg<D, false>::BARS;
    uint64_t a;
    asm volatile("ld.shared.b64 %0, [%1];\n" : "=l"(a) : "r"((bar & ~(BARS - 1)) + BARS - 16 + 8 * i));
    return a;
  }
  __device__ __forceinline__ bool marked() const { return *reinterpret_cast<volatile int*>(address(0)) != 0; }
  __device__ __forceinline__ void mark() const { atomicExch(reinterpret_cast<int*>(address(0)), 1); }
  __device__ __forceinline__ void report() const { set_status(reinterpret_cast<int*>(address(1)), ST_WAIT_TIMEOUT); }
};
template <int D>
__device__ __noinline__ bool wide_wait_slow(uint32_t bar, uint32_t parity) {
  return bounded_wait<1 << 20, 64>(bar, parity, WideGiveUp<D>{bar});
}
template <int D>
__device__ __forceinline__ bool wide_wait(uint32_t bar, uint32_t parity) {
  return mbar_try_wait(bar, parity) || wide_wait_slow<D>(bar, parity);
}
__device__ __noinline__ void wide_drain(uint32_t bar, uint32_t parity) {
  for (int i = 0; i < (1 << 20); ++i)
    if (mbar_try_wait(bar, parity)) return;
}
__device__ __forceinline__ void wide_barrier(int id, int n) { asm volatile("bar.sync %0, %1;\n" ::"r"(id), "r"(n) : "memory"); }

// The pieces of a CTA, walked alike by every role.
struct Pieces {
  int s, s1;          // steps of the team's run not walked yet
  int team, q, size;  // team, the CTA's place in it, CTAs of a team
  int run;
  int g, base;        // group and its first step
  int4 grp;           // shared keys, first sequence, sequences, leader
  WideShape sh;
  // the piece
  int seg, kvh, t, n;  // (pass, kv head), key tiles [t, t + n)
  int row0, live;      // first row of the CTA's row tiles in the group, rows of them
  bool two;            // two row tiles (else one, whose key tiles alternate between the streams)
  int part, lane;

  __device__ __forceinline__ Pieces(const SharedParams& p, const int4& head, int cta, int g0) {
    size = head.x;
    team = cta / size;
    q = cta - team * size;
    run = head.y;
    s = min(team * run, head.z);
    s1 = min(s + run, head.z);
    g = g0 - 1;
    base = -1;
    if (s < s1) {
      g = g0;
      group(p);
    }
  }
  __device__ __forceinline__ void group(const SharedParams& p) {
    grp = p.grp[g];
    base = p.step0[g];
    sh = WideShape(grp.x, grp.z, p.maxq * p.G, size);
  }
  __device__ __forceinline__ bool next(const SharedParams& p) {
    while (s < s1) {
      const int len = sh.steps();
      if (s - base >= sh.passes * p.Hkv * len) {  // a group with steps is still ahead
        do {
          ++g;
        } while (p.grp[g].x == 0);
        group(p);
        continue;
      }
      const int off = s - base;
      seg = off / len;
      const int a = off - seg * len, b = min(len, a + s1 - s);
      s += b - a;
      const int pass = seg / p.Hkv;
      kvh = seg - pass * p.Hkv;
      const int lanes = min(sh.lanes, sh.RP - pass * sh.lanes);  // the last pass may have fewer pairs
      part = q / sh.lanes;
      lane = q - part * sh.lanes;
      if (part >> sh.lparts || lane >= lanes) continue;
      if (a >= sh.steps()) continue;
      t = wide_tiles(sh, a, min(b, sh.steps()), part, n);
      if (n <= 0) continue;
      row0 = (pass * sh.lanes + lane) * 2 * kWideRows;
      live = min(2 * kWideRows, sh.rows - row0);
      two = live > kWideRows;
      return true;
    }
    return false;
  }
  __device__ __forceinline__ int units() const { return two ? 2 * n : n; }  // products of a row tile and a key tile
  __device__ __forceinline__ int tile(int u) const { return two ? u >> 1 : u; }
};

template <int D, bool MMA_BF16, bool QBF16, bool I8>
__global__ void __launch_bounds__(WideCfg<D, I8>::THREADS, 1)
    prefix_wide_kernel(const SharedParams p, const __grid_constant__ KvMaps maps) {
  using C = WideCfg<D, I8>;
  constexpr int KST = C::KST, VST = C::VST, TILE = C::TILE;
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const uint32_t raw = smem_u32(smem_raw);
  const uint32_t base = (raw + 1023u) & ~1023u;
  unsigned char* sm = smem_raw + (base - raw);
  auto bar = [&](int i) { return base + C::BAR + 8u * i; };
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (tid == 32) {
    mbar_init(bar(C::B_QREADY), 32 * W_SOFTMAX);
    mbar_init(bar(C::B_QEMPTY), 1);
    mbar_init(bar(C::B_LAST), 1);
    for (int x = 0; x < 2; ++x) {
      mbar_init(bar(C::B_SFULL + x), 1);
      mbar_init(bar(C::B_PFULL + x), 16 * W_SOFTMAX);
      mbar_init(bar(C::B_ODONE + x), 1);
    }
    for (int s = 0; s < KST; ++s) {
      mbar_init(bar(C::B_KFULL + s), I8 ? 32 * W_CONVERTERS : 1);
      mbar_init(bar(C::B_KEMPTY + s), 1);
    }
    for (int s = 0; s < VST; ++s) {
      mbar_init(bar(C::B_VFULL + s), I8 ? 32 * W_CONVERTERS : 1);
      mbar_init(bar(C::B_VEMPTY + s), 1);
    }
    for (int s = 0; s < C::RST; ++s) {
      mbar_init(bar(C::B_RFULL + s), 1);
      mbar_init(bar(C::B_REMPTY + s), 32 * W_CONVERTERS);
    }
    uint64_t* at = reinterpret_cast<uint64_t*>(sm + C::BAR + C::BARS - 16);
    at[0] = reinterpret_cast<uint64_t>(&p.head[0].w);
    at[1] = reinterpret_cast<uint64_t>(p.status);
    fence_mbar_init();
  }
  pdl_enter();
  const int4 head = p.head[0];
  const int team = static_cast<int>(blockIdx.x) / head.x;
  const int s_first = team * head.y;
  if (team >= p.wide_ctas / head.x || s_first >= head.z) return;  // no whole team, or no steps for it
  if (warp == 0) {
    // the group of step s_first: the last with step0[g] <= s_first, found 32 at a time
    int lo = 0, hi = p.groups;  // step0[lo] <= s_first < step0[hi]
    while (hi - lo > 1) {
      const int step = (hi - lo + 31) / 32;
      const int at = lo + lane * step;
      const unsigned le = __ballot_sync(0xffffffffu, at < hi && p.step0[min(at, hi)] <= s_first);
      const int last = 31 - __clz(le);  // lane 0 always holds
      lo += last * step;
      hi = min(hi, lo + step);
    }
    if (lane == 0) *reinterpret_cast<volatile int*>(sm + C::BAR + 8 * C::B_PLACE) = lo;
  }
  if (warp == W_MMA) {
    tmem_alloc(bar(C::B_SLOT), W_TMEM);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *reinterpret_cast<volatile uint32_t*>(sm + C::BAR + 8 * C::B_SLOT);
  Pieces it(p, head, blockIdx.x, *reinterpret_cast<volatile int*>(sm + C::BAR + 8 * C::B_PLACE));

  if (warp == W_PRODUCER) {
    // ------------------------------------------------------------ producer
    // Lane i owns box i of every tile; the block ids of a tile are fetched one tile ahead.
    const int boxs = p.BS < 16 ? p.BS : 16;
    const int nbox = kWideKeys / boxs;  // <= 16 (block_size >= 8)
    int issued[2] = {0, 0};  // K and V tiles (INT8: [0] raw tiles) so far
    bool going = true;       // false: a wait gave up
    while (going && it.next(p)) {
      const int* bt_row = p.bt + static_cast<long long>(it.grp.w) * p.bt_ss;
      auto fetch = [&](int j) {
        const int key = (it.t + j) * kWideKeys + lane * boxs;
        int blk = p.NB;  // out of range: TMA fills the box with zeros
        if (lane < nbox && key < it.grp.x) {
          const int x = bt_row[static_cast<long long>(key >> p.log2BS) * p.bt_sc];
          if (x >= 0 && x < p.NB) blk = x;
          else set_status(p.status, ST_BAD_BLOCK_ID);
        }
        return blk;
      };
      // The order of the loads is K0, K1 V0, K2 V1, ...: a key tile's K is wanted a product before its V, and a
      // V stage comes free late.
      auto load = [&](int v, int j, int blk) {
        if (!going) return;
        const int slot = blk < p.NB ? ((it.t + j) * kWideKeys + lane * boxs) & (p.BS - 1) : 0;
        uint32_t dst, full, empty;
        int turn;  // how often the stage was used
        if constexpr (I8) {
          const int s = issued[0] % C::RST;
          turn = issued[0] / C::RST;
          full = bar(C::B_RFULL + s);
          empty = bar(C::B_REMPTY + s);
          dst = base + C::R0 + s * C::RAW + lane * boxs * D;
        } else {
          const int st = v ? VST : KST, s = issued[v] % st;
          turn = issued[v] / st;
          full = bar((v ? C::B_VFULL : C::B_KFULL) + s);
          empty = bar((v ? C::B_VEMPTY : C::B_KEMPTY) + s);
          dst = base + (v ? C::V0 : C::K0) + s * TILE + lane * boxs * 128;
        }
        if (lane == 0) {
          // free again, and its last copies have arrived (known, unless a reader gave up)
          going = turn == 0 || (wide_wait<D>(empty, (turn - 1) & 1) && wide_wait<D>(full, (turn - 1) & 1));
          if (going) mbar_arrive_expect_tx(full, I8 ? C::RAW : TILE);
        }
        going = __shfl_sync(0xffffffffu, going, 0);
        if (!going) return;
        ++issued[I8 ? 0 : v];
        if (lane < nbox) {
          const CUtensorMap* m = v ? &maps.v : &maps.k;
          tma_load_4d(dst, m, full, 0, it.kvh, slot, blk);
          if constexpr (!I8 && D == 128) tma_load_4d(dst + W_HALF, m, full, 64, it.kvh, slot, blk);
        }
      };
      const int n = it.n;
      int b0 = fetch(0), b1 = n > 1 ? fetch(1) : p.NB;
      load(0, 0, b0);
      for (int j = 0; j < n; ++j) {
        const int b2 = j + 2 < n ? fetch(j + 2) : p.NB;
        if (j + 1 < n) load(0, j + 1, b1);
        load(1, j, b0);
        b0 = b1;
        b1 = b2;
      }
    }
    if (lane == 0) {  // no copy is in flight when the CTA ends
      const int k = issued[0], v = issued[1], kst = I8 ? C::RST : KST;
      for (int s = 0; s < kst && s < k; ++s) wide_drain(bar((I8 ? C::B_RFULL : C::B_KFULL) + s), ((k - 1 - s) / kst) & 1);
      for (int s = 0; s < VST && s < v; ++s) wide_drain(bar(C::B_VFULL + s), ((v - 1 - s) / VST) & 1);
    }
  } else if (warp == W_MMA) {
    // ------------------------------------------------------------ MMA issuer
    // The whole warp walks along, one elected lane issues.
    constexpr uint32_t IDESC_QK = instr_desc_f16(MMA_BF16, false, false, kWideRows, kWideKeys);
    constexpr uint32_t IDESC_PV = instr_desc_f16(MMA_BF16, false, true, kWideRows, D);
    int gt = 0, piece = 0;
    int px0 = 0, px1 = 0;  // probabilities taken of each stream
    for (; it.next(p); ++piece) {
      // unit u: stream u & 1; both streams of a pair of row tiles take the same key tile
      const int nu = it.units();
      const bool two = it.two;
      auto qk = [&](int u) {
        const int x = u & 1, tile = gt + it.tile(u), s = tile % KST;
        wide_wait<D>(bar(C::B_KFULL + s), (tile / KST) & 1);
        tc_fence_after();
        tc_elect_mma_ss<D / 16, W_HALF / 16, W_HALF / 16>(tmem + 128u * x, smem_desc(base + (two ? x * TILE : 0), 16, 1024),
                                                          smem_desc(base + C::K0 + s * TILE, 16, 1024), IDESC_QK);
        tc_elect_commit(bar(C::B_SFULL + x));
        if (!two || x) tc_elect_commit(bar(C::B_KEMPTY + s));
        if (u == nu - 1) tc_elect_commit(bar(C::B_QEMPTY));
      };
      wide_wait<D>(bar(C::B_QREADY), piece & 1);
      tc_fence_after();
      qk(0);
      if (nu > 1) qk(1);
      for (int u = 0; u < nu; ++u) {
        const int x = u & 1, tile = gt + it.tile(u), s = tile % VST;
        wide_wait<D>(bar(C::B_VFULL + s), (tile / VST) & 1);
        wide_wait<D>(bar(C::B_PFULL + x), (x ? px1 : px0) & 1);
        px0 += x ^ 1;
        px1 += x;
        tc_fence_after();
        tc_elect_mma_ts8(tmem + W_OCOL + 128u * x, tmem + 128u * x, smem_desc(base + C::V0 + s * TILE, W_HALF, 1024), IDESC_PV,
                         u >= 2 ? 1u : 0u);
        if (!two || x) tc_elect_commit(bar(C::B_VEMPTY + s));
        tc_elect_commit(bar(C::B_ODONE + x));
        if (u + 2 < nu) qk(u + 2);
      }
      gt += it.n;
    }
    // No product is in flight when the CTA gives its tensor memory back and ends.  (The softmax has waited for the last ones,
    // unless a wait of its gave up.)
    tc_elect_commit(bar(C::B_LAST));
    wide_drain(bar(C::B_LAST), 0);
  } else if (warp >= W_CONVERT) {
    // ------------------------------------------------------------ INT8 -> fp16 tiles
    if constexpr (I8) {
      // Warp c converts rows ROWS c .. ROWS c + ROWS - 1 of every tile; lane l holds the scales of row ROWS c + l % ROWS.  A lane takes 16
      // dims of a row at a time.  The eight lanes that a shared-memory access serves at once are four pieces of rows a
      // and a ^ 5: swizzled, those lie in different banks, in the raw tile (16 bytes a piece) as in the operand tile (twice
      // 16 bytes, two apart).
      constexpr int RPI = 32 / (D / 16);  // rows an iteration of a warp
      constexpr int UNROLL = 4;
      constexpr int ROWS = kWideKeys / W_CONVERTERS;  // of a tile, a warp
      const int r0 = ROWS * (warp - W_CONVERT), mine_at = r0 + (lane & (ROWS - 1));
      const int half = D == 128 ? (lane >> 3) & 1 : 0;
      const int ch = 4 * half + (lane & 3);                    // 16-byte piece of the raw row
      const int pair = D == 128 ? lane >> 4 : lane >> 3;       // row pairs 0 5, 1 4, 2 7, 3 6 of eight rows
      const int flip = (lane >> 2) & 1 ? 5 : 0;
      int gt = 0, gr = 0;
      while (it.next(p)) {
        const int* bt_row = p.bt + static_cast<long long>(it.grp.w) * p.bt_ss;
        const int n = it.n;
        auto block = [&](int j) {
          const int key = (it.t + j) * kWideKeys + mine_at;
          return j < n && key < it.grp.x ? bt_row[static_cast<long long>(key >> p.log2BS) * p.bt_sc] : -1;
        };
        auto scales = [&](int j, int blk, uint32_t& k, uint32_t& v) {  // as they are stored; 0: no block, or past the end
          const bool is = blk >= 0 && blk < p.NB;
          const int slot = ((it.t + j) * kWideKeys + mine_at) & (p.BS - 1);
          k = scale_bits(p.ks, is ? blk * p.ks_sblk + slot * p.ks_sslot + it.kvh * p.ks_shead : 0, is, p.scale_f32);
          v = scale_bits(p.vs, is ? blk * p.vs_sblk + slot * p.vs_sslot + it.kvh * p.vs_shead : 0, is, p.scale_f32);
        };
        auto as_float = [&](uint32_t bits) {
          return p.scale_f32 ? __uint_as_float(bits) : __half2float(__ushort_as_half(static_cast<unsigned short>(bits)));
        };
        // Keys and values that would leave fp16's range (127 times a scale above 512) are divided by a power of two, one for the
        // warp's rows of a tile, which the logits or probabilities are multiplied by in turn.
        auto power = [&](float mine) {
          const unsigned most = __reduce_max_sync(0xffffffffu, __float_as_uint(fabsf(mine)));
          return most > __float_as_uint(512.f) && most < 0x7f800000u ? __uint_as_float(((most >> 23) - 8u) << 23) : 1.f;
        };
        auto inverse = [&](float pow2) { return __uint_as_float((254u << 23) - __float_as_uint(pow2)); };
        // later_bits: the scales of the same tile's V, at its K
        auto convert = [&](int v, int j, uint32_t mine_bits, uint32_t later_bits) {
          const int st = v ? VST : KST, g = gt + j, s = g % st, rs = gr % C::RST;
          const unsigned char* src = sm + C::R0 + rs * C::RAW;
          unsigned char* dst = sm + (v ? C::V0 : C::K0) + s * TILE;
          wide_wait<D>(bar(C::B_RFULL + rs), (gr / C::RST) & 1);
          if (g >= st) wide_wait<D>(bar((v ? C::B_VEMPTY : C::B_KEMPTY) + s), (g / st - 1) & 1);
          ++gr;
          float mine = as_float(mine_bits), range = 1.f, later = 1.f;
          const float next = v == 0 ? as_float(later_bits) : 0.f;
          if (__any_sync(0xffffffffu, fabsf(mine) > 512.f || fabsf(next) > 512.f)) {
            range = power(mine);
            later = power(next);
            mine *= inverse(range);
          }
          if (v == 0 && lane == 0) {
            float* at = reinterpret_cast<float*>(sm + C::RANGE) + (g % C::RANGES) * 2 * W_CONVERTERS + warp - W_CONVERT;
            at[0] = range, at[W_CONVERTERS] = later;
          }
          auto rows = [&](auto fp32_scale) {
#pragma unroll UNROLL
            for (int k = 0; k < ROWS / RPI; ++k) {
              const int lr = (D == 128 ? 8 * (k >> 1) + 2 * (k & 1) : 8 * k) + pair;  // row within the warp's
              const int row = lr ^ flip;
              const int r = r0 + row;
              const float f = __shfl_sync(0xffffffffu, mine, row);
              const int at = D == 128 ? r * 128 + ((ch ^ (r & 7)) << 4) : r * 64 + ((ch ^ ((r >> 1) & 3)) << 4);
              const uint4 w = *reinterpret_cast<const uint4*>(src + at);
              const uint32_t x[4] = {w.x, w.y, w.z, w.w};
              uint32_t o[8];
              if constexpr (decltype(fp32_scale)::value) {
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  uint32_t a, b;
                  i8x4_to_f16x4(x[q], a, b);
                  const float2 fa = __half22float2(*reinterpret_cast<__half2*>(&a));
                  const float2 fb = __half22float2(*reinterpret_cast<__half2*>(&b));
                  o[2 * q] = pack_f16(fa.x * f, fa.y * f);
                  o[2 * q + 1] = pack_f16(fb.x * f, fb.y * f);
                }
              } else {
                // an fp16 scale times a code has at most 18 significant bits: one rounding either way
                const __half2 h = __float2half2_rn(f);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                  i8x4_to_f16x4(x[q], o[2 * q], o[2 * q + 1]);
                  __half2* y = reinterpret_cast<__half2*>(o + 2 * q);
                  y[0] = __hmul2(y[0], h);
                  y[1] = __hmul2(y[1], h);
                }
              }
              unsigned char* d = dst + half * W_HALF + r * 128;
              const int p0 = 2 * (ch & 3);
              *reinterpret_cast<uint4*>(d + ((p0 ^ (r & 7)) << 4)) = make_uint4(o[0], o[1], o[2], o[3]);
              *reinterpret_cast<uint4*>(d + (((p0 + 1) ^ (r & 7)) << 4)) = make_uint4(o[4], o[5], o[6], o[7]);
            }
          };
          if (p.scale_f32) rows(std::true_type{});
          else rows(std::false_type{});
          fence_proxy_async_smem();
          mbar_arrive(bar((v ? C::B_VFULL : C::B_KFULL) + s));
          mbar_arrive(bar(C::B_REMPTY + rs));
        };
        // In the order of the loads: K of a tile, V of the one before.  The scales are fetched a tile ahead, the block ids
        // two.
        uint32_t k1, v1, k2, v2, v0 = 0;
        scales(0, block(0), k1, v1);
        int blk2 = block(1);
#pragma unroll 1
        for (int j = -1; j < n; ++j) {
          scales(j + 2, blk2, k2, v2);
          blk2 = block(j + 3);
#pragma unroll 1
          for (int v = 0; v < 2; ++v)
            if (j + 1 - v >= 0 && j + 1 - v < n) convert(v, j + 1 - v, v ? v0 : k1, v1);
          v0 = v1, k1 = k2, v1 = v2;
        }
        gt += n;
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
    int gt = 0;            // key tiles before the piece
    int done[2] = {0, 0};  // units of each stream
    int q_done = 0;
    for (; it.next(p);) {
      const int nu = it.units();
      const bool two = it.two;
      const int mine0 = two ? x * kWideRows : 0;                  // first row of this stream's tile
      const int live = min(kWideRows, it.live - mine0);           // rows of it
      const bool busy = 32 * (warp & 3) < live;                   // this warp holds one
      // ---- Q: half a row a thread, converted to the operand type, swizzled
      if (done[0] > 0) wide_wait<D>(bar(C::B_QEMPTY), q_done & 1), ++q_done;
#pragma unroll 1
      for (int y = 0; y < (two ? 2 : 1); ++y) {
        const int row = tid >> 1, c0 = (tid & 1) * (D / 16);
        const int R = it.row0 + y * kWideRows + row;
        uint4 w[D / 16];
#pragma unroll
        for (int c = 0; c < D / 16; ++c) w[c] = make_uint4(0, 0, 0, 0);
        if (y * kWideRows + row < it.live) {
          const int m = R / per, rem = R - m * per;
          const int qi = rem / p.G, b = it.grp.y + m;
          if (qi < seq_rows(p, b)) {
            const uint4* src = reinterpret_cast<const uint4*>(
                static_cast<const unsigned short*>(p.q) + q_seq_base(p, b) + (it.kvh * p.G + rem - qi * p.G) * p.q_sh +
                static_cast<long long>(qi) * p.q_sm) + c0;
#pragma unroll
            for (int c = 0; c < D / 16; ++c) w[c] = src[c];
          }
        }
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          w[c].x = cvt_pair<QBF16, MMA_BF16>(w[c].x);
          w[c].y = cvt_pair<QBF16, MMA_BF16>(w[c].y);
          w[c].z = cvt_pair<QBF16, MMA_BF16>(w[c].z);
          w[c].w = cvt_pair<QBF16, MMA_BF16>(w[c].w);
          const int k = c0 + c;
          *reinterpret_cast<uint4*>(sm + y * TILE + (k >> 3) * W_HALF + row * 128 + (((k & 7) ^ (row & 7)) << 4)) = w[c];
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(bar(C::B_QREADY));

      float m_ref = -INFINITY, l = 0.f;
      for (int u = x; u < nu; u += 2) {
        wide_wait<D>(bar(C::B_SFULL + x), (done[x] + (u >> 1)) & 1);
        tc_fence_after();
        if (busy) {
          const int left = it.grp.x - (it.t + it.tile(u)) * kWideKeys;  // keys of this tile, maybe more than 128
          // first look: the row's maximum.  The logits are read again below: 128 of them do not fit the registers
          // beside the rest, and a second read of TMEM is cheap
          float mx4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
          // INT8: the powers of the keys [32 c, 32 c + 32), then of the values
          static_assert(!I8 || kWideKeys / W_CONVERTERS == 32, "a converting warp's keys are those of one step below");
          const float* range = reinterpret_cast<const float*>(sm + C::RANGE) + (I8 ? (gt + it.tile(u)) % C::RANGES * 2 * W_CONVERTERS : 0);
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
            if constexpr (I8) {
              float a[2] = {-INFINITY, -INFINITY}, b[2] = {-INFINITY, -INFINITY};
#pragma unroll
              for (int i = 0; i < 32; i += 2) {
                const int k = (i >> 1) & 1;
                a[k] = fmax3f(a[k], __uint_as_float(r0[i]), __uint_as_float(r0[i + 1]));
                b[k] = fmax3f(b[k], __uint_as_float(r1[i]), __uint_as_float(r1[i + 1]));
              }
              mx4[2 * c] = fmaxf(a[0], a[1]) * range[2 * c];
              mx4[2 * c + 1] = fmaxf(b[0], b[1]) * range[2 * c + 1];
            } else {
#pragma unroll
              for (int i = 0; i < 32; ++i) mx4[i & 3] = fmax3f(mx4[i & 3], __uint_as_float(r0[i]), __uint_as_float(r1[i]));
            }
          }
          const float mx = fmaxf(fmaxf(mx4[0], mx4[1]), fmaxf(mx4[2], mx4[3])) * p.scale_log2;
          float alpha = 1.f;
          bool resc = false;
          if (mx > m_ref + W_THRESHOLD) {  // also the first finite maximum
            alpha = ex2(m_ref - mx);
            resc = u >= 2;  // O holds this stream's earlier tiles
            m_ref = mx;
          }
          const float neg_m = m_ref == -INFINITY ? 0.f : -m_ref;
          uint64_t sum[2] = {f2_pack(0.f, 0.f), f2_pack(0.f, 0.f)};
          // P of keys [32 c, 32 c + 32) takes TMEM columns [16 c, 16 c + 16): behind the logits still to be read
          uint32_t rr[2][32];
          tmem_ld32(scol, rr[0]);
#pragma unroll
          for (int c = 0; c < 4; ++c) {
            tmem_wait_ld();
            if (c < 3) tmem_ld32(scol + 32 * (c + 1), rr[(c + 1) & 1]);
            const uint32_t* s = rr[c & 1];
            const float c2 = I8 ? p.scale_log2 * range[c] : p.scale_log2;
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
            if constexpr (I8) {
              const float of_v = range[W_CONVERTERS + c];
              if (of_v != 1.f) {  // the warp as one; exact, but for numbers below fp16's normal range
                const __half2 h = __float2half2_rn(of_v);
#pragma unroll
                for (int i = 0; i < 16; ++i) reinterpret_cast<__half2*>(pk)[i] = __hmul2(reinterpret_cast<__half2*>(pk)[i], h);
              }
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
      done[0] += (nu + 1) / 2;
      done[1] += nu / 2;
      gt += it.n;
      // ---- end of the piece: its rows go to the workspace ---------------------------
      const long long prow = shared_wide_row(p, it.sh, it.grp.y, it.seg, it.team, it.size, it.part, it.lane) + mine0;
      const int rb = (warp & 3) * 32 + (lane & ~7);
      // coalesced: the eight lanes of a group exchange their pieces, store k writes row 8 g + k
      auto store = [&](uint4 (&ov)[8], int col) {
        transpose8_u4(ov, lane & 7);
#pragma unroll
        for (int k = 0; k < 8; ++k)
          if (rb + k < live) *reinterpret_cast<uint4*>(p.part_o + (prow + rb + k) * D + col + 4 * (lane & 7)) = ov[k];
      };
      if (two) {
        wide_wait<D>(bar(C::B_ODONE + x), (done[x] - 1) & 1);  // the stream's last P*V
        tc_fence_after();
        if (busy) {
#pragma unroll 1
          for (int c = 0; c < D / 32; ++c) {
            uint32_t a[32];
            tmem_ld32(ocol + 32 * c, a);
            tmem_wait_ld();
            uint4 ov[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) ov[i] = make_uint4(a[4 * i], a[4 * i + 1], a[4 * i + 2], a[4 * i + 3]);
            store(ov, 32 * c);
          }
          if (r < live) *reinterpret_cast<float2*>(p.part_ml + (prow + r) * 2) = make_float2(m_ref, l);
        }
        tc_fence_before();
        continue;
      }
      // one row tile: the two streams' results joined first
      const bool both = nu > 1;
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
      // every stream's last P*V; past the exchange both have seen the S of their last unit, so that neither
      // barrier is more than one phase behind
      wide_wait<D>(bar(C::B_ODONE), (done[0] - 1) & 1);
      if (both) wide_wait<D>(bar(C::B_ODONE + 1), (done[1] - 1) & 1);
      tc_fence_after();
      if (busy) {
        // this thread's stream names its half of the columns
#pragma unroll 1
        for (int c = 0; c < D / 64; ++c) {
          const int col = (D / 2) * x + 32 * c;
          uint32_t a[32], b[32];
          tmem_ld32(trow + W_OCOL + col, a);
          if (both) tmem_ld32(trow + W_OCOL + 128 + col, b);
          tmem_wait_ld();
          uint4 ov[8];
#pragma unroll
          for (int i = 0; i < 32; ++i) {
            float v = __uint_as_float(a[i]) * f0;
            if (both) v += __uint_as_float(b[i]) * f1;
            (&ov[i >> 2].x)[i & 3] = __float_as_uint(v);
          }
          store(ov, col);
        }
        if (x == 0 && r < live)
          *reinterpret_cast<float2*>(p.part_ml + (prow + r) * 2) = make_float2(M, l * fm + (both ? l_o * fo : 0.f));
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

cudaError_t launch_prefix_wide(const SharedParams& p, const KvMaps& maps, int kv_kind, int D, cudaStream_t stream) {
  return D == 64 ? launch_wide_d<64>(p, maps, kv_kind, stream) : launch_wide_d<128>(p, maps, kv_kind, stream);
}

}  // namespace pa
