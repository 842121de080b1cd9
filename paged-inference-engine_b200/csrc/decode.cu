// Launches of the split-K decode kernel (decode_kernel.cuh), its merge kernel,
// and the cross-GPU barrier of a peer output exchange.
#include "decode_kernel.cuh"

namespace pa {
namespace {

// Combine the split-K partials of every segment that straddles warp ranges.
// grid (Hkv, B), 128 threads.
template <int D>
__global__ void __launch_bounds__(128) pa_decode_merge_kernel(const AttnParams p) {
  pdl_enter();
  const int kvh = blockIdx.x;
  const int b = blockIdx.y;
  const int qlen = seq_qlen(p, b);
  if (qlen <= 0) return;
  const int ncols = min(qlen * p.G, NC_MAX);
  const int nt_b = p.tstart[b + 1] - p.tstart[b];
  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  if (nt_b == 0) {
    // no visible keys: O = 0, L = -inf
    for (int col = warp; col < ncols; col += 4) {
      const int qi = col / p.G, hq = col - (col / p.G) * p.G;
      const long long orow = o_seq_base(p, b) + (kvh * p.G + hq) * p.o_sh + static_cast<long long>(qi) * p.o_sm;
      for (int d = lane; d < D; d += 32) store_o(p, orow + d, __float2half_rn(0.f));
      if (lane == 0 && p.lse)
        static_cast<__half*>(p.lse)[l_seq_base(p, b) + (kvh * p.G + hq) * p.l_sh + static_cast<long long>(qi) * p.l_sm] =
            __float2half_rn(-INFINITY);
    }
    peer_store_fence(p);
    return;
  }
  const int total = p.tstart[p.B] * p.Hkv;
  const int W = p.num_warps_total;
  const int chunk = (total + W - 1) / W;
  const int S0 = p.tstart[b] * p.Hkv + kvh * nt_b;
  const int S1 = S0 + nt_b;
  const int w0 = S0 / chunk;
  const int w1 = (S1 - 1) / chunk;
  if (w0 == w1) return;  // written directly by the split kernel
  // slot of warp w's partial for this segment: its second slot when the segment starts inside w's range
  auto slot_of = [&](int w) { return (w == w0 && w0 * chunk < S0) ? 2 * w + 1 : 2 * w; };
  for (int col = warp; col < ncols; col += 4) {
    const int qi = col / p.G, hq = col - (col / p.G) * p.G;
    // lane i reads partial w0 + i (32 at a time): the maxima and the sums are
    // warp reductions instead of a chain of dependent L2 reads
    float M = -INFINITY;
    for (int w = w0 + lane; w <= w1; w += 32)
      M = fmaxf(M, p.part_ml[(static_cast<long long>(slot_of(w)) * NC_MAX + col) * 2]);
    M = warp_max_xor(M, 1);
    const float Mu = (M == -INFINITY) ? 0.f : M;
    float l = 0.f;
    float o[D / 32];
#pragma unroll
    for (int k = 0; k < D / 32; ++k) o[k] = 0.f;
    for (int base = w0; base <= w1; base += 32) {
      float f = 0.f;
      if (base + lane <= w1) {
        const float* pm = p.part_ml + (static_cast<long long>(slot_of(base + lane)) * NC_MAX + col) * 2;
        f = ex2(pm[0] - Mu);
        l += pm[1] * f;
      }
      const int n = min(32, w1 - base + 1);
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const float fj = __shfl_sync(0xffffffffu, f, j);
        const float* po = p.part_o + (static_cast<long long>(slot_of(base + j)) * NC_MAX + col) * D;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) o[k] += po[lane + 32 * k] * fj;
      }
    }
    l = warp_sum_xor(l, 1);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const long long orow = o_seq_base(p, b) + (kvh * p.G + hq) * p.o_sh + static_cast<long long>(qi) * p.o_sm;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) store_o(p, orow + lane + 32 * k, __float2half_rn(o[k] * inv));
    if (lane == 0 && p.lse) {
      const float L = l > 0.f ? (M + lg2(l)) * 0.6931471805599453f : -INFINITY;
      static_cast<__half*>(p.lse)[l_seq_base(p, b) + (kvh * p.G + hq) * p.l_sh + static_cast<long long>(qi) * p.l_sm] =
          __float2half_rn(L);
    }
  }
  peer_store_fence(p);
}

template <int D, int KVT, int QT, int NT, bool TMA>
struct DecodeInst {
  using Lay = DecLayout<D, KVT, NT>;
  static cudaError_t allow() {  // launches' sizes go by B
    static std::atomic<unsigned long long> done{0};
    return allow_smem(pa_decode_kernel<D, KVT, QT, NT, TMA>, SMEM_LIMIT, done);
  }
  static int plan(int B, DecodeLaunch* out) {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return -1;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -1;
    const int ts_bytes = ((B + 1) * 4 + 127) & ~127;
    const int fixed = ts_bytes + 1024;  // scan + alignment slack
    int nw = (SMEM_LIMIT - fixed) / Lay::WARPB;
    if (nw > max_warps<NT>()) nw = max_warps<NT>();
    if (nw < 1) return -1;
    out->warps_per_cta = nw;
    out->smem = static_cast<size_t>(fixed + nw * Lay::WARPB);
    auto kern = pa_decode_kernel<D, KVT, QT, NT, TMA>;
    if (allow() != cudaSuccess) return -1;
    int per_sm = 0;
    cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, nw * 32, out->smem);
    if (per_sm < 1) per_sm = 1;
    out->ctas = sms * per_sm;
    return 0;
  }
  static cudaError_t launch(const AttnParams& p, const KvMaps& maps, const DecodeLaunch& pl, int phase,
                            cudaStream_t stream) {
    cudaError_t e;
    if (phase != DECODE_MERGE) {
      auto kern = pa_decode_kernel<D, KVT, QT, NT, TMA>;
      e = allow();
      if (e != cudaSuccess) return e;
      e = launch_pdl(kern, dim3(pl.ctas), dim3(pl.warps_per_cta * 32), pl.smem, stream, p, maps);
      if (e != cudaSuccess) return e;
      e = cudaGetLastError();
      if (e != cudaSuccess) return e;
      if (phase == DECODE_SPLIT) return cudaSuccess;
    }
    e = launch_pdl(pa_decode_merge_kernel<D>, dim3(p.Hkv, p.B), dim3(128), 0, stream, p);
    if (e != cudaSuccess) return e;
    return cudaGetLastError();
  }
};

template <int D, int KVT, int QT>
struct Sel {
  static int plan(int nt, int B, bool tma, DecodeLaunch* o) {
    if (nt == 1) return tma ? DecodeInst<D, KVT, QT, 1, true>::plan(B, o) : DecodeInst<D, KVT, QT, 1, false>::plan(B, o);
    return tma ? DecodeInst<D, KVT, QT, 2, true>::plan(B, o) : DecodeInst<D, KVT, QT, 2, false>::plan(B, o);
  }
  static cudaError_t launch(const AttnParams& p, const KvMaps& m, int nt, bool tma, const DecodeLaunch& pl, int ph,
                            cudaStream_t s) {
    if (nt == 1)
      return tma ? DecodeInst<D, KVT, QT, 1, true>::launch(p, m, pl, ph, s)
                 : DecodeInst<D, KVT, QT, 1, false>::launch(p, m, pl, ph, s);
    return tma ? DecodeInst<D, KVT, QT, 2, true>::launch(p, m, pl, ph, s)
               : DecodeInst<D, KVT, QT, 2, false>::launch(p, m, pl, ph, s);
  }
};

template <int D>
int plan_kv(int kv, int qbf, int nt, int B, bool tma, DecodeLaunch* o) {
  if (kv == KV_F16) return qbf ? Sel<D, KV_F16, Q_BF16>::plan(nt, B, tma, o) : Sel<D, KV_F16, Q_F16>::plan(nt, B, tma, o);
  if (kv == KV_BF16) return qbf ? Sel<D, KV_BF16, Q_BF16>::plan(nt, B, tma, o) : Sel<D, KV_BF16, Q_F16>::plan(nt, B, tma, o);
  return qbf ? Sel<D, KV_I8, Q_BF16>::plan(nt, B, tma, o) : Sel<D, KV_I8, Q_F16>::plan(nt, B, tma, o);
}
template <int D>
cudaError_t launch_kv(const AttnParams& p, const KvMaps& m, int kv, int qbf, int nt, bool tma, const DecodeLaunch& pl,
                      int ph, cudaStream_t s) {
  if (ph == DECODE_MERGE)  // the merge kernel depends on head_dim only
    return Sel<D, KV_F16, Q_F16>::launch(p, m, nt, tma, pl, ph, s);
  if (kv == KV_F16)
    return qbf ? Sel<D, KV_F16, Q_BF16>::launch(p, m, nt, tma, pl, ph, s)
               : Sel<D, KV_F16, Q_F16>::launch(p, m, nt, tma, pl, ph, s);
  if (kv == KV_BF16)
    return qbf ? Sel<D, KV_BF16, Q_BF16>::launch(p, m, nt, tma, pl, ph, s)
               : Sel<D, KV_BF16, Q_F16>::launch(p, m, nt, tma, pl, ph, s);
  return qbf ? Sel<D, KV_I8, Q_BF16>::launch(p, m, nt, tma, pl, ph, s)
             : Sel<D, KV_I8, Q_F16>::launch(p, m, nt, tma, pl, ph, s);
}

}  // namespace

int decode_plan(int kv_kind, int q_bf16, int D, int nt, int B, int use_tma, DecodeLaunch* out) {
  if (D == 64) return plan_kv<64>(kv_kind, q_bf16, nt, B, use_tma != 0, out);
  if (D == 128) return plan_kv<128>(kv_kind, q_bf16, nt, B, use_tma != 0, out);
  return -1;
}

namespace {
// One CTA: thread t posts `epoch` into slot `rank` of peer t's flags, then
// waits for slot t of this GPU's flags to reach `epoch` (system-scope
// release / acquire; each wait gives up after ~0.4 s with a status bit).
// A peer can pass this barrier as soon as this GPU has posted, run its next
// step and post epoch + 1 before this GPU has read the slot, so any value at
// or past `epoch` ends the wait (a peer is never more than one epoch ahead).
__global__ void __launch_bounds__(32) pa_peer_barrier_kernel(int* local_flags, const PeerFlags peers, int n,
                                                              int rank, int epoch, int* status) {
  pdl_enter();
  const int t = threadIdx.x;
  if (t < n) {
    asm volatile("fence.acq_rel.sys;\n" ::: "memory");
    asm volatile("st.release.sys.global.b32 [%0], %1;\n" ::"l"(peers.flag[t] + rank), "r"(epoch) : "memory");
  }
  __syncwarp();
  if (t < n) {
    bool ok = false;
    for (int i = 0; i < (1 << 22); ++i) {
      int v;
      asm volatile("ld.acquire.sys.global.b32 %0, [%1];\n" : "=r"(v) : "l"(local_flags + t) : "memory");
      if (v - epoch >= 0) {  // epochs only grow; a peer may already have posted the next one
        ok = true;
        break;
      }
      __nanosleep(100);
    }
    if (!ok) set_status(status, ST_PEER_TIMEOUT);
  }
  __syncwarp();
}
}  // namespace

cudaError_t launch_peer_barrier(int* local_flags, const PeerFlags& peers, int n, int rank, int epoch, int* status,
                                cudaStream_t stream) {
  if (n < 1 || n > kMaxPeers) return cudaErrorInvalidValue;
  cudaError_t e = launch_pdl(pa_peer_barrier_kernel, dim3(1), dim3(32), 0, stream, local_flags, peers, n, rank, epoch,
                             status);
  if (e != cudaSuccess) return e;
  return cudaGetLastError();
}

cudaError_t launch_decode(const AttnParams& p, const KvMaps* maps, int kv_kind, int q_bf16, int D, int nt,
                          const DecodeLaunch& plan, cudaStream_t stream, int phase) {
  KvMaps none{};
  const KvMaps& m = maps ? *maps : none;
  const bool tma = maps != nullptr;
  if (D == 64) return launch_kv<64>(p, m, kv_kind, q_bf16, nt, tma, plan, phase, stream);
  if (D == 128) return launch_kv<128>(p, m, kv_kind, q_bf16, nt, tma, plan, phase, stream);
  return cudaErrorInvalidValue;
}

}  // namespace pa
