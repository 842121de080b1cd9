// The split-K decode kernel over the work list of a shared-prefix problem, for
// one pool type (one translation unit each, so that they compile side by side).
#pragma once

#include "decode_kernel.cuh"

namespace pa {
namespace {

template <int D, int KVT, int QT, int NT, bool TMA>
struct SharedInst {
  using Lay = DecLayout<D, KVT, NT>;
  static constexpr auto kern = pa_decode_kernel<D, KVT, QT, NT, TMA, true>;
  static int plan(int B, DecodeLaunch* out) {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess) return -1;
    if (cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess) return -1;
    const int fixed = (((2 * B + 1) * 4 + 127) & ~127) + 1024;  // scan + alignment slack
    int nw = (SMEM_LIMIT - fixed) / Lay::WARPB;
    if (nw > max_warps<NT>()) nw = max_warps<NT>();
    if (nw < 1) return -1;
    out->warps_per_cta = nw;
    out->smem = static_cast<size_t>(fixed + nw * Lay::WARPB);
    out->ctas = sms;  // the ring takes most of an SM's shared memory: one CTA each
    return 0;
  }
  static cudaError_t launch(const SharedParams& p, const KvMaps& maps, const DecodeLaunch& pl, cudaStream_t stream) {
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = allow_smem(kern, SMEM_LIMIT, done);  // pl.smem goes by B
    if (e != cudaSuccess) return e;
    return launch_pdl(kern, dim3(pl.ctas), dim3(pl.warps_per_cta * 32), pl.smem, stream, p, maps);
  }
};

template <int KVT, class F>
auto shared_select(int q_bf16, int D, int nt, bool tma, F&& f) {
  auto by_tma = [&](auto d, auto q, auto n) {
    constexpr int DD = decltype(d)::value, QQ = decltype(q)::value, NN = decltype(n)::value;
    return tma ? f(SharedInst<DD, KVT, QQ, NN, true>{}) : f(SharedInst<DD, KVT, QQ, NN, false>{});
  };
  auto by_nt = [&](auto d, auto q) {
    return nt == 1 ? by_tma(d, q, std::integral_constant<int, 1>{}) : by_tma(d, q, std::integral_constant<int, 2>{});
  };
  auto by_q = [&](auto d) {
    return q_bf16 ? by_nt(d, std::integral_constant<int, Q_BF16>{}) : by_nt(d, std::integral_constant<int, Q_F16>{});
  };
  return D == 64 ? by_q(std::integral_constant<int, 64>{}) : by_q(std::integral_constant<int, 128>{});
}

}  // namespace

template <int KVT>
int prefix_decode_plan_kv(int q_bf16, int D, int nt, int B, bool tma, DecodeLaunch* out) {
  return shared_select<KVT>(q_bf16, D, nt, tma, [&](auto i) { return i.plan(B, out); });
}
template <int KVT>
cudaError_t prefix_decode_launch_kv(const SharedParams& p, const KvMaps& m, int D, int nt, bool tma, const DecodeLaunch& pl,
                                    cudaStream_t s) {
  return shared_select<KVT>(p.q_bf16, D, nt, tma, [&](auto i) { return i.launch(p, m, pl, s); });
}

}  // namespace pa
