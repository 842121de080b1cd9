// Attention of a batch whose groups share a prefix: the work list and the join.
//
// Softmax attention over a set of keys is known by three values a row, its
// maximum logit m, the sum l of 2^(s - m) and the sum o of 2^(s - m) v (base 2, scaled
// logits), and two disjoint sets join as m = max(m1, m2), (l, o) = 2^(m1 - m) (l1, o1) +
// 2^(m2 - m) (l2, o2).  So the keys that a group's sequences share are read once for all of
// them, by one of two kernels, what each has to itself once by the split-K kernel, and
// prefix_merge_kernel joins the pieces.  The reference attends for every sequence
// by itself (kernels/flash_attention.py:38-123).
//
// prefix_plan_kernel settles, from lengths that only the device may know, what a group
// shares: min(prefix_len, what every row of every member sees), in whole blocks, read through
// the block table of its first member with keys.  No key of a shared part is masked for
// any row, so what a masked slot holds (another sequence's NaN) is never multiplied in.  Groups with fewer
// than two such members share nothing.
#include <climits>

#include "pa_common.cuh"

namespace pa {
namespace {

constexpr int PLAN_THREADS = 1024;

// Visible keys of sequence b's last row (0 for a sequence without rows).
__device__ __forceinline__ int plan_keys(const SharedParams& p, int b, int rows) {
  if (rows <= 0) return 0;
  const long long cap = static_cast<long long>(max(0, min(p.nblk[b], p.bt_cols))) << p.log2BS;
  return static_cast<int>(max(0LL, min(static_cast<long long>(p.kvlen[b]), cap)));
}

// The group of sequence b in the rising starts s_start[0..G], or -1.
__device__ __forceinline__ int group_of(const int* s_start, int G, int b) {
  if (G <= 0 || b < s_start[0] || b >= s_start[G]) return -1;
  int lo = 0, hi = G - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (s_start[mid] <= b) lo = mid;
    else hi = mid - 1;
  }
  return lo;
}

// Exclusive scan of at[0..n) in place by the whole CTA, the sum to at[n].
__device__ void scan_cta(int* at, int n, int* s_warp) {
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int per = (n + PLAN_THREADS - 1) / PLAN_THREADS;
  const int i0 = min(tid * per, n), i1 = min(i0 + per, n);
  int sum = 0;
  for (int i = i0; i < i1; ++i) sum += at[i];
  int x = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, x, o);
    if (lane >= o) x += y;
  }
  if (lane == 31) s_warp[warp] = x;
  __syncthreads();
  if (warp == 0) {
    int v = s_warp[lane];
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, v, o);
      if (lane >= o) v += y;
    }
    s_warp[lane] = v;
  }
  __syncthreads();
  int run = x - sum + (warp ? s_warp[warp - 1] : 0);
  for (int i = i0; i < i1; ++i) {
    const int v = at[i];
    at[i] = run;
    run += v;
  }
  if (tid == PLAN_THREADS - 1) at[n] = run;
  __syncthreads();
}

__global__ void __launch_bounds__(PLAN_THREADS) prefix_plan_kernel(const SharedParams p) {
  pdl_enter();
  extern __shared__ int s_plan[];
  const int tid = threadIdx.x, G = p.groups, B = p.B;
  int* s_start = s_plan;            // [G + 1]
  int* s_keys = s_start + G + 1;    // [G] shared keys
  int* s_lead = s_keys + G;         // [G]
  int* s_count = s_lead + G;        // [G]
  int* s_unit = s_count + G;        // [G + 1]
  int* s_tile = s_unit + G + 1;     // [2 B + 1]
  __shared__ int s_warp[32];

  int bad = 0;
  for (int i = tid; i <= G; i += PLAN_THREADS) {
    const int s = p.group_start[i];
    s_start[i] = s;
    bad |= s < 0 || s > B || (i > 0 && p.group_start[i - 1] > s);
    if (i < G) {
      s_keys[i] = max(0, p.prefix_len[i]);
      s_lead[i] = INT_MAX;
      s_count[i] = 0;
    }
  }
  bad = __syncthreads_or(bad);
  if (bad && tid == 0) set_status(p.status, ST_BAD_SEQ_INDEX);

  for (int b = tid; b < B; b += PLAN_THREADS) {
    const int rows = seq_rows(p, b);
    const int keys = plan_keys(p, b, rows);
    if (rows > 0 && p.nblk[b] > p.bt_cols) set_status(p.status, ST_BAD_NUM_BLOCKS);
    const int g = bad || keys == 0 ? -1 : group_of(s_start, G, b);
    if (g < 0) continue;
    atomicMin(&s_keys[g], min(keys, max(0, p.kvlen[b] - rows + 1)));  // what its first row sees
    atomicMin(&s_lead[g], b);
    atomicAdd(&s_count[g], 1);
  }
  __syncthreads();
  const int per = p.maxq * p.G;
  for (int g = tid; g < G; g += PLAN_THREADS) {
    const int keys = s_count[g] < 2 ? 0 : s_keys[g] & ~(p.BS - 1);
    s_keys[g] = keys;
    int units = 0;
    if (p.wide && keys > 0) {
      const int n = s_start[g + 1] - s_start[g];
      units = p.Hkv * ((n * per + kWideRows - 1) / kWideRows) * ((keys + kWideKeys - 1) / kWideKeys);
    }
    s_unit[g] = units;
    p.grp[g] = make_int4(keys, s_start[g], keys > 0 ? s_start[g + 1] - s_start[g] : 0, s_lead[g]);
  }
  __syncthreads();
  if (p.wide) {
    scan_cta(s_unit, G, s_warp);
    for (int g = tid; g <= G; g += PLAN_THREADS) p.unit0[g] = s_unit[g];
  }

  for (int b = tid; b < B; b += PLAN_THREADS) {
    const int keys = plan_keys(p, b, seq_rows(p, b));
    const int g = bad ? -1 : group_of(s_start, G, b);
    int4 chunk = make_int4(0, 0, 0, 0), own = make_int4(keys, 0, 0, 0);
    if (g >= 0 && s_keys[g] > 0) {
      const int first = s_start[g], last = s_start[g + 1];
      if (p.wide) {
        chunk.y = s_unit[g];
        own.z = first;
        own.w = last - first;
      } else {
        const int lead = first + (b - first) / p.cpm * p.cpm;
        const int n = min(p.cpm, last - lead);
        if (b == lead) chunk = make_int4(s_keys[g], 0, s_lead[g], n);
        own.z = lead;
        own.w = n;
      }
      if (keys > 0) {
        own.x = keys - s_keys[g];
        own.y = s_keys[g];
      }
    }
    p.rec[b] = chunk;
    p.rec[B + b] = own;
    s_tile[b] = (chunk.x + p.decode_tile - 1) / p.decode_tile;
    s_tile[B + b] = (own.x + p.decode_tile - 1) / p.decode_tile;
  }
  __syncthreads();
  scan_cta(s_tile, 2 * B, s_warp);
  for (int i = tid; i <= 2 * B; i += PLAN_THREADS) p.tstart[i] = s_tile[i];
}

// Joins the pieces of every output row.  Grid (Hkv, B), a warp per (row, head) column: lane i reads the statistics of piece
// i, 32 at a time; the rows of the pieces are then added up with their weights.
template <int D>
__global__ void __launch_bounds__(128) prefix_merge_kernel(const SharedParams p) {
  pdl_enter();
  const int kvh = blockIdx.x, b = blockIdx.y;
  const int rows = seq_rows(p, b);
  if (rows <= 0) return;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int per = p.maxq * p.G;
  const int4 own = p.rec[p.B + b];
  const int W = p.num_warps_total;
  const int total = p.tstart[2 * p.B] * p.Hkv;
  const int chunk = max(1, (total + W - 1) / W);
  // pieces of the list entries [s0, s0 + n)
  int o0 = 0, on = 0;
  {
    const int t0 = p.tstart[p.B + b], n = p.tstart[p.B + b + 1] - t0;
    if (n > 0) {
      const int s0 = t0 * p.Hkv + kvh * n;
      o0 = s0 / chunk;
      on = (s0 + n - 1) / chunk - o0 + 1;
    }
  }
  if (own.y == 0 && on == 1) return;  // written by the split-K kernel
  const int head0 = kvh * p.G;
  for (int col = warp; col < rows * p.G; col += 4) {
    const int qi = col / p.G, hq = col - qi * p.G;
    int c0 = 0, cn = 0;
    long long crow = 0;  // partial row of piece 0
    int cstep = 0;
    if (own.y > 0) {
      if (p.wide) {
        const int R = (b - own.z) * per + col, rows_g = own.w * per;
        const int KT = (own.y + kWideKeys - 1) / kWideKeys, RT = (rows_g + kWideRows - 1) / kWideRows;
        const int units = p.unit0[p.groups];
        const int wchunk = (units + p.wide_ctas - 1) / p.wide_ctas;
        const int s0 = p.rec[b].y + (kvh * RT + R / kWideRows) * KT;
        c0 = s0 / wchunk;
        cn = (s0 + KT - 1) / wchunk - c0 + 1;
        crow = shared_wide_row(p, own.z, rows_g, kvh, R / kWideRows, c0) + R % kWideRows;
        cstep = kWideRows;
      } else {
        const int t0 = p.tstart[own.z], n = p.tstart[own.z + 1] - t0;
        const int s0 = t0 * p.Hkv + kvh * n;
        c0 = s0 / chunk;
        cn = (s0 + n - 1) / chunk - c0 + 1;
        crow = shared_chunk_row(p, own.z, own.w, kvh, c0) + (b - own.z) * per + col;
        cstep = kChunkCols;
      }
    }
    const long long orow0 = shared_own_row(p, b, kvh, o0) + col;
    auto piece = [&](int i) { return i < on ? orow0 + static_cast<long long>(i) * per : crow + static_cast<long long>(i - on) * cstep; };
    const int np = on + cn;
    float M = -INFINITY;
    for (int i = lane; i < np; i += 32) M = fmaxf(M, p.part_ml[piece(i) * 2]);
    M = warp_max_xor(M, 1);
    const float Mu = M == -INFINITY ? 0.f : M;
    float l = 0.f, o[D / 32];
#pragma unroll
    for (int k = 0; k < D / 32; ++k) o[k] = 0.f;
    for (int base = 0; base < np; base += 32) {
      float f = 0.f;
      if (base + lane < np) {
        const float2 ml = *reinterpret_cast<const float2*>(p.part_ml + piece(base + lane) * 2);
        f = ex2(ml.x - Mu);
        l += ml.y * f;
      }
      const int n = min(32, np - base);
#pragma unroll 4
      for (int j = 0; j < n; ++j) {
        const float fj = __shfl_sync(0xffffffffu, f, j);
        const float* po = p.part_o + piece(base + j) * D;
#pragma unroll
        for (int k = 0; k < D / 32; ++k) o[k] += po[lane + 32 * k] * fj;
      }
    }
    l = warp_sum_xor(l, 1);
    const float inv = l > 0.f ? 1.f / l : 0.f;
    const long long orow = o_seq_base(p, b) + (head0 + hq) * p.o_sh + static_cast<long long>(qi) * p.o_sm;
#pragma unroll
    for (int k = 0; k < D / 32; ++k) static_cast<__half*>(p.o)[orow + lane + 32 * k] = __float2half_rn(o[k] * inv);
    if (lane == 0 && p.lse) {
      const float L = l > 0.f ? (M + lg2(l)) * 0.6931471805599453f : -INFINITY;
      static_cast<__half*>(p.lse)[l_seq_base(p, b) + (head0 + hq) * p.l_sh + static_cast<long long>(qi) * p.l_sm] =
          __float2half_rn(L);
    }
  }
}

}  // namespace

cudaError_t launch_prefix_plan(const SharedParams& p, cudaStream_t stream) {
  const size_t smem = (5 * static_cast<size_t>(p.groups) + 2 + 2 * static_cast<size_t>(p.B) + 1) * sizeof(int);
  if (smem > 48 * 1024) {
    cudaError_t e = cudaFuncSetAttribute(prefix_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
  }
  return launch_pdl(prefix_plan_kernel, dim3(1), dim3(PLAN_THREADS), smem, stream, p);
}

cudaError_t launch_prefix_merge(const SharedParams& p, int D, cudaStream_t stream) {
  return launch_pdl(D == 64 ? prefix_merge_kernel<64> : prefix_merge_kernel<128>, dim3(p.Hkv, p.B), dim3(128), 0, stream, p);
}

}  // namespace pa

// Launches of the split-K kernel over the work list, by the pool's type (csrc/prefix_decode_*.cu).
namespace pa {
template <int KVT>
int prefix_decode_plan_kv(int q_bf16, int D, int nt, int B, bool tma, DecodeLaunch* out);
template <int KVT>
cudaError_t prefix_decode_launch_kv(const SharedParams& p, const KvMaps& m, int D, int nt, bool tma, const DecodeLaunch& pl,
                                    cudaStream_t s);

int prefix_decode_plan(int kv_kind, int q_bf16, int D, int nt, int B, int use_tma, DecodeLaunch* out) {
  switch (kv_kind) {
    case KV_F16:
      return prefix_decode_plan_kv<KV_F16>(q_bf16, D, nt, B, use_tma, out);
    case KV_BF16:
      return prefix_decode_plan_kv<KV_BF16>(q_bf16, D, nt, B, use_tma, out);
    default:
      return prefix_decode_plan_kv<KV_I8>(q_bf16, D, nt, B, use_tma, out);
  }
}

cudaError_t launch_prefix_decode(const SharedParams& p, const KvMaps* maps, int kv_kind, int D, int nt,
                                 const DecodeLaunch& plan, cudaStream_t stream) {
  KvMaps none{};
  const KvMaps& m = maps ? *maps : none;
  const bool tma = maps != nullptr;
  switch (kv_kind) {
    case KV_F16:
      return prefix_decode_launch_kv<KV_F16>(p, m, D, nt, tma, plan, stream);
    case KV_BF16:
      return prefix_decode_launch_kv<KV_BF16>(p, m, D, nt, tma, plan, stream);
    default:
      return prefix_decode_launch_kv<KV_I8>(p, m, D, nt, tma, plan, stream);
  }
}
}  // namespace pa
