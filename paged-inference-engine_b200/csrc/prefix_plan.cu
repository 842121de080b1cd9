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

// Rows of sequence b, the keys that its last row sees (0 without rows), and the keys that its first does.  The
// loads do not wait for one another.
struct SeqKeys {
  int rows, keys, first;
  bool bad;
  __device__ __forceinline__ SeqKeys(const SharedParams& p, int b) {
    const int n = p.nblk[b], len = p.kvlen[b];
    rows = seq_rows(p, b);
    const long long cap = static_cast<long long>(max(0, min(n, p.bt_cols))) << p.log2BS;
    keys = rows > 0 ? static_cast<int>(max(0LL, min(static_cast<long long>(len), cap))) : 0;
    first = min(keys, max(0, len - rows + 1));
    bad = rows > 0 && n > p.bt_cols;
  }
};

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
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, T = blockDim.x;
  const int per = (n + T - 1) / T;
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
    int v = lane < (T >> 5) ? s_warp[lane] : 0;
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
  if (tid == T - 1) at[n] = run;
  __syncthreads();
}

__global__ void __launch_bounds__(1024) prefix_plan_kernel(const SharedParams p) {
  pdl_enter();
  extern __shared__ int s_plan[];
  const int tid = threadIdx.x, T = blockDim.x, G = p.groups, B = p.B;
  int* s_start = s_plan;            // [G + 1]
  int* s_keys = s_start + G + 1;    // [G] shared keys
  int* s_lead = s_keys + G;         // [G]
  int* s_count = s_lead + G;        // [G]
  int* s_unit = s_count + G;        // [G + 1]
  int* s_tile = s_unit + G + 1;     // [2 B + 1]
  __shared__ int s_warp[32];
  __shared__ int s_team;

  const SeqKeys mine(p, min(tid, B - 1));  // asked for together with the groups
  int bad = 0;
  for (int i = tid; i <= G; i += T) {
    const int s = p.group_start[i];
    s_start[i] = s;
    bad |= s < 0 || s > B || (i > 0 && p.group_start[i - 1] > s);
    if (i < G) {
      s_keys[i] = max(0, p.prefix_len[i]);
      s_lead[i] = INT_MAX;
      s_count[i] = 0;
    }
  }
  if (tid == 0) s_team = 1;
  bad = __syncthreads_or(bad);
  if (bad && tid == 0) set_status(p.status, ST_BAD_SEQ_INDEX);

  for (int b = tid; b < B; b += T) {
    const SeqKeys s = b == tid ? mine : SeqKeys(p, b);
    if (s.bad) set_status(p.status, ST_BAD_NUM_BLOCKS);
    const int g = bad || s.keys == 0 ? -1 : group_of(s_start, G, b);
    if (g < 0) continue;
    atomicMin(&s_keys[g], s.first);
    atomicMin(&s_lead[g], b);
    atomicAdd(&s_count[g], 1);
  }
  __syncthreads();
  const int per = p.maxq * p.G;
  for (int g = tid; g < G; g += T) {
    const int keys = s_count[g] < 2 ? 0 : s_keys[g] & ~(p.BS - 1);
    s_keys[g] = keys;
    const int n = keys > 0 ? s_start[g + 1] - s_start[g] : 0;
    p.grp[g] = make_int4(keys, s_start[g], n, s_lead[g]);
    if (p.wide && n > 0) atomicMax(&s_team, min(p.wide_ctas, (n * per + 2 * kWideRows - 1) / (2 * kWideRows)));
  }
  __syncthreads();
  if (p.wide) {
    const int team = s_team, teams = p.wide_ctas / team;
    for (int g = tid; g < G; g += T) {
      int steps = 0;
      if (s_keys[g] > 0) {
        const WideShape s(s_keys[g], s_start[g + 1] - s_start[g], per, team);
        steps = s.passes * p.Hkv * s.steps();
      }
      s_unit[g] = steps;
    }
    __syncthreads();
    scan_cta(s_unit, G, s_warp);
    for (int g = tid; g <= G; g += T) p.step0[g] = s_unit[g];
    // (Runs made longer, so that none crosses from one list entry into the next, left more teams idle than the crossings
    // cost: 54 against 50-51 us for 64 sequences over 8192 keys, 125 against 113-116 for 4 groups of 32 over 16384 INT8 keys.)
    if (tid == 0) p.head[0] = make_int4(team, (s_unit[G] + teams - 1) / teams, s_unit[G], 0);  // no wait has given up
  }

  for (int b = tid; b < B; b += T) {
    const int keys = (b == tid ? mine : SeqKeys(p, b)).keys;
    const int g = bad ? -1 : group_of(s_start, G, b);
    int4 chunk = make_int4(0, 0, 0, 0), own = make_int4(keys, 0, 0, 0);
    if (g >= 0 && s_keys[g] > 0) {
      const int first = s_start[g], last = s_start[g + 1];
      if (p.wide) {
        p.info[b] = make_int4(s_unit[g], 0, 0, 0);
        own.z = first;
        own.w = last - first;
      } else {
        const int lead = first + (b - first) / p.cpm * p.cpm;
        const int n = min(p.cpm, last - lead);
        if (b == lead) chunk = make_int4(s_keys[g], 0, s_lead[g], n);  // (split-K form: the leader is still there)
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
  for (int i = tid; i <= 2 * B; i += T) p.tstart[i] = s_tile[i];
  if (!p.wide) {
    for (int b = tid; b < B; b += T) {
      const int g = bad ? -1 : group_of(s_start, G, b);
      if (g < 0 || s_keys[g] == 0) continue;
      const int lead = s_start[g] + (b - s_start[g]) / p.cpm * p.cpm;
      p.info[b] = make_int4(s_tile[lead], s_tile[lead + 1] - s_tile[lead], 0, 0);
    }
  }
}

constexpr int MERGE_WARPS = 8;

// Joins the pieces of every output row.  Grid (Hkv * column sets, B); a column (query row and head) is taken by SHARE
// warps, warp w having every SHARE-th piece: lane i reads the statistics of its i-th, then all lanes add up the pieces' rows with
// their weights, 16 bytes a lane and eight rows in flight; the warps' results meet in shared memory.  Few rows are bound by
// the latency of dependent loads: four warps a column, 5.7 us for one request of four beams against 9.8 with one.  Many
// are bound by how many warps there is room for: one a column, 10 us for 128 sequences of 32 heads against 24 with four.
template <int D, int SHARE>
__global__ void __launch_bounds__(32 * MERGE_WARPS, 3) prefix_merge_kernel(const SharedParams p) {
  pdl_enter();
  __shared__ float s_o[SHARE > 1 ? MERGE_WARPS : 1][D];
  __shared__ float2 s_ml[MERGE_WARPS];
  constexpr int COLS = MERGE_WARPS / SHARE;
  const int b = blockIdx.y;
  const int per = p.maxq * p.G;
  const int sets = (per + COLS - 1) / COLS;
  const int kvh = blockIdx.x / sets;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int col = (blockIdx.x - kvh * sets) * COLS + warp / SHARE;
  const int share = warp % SHARE;
  const int rows = seq_rows(p, b);
  const int4 own = p.rec[p.B + b];
  const int4 info = p.info[b];
  const int t_own = p.tstart[p.B + b], n_own = p.tstart[p.B + b + 1] - t_own;
  const int tiles = p.tstart[2 * p.B];
  const int4 head = p.wide ? p.head[0] : make_int4(1, 1, 0, 0);
  const int chunk = max(p.min_chunk, (tiles * p.Hkv + p.num_warps_total - 1) / p.num_warps_total);
  int o0 = 0, on = 0;  // first piece of the sequence's own keys, pieces
  if (n_own > 0) {
    const int s0 = t_own * p.Hkv + kvh * n_own;
    o0 = s0 / chunk;
    on = (s0 + n_own - 1) / chunk - o0 + 1;
  }
  if (own.y == 0 && on == 1) return;  // written by the split-K kernel
  const bool mine = col < rows * p.G;
  if (SHARE == 1 && !mine) return;
  const bool wide = p.wide && own.y > 0;
  // pieces of the shared part: `cn`, the first of worker or team f0
  WideShape shape;
  int f0 = 0, cn = 0, s0 = 0;
  int crow = 0;  // (partial rows fit 32 bits: checked on the host)
  if (wide) {
    shape = WideShape(own.y, own.w, per, head.x);
    const int R = (b - own.z) * per + col;
    int rp = R / (2 * kWideRows), seg = kvh;
    const int in_pair = R - rp * 2 * kWideRows;
    if (shape.passes > 1) {
      seg += rp / shape.lanes * p.Hkv;
      rp %= shape.lanes;
    }
    s0 = info.x + seg * shape.steps();
    f0 = s0 / head.y;
    cn = ((s0 + shape.steps() - 1) / head.y - f0 + 1) << shape.lparts;
    crow = static_cast<int>(shared_wide_row(p, shape, own.z, seg, f0, head.x, 0, rp)) + in_pair;
  } else if (own.y > 0) {
    s0 = info.x * p.Hkv + kvh * info.y;
    f0 = s0 / chunk;
    cn = (s0 + info.y - 1) / chunk - f0 + 1;
    crow = static_cast<int>(shared_chunk_row(p, own.z, own.w, kvh, f0)) + (b - own.z) * per + col;
  }
  const int orow = static_cast<int>(shared_own_row(p, b, kvh, o0)) + col;
  // the partial row of piece i, or -1 where a team's part is empty
  auto piece = [&](int i) -> int {
    if (i < on) return orow + i * per;
    i -= on;
    if (!wide) return crow + i * kChunkCols;
    const int t = i >> shape.lparts, q = i - (t << shape.lparts);
    const int a = (f0 + t) * head.y - s0;
    int n;
    wide_tiles(shape, max(0, a), min(shape.steps(), a + head.y), q, n);
    return n > 0 ? crow + t * head.x * 2 * kWideRows + q * shape.lanes * shape.room : -1;
  };
  const int np = mine ? on + cn : 0;
  constexpr int LPR = D / 4;     // lanes of a row (16 bytes each)
  constexpr int RPI = 32 / LPR;  // rows of a load instruction
  const int sub = lane / LPR, at = lane % LPR;
  float M = -INFINITY, l = 0.f;
  float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int base = share; base < np; base += 32 * SHARE) {
    const int i = base + lane * SHARE;
    const int r = i < np ? piece(i) : -1;
    float2 ml = make_float2(-INFINITY, 0.f);
    if (r >= 0) ml = reinterpret_cast<const float2*>(p.part_ml)[r];
    // joined with what the pieces before gave
    const float Mn = fmaxf(M, warp_max_xor(ml.x, 1));
    const float Mu = Mn == -INFINITY ? 0.f : Mn;
    const float old = ex2(M - Mu), f = ex2(ml.x - Mu);
    M = Mn;
    l = l * old + ml.y * f;
    acc.x *= old, acc.y *= old, acc.z *= old, acc.w *= old;
    const int n = min(32, (np - base + SHARE - 1) / SHARE);
#pragma unroll 1
    for (int j0 = 0; j0 < n; j0 += 8 * RPI) {
      float4 v[8];
      float w[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        const int j = j0 + k * RPI + sub;
        const int rj = __shfl_sync(0xffffffffu, r, j & 31);
        w[k] = __shfl_sync(0xffffffffu, f, j & 31);
        v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (j < n && rj >= 0) v[k] = *reinterpret_cast<const float4*>(p.part_o + static_cast<long long>(rj) * D + 4 * at);
        else w[k] = 0.f;
      }
#pragma unroll
      for (int k = 0; k < 8; ++k) acc.x += v[k].x * w[k], acc.y += v[k].y * w[k], acc.z += v[k].z * w[k], acc.w += v[k].w * w[k];
    }
  }
  l = warp_sum_xor(l, 1);
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1) {
    acc.x += __shfl_xor_sync(0xffffffffu, acc.x, o);
    acc.y += __shfl_xor_sync(0xffffffffu, acc.y, o);
    acc.z += __shfl_xor_sync(0xffffffffu, acc.z, o);
    acc.w += __shfl_xor_sync(0xffffffffu, acc.w, o);
  }
  const int qi = col / p.G, hq = col - qi * p.G + kvh * p.G;
  __half* out = static_cast<__half*>(p.o) + o_seq_base(p, b) + hq * p.o_sh + static_cast<long long>(qi) * p.o_sm;
  auto store_lse = [&](float m, float sum) {
    const float L = sum > 0.f ? (m + lg2(sum)) * 0.6931471805599453f : -INFINITY;
    static_cast<__half*>(p.lse)[l_seq_base(p, b) + hq * p.l_sh + static_cast<long long>(qi) * p.l_sm] = __float2half_rn(L);
  };
  if constexpr (SHARE == 1) {
    const float inv = l > 0.f ? 1.f / l : 0.f;
    if (sub == 0) {
      reinterpret_cast<__half2*>(out + 4 * at)[0] = __floats2half2_rn(acc.x * inv, acc.y * inv);
      reinterpret_cast<__half2*>(out + 4 * at)[1] = __floats2half2_rn(acc.z * inv, acc.w * inv);
    }
    if (lane == 0 && p.lse) store_lse(M, l);
  } else {
    if (sub == 0) *reinterpret_cast<float4*>(&s_o[warp][4 * at]) = acc;
    if (lane == 0) s_ml[warp] = make_float2(M, l);
    __syncthreads();
    if (!mine || share != 0) return;
    float Mt = M;
#pragma unroll
    for (int k = 1; k < SHARE; ++k) Mt = fmaxf(Mt, s_ml[warp + k].x);
    const float Mu = Mt == -INFINITY ? 0.f : Mt;
    float lt = 0.f;
    float o[D / 32];
#pragma unroll
    for (int i = 0; i < D / 32; ++i) o[i] = 0.f;
#pragma unroll
    for (int k = 0; k < SHARE; ++k) {
      const float f = ex2(s_ml[warp + k].x - Mu);
      lt += s_ml[warp + k].y * f;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) o[i] += s_o[warp + k][lane * (D / 32) + i] * f;
    }
    const float inv = lt > 0.f ? 1.f / lt : 0.f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i)
      reinterpret_cast<__half2*>(out + lane * (D / 32))[i] = __floats2half2_rn(o[2 * i] * inv, o[2 * i + 1] * inv);
    if (lane == 0 && p.lse) store_lse(Mt, lt);
  }
}

}  // namespace

cudaError_t launch_prefix_plan(const SharedParams& p, cudaStream_t stream) {
  const auto bytes = [](size_t groups, size_t B) { return (5 * groups + 2 + 2 * B + 1) * sizeof(int); };
  const size_t smem = bytes(p.groups, p.B);
  if (smem > 48 * 1024) {
    static std::atomic<unsigned long long> done{0};
    const cudaError_t e = allow_smem(prefix_plan_kernel, static_cast<int>(bytes(kMaxSharedSeqs, kMaxSharedSeqs)), done);
    if (e != cudaSuccess) return e;
  }
  // a thread for each work list entry: barriers cost more the more threads meet at them
  const int most = 2 * p.B > p.groups ? 2 * p.B : p.groups;
  const int threads = most >= 1024 ? 1024 : most <= 128 ? 128 : (most + 31) / 32 * 32;
  return launch_pdl(prefix_plan_kernel, dim3(1), dim3(threads), smem, stream, p);
}

cudaError_t launch_prefix_merge(const SharedParams& p, int D, cudaStream_t stream) {
  const int per = p.maxq * p.G;
  auto go = [&](auto kern, int share) {
    const int cols = MERGE_WARPS / share;
    return launch_pdl(kern, dim3(p.Hkv * ((per + cols - 1) / cols), p.B), dim3(32 * MERGE_WARPS), 0, stream, p);
  };
  if (static_cast<long long>(p.B) * p.Hkv * per <= 8 * device_sm_count())
    return D == 64 ? go(prefix_merge_kernel<64, 4>, 4) : go(prefix_merge_kernel<128, 4>, 4);
  return D == 64 ? go(prefix_merge_kernel<64, 1>, 1) : go(prefix_merge_kernel<128, 1>, 1);
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
