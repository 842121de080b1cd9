// torch.library registration of the paged-attention C ABI (libpaged_attn_b200.so):
// the thin torch extension the Python drop-in calls.
//
//   pie_b200::paged_attention(_out)         flash_attention_forward
//                                           (kernels/flash_attention.py:139-172)
//   pie_b200::paged_attention_varlen(_out)  the same over packed query rows
//   pie_b200::write_kv                      the quantise-on-write / copy of new
//                                           K/V rows (transformer/model.py:85-122)
//   pie_b200::project_write_kv              the K/V projection with that write in
//                                           its epilogue (transformer/model.py:75-122)
//   pie_b200::shared_prefix_attention(_out)       decode attention over groups that share a prefix
//   pie_b200::rotate_write_kv(_out)               new query and key rows rotated by their
//                                           positions, K/V rows written
//   pie_b200::adjust_logits(_out)                 penalties, biases and masks on logits
//   pie_b200::copy_blocks                   page copies inside the pools of all layers
//   pie_b200::reorder_beams                 beams take over their parents' pool rows
//   pie_b200::compact_blocks                the blocks in use move to the lowest ids
//   pie_b200::beam_select                   the best continuations of every
//                                           sequence's beams
//
// Each op reads pointers, sizes and element strides from its tensors, fills the
// C structs of include/paged_attn_b200.h and calls the library on the current
// CUDA stream of the tensors' device; a nonzero return code becomes a
// TORCH_CHECK failure (RuntimeError) carrying paged_attn_error_string().  The
// split-K workspace is one cached uint8 tensor per device from torch's
// allocator, grown on demand.  Meta kernels give shapes for fake tensors.
// Malformed arguments raise ValueError (TORCH_CHECK_VALUE), as the Python
// front end does; a failing library call raises RuntimeError.
//
// Pools arrive as [num_blocks, block_size, num_kv_heads, head_dim] views (the
// launcher's [block, slot, head, d] reading, kernels/flash_attention.py:158-159);
// scales as [num_blocks, num_kv_heads] (per block) or
// [num_blocks, block_size, num_kv_heads] (per token).
#include <ATen/ATen.h>
#include <ATen/cuda/EmptyTensor.h>
#include <c10/cuda/CUDAGuard.h>
#include <c10/cuda/CUDAStream.h>
#include <torch/library.h>

#include <mutex>
#include <optional>
#include <vector>

#include "paged_attn_b200.h"

namespace {

int pa_dtype(at::ScalarType t) {
  switch (t) {
    case at::kHalf:
      return PA_DTYPE_F16;
    case at::kBFloat16:
      return PA_DTYPE_BF16;
    case at::kChar:
      return PA_DTYPE_I8;
    case at::kFloat:
      return PA_DTYPE_F32;
    default:
      TORCH_CHECK_VALUE(false, "pie_b200: unsupported dtype ", t);
  }
  return -1;
}

void check_rc(int rc, const char* fn) {
  TORCH_CHECK(rc == PA_OK, fn, " failed (code ", rc, "): ", paged_attn_error_string());
}

void* ptr(const at::Tensor& t) { return t.data_ptr(); }
template <typename T>
T* opt_ptr(const std::optional<at::Tensor>& t) {
  return t.has_value() ? static_cast<T*>(t->data_ptr()) : nullptr;
}

void check_device(const at::Tensor& ref, const at::Tensor& t, const char* name) {
  TORCH_CHECK_VALUE(t.is_cuda() && t.device() == ref.device(), "pie_b200: ", name, " must be on ", ref.device());
}
void check_i32(const at::Tensor& ref, const at::Tensor& t, const char* name, int64_t n) {
  check_device(ref, t, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.dim() == 1 && t.is_contiguous(), "pie_b200: ", name,
              " must be a contiguous int32 vector");
  TORCH_CHECK_VALUE(t.numel() == n, "pie_b200: ", name, " has ", t.numel(), " entries, expected ", n);
}

void check_vec(const at::Tensor& ref, const at::Tensor& t, const char* name) {
  check_device(ref, t, name);
  TORCH_CHECK_VALUE(t.scalar_type() == at::kInt && t.is_contiguous(), "pie_b200: ", name, " must be contiguous int32");
}

void check_status(const at::Tensor& ref, const std::optional<at::Tensor>& status) {
  if (status.has_value()) {
    check_vec(ref, *status, "status");
    TORCH_CHECK_VALUE(status->numel() >= 1, "pie_b200: status holds no word");
  }
}

pa_kv_cache_t kv_desc(const at::Tensor& K, const at::Tensor& V, const std::optional<at::Tensor>& ks,
                      const std::optional<at::Tensor>& vs) {
  TORCH_CHECK_VALUE(K.dim() == 4 && V.dim() == 4 && K.sizes() == V.sizes() && K.scalar_type() == V.scalar_type(),
              "pie_b200: K and V pools must be 4-D [num_blocks, block_size, num_kv_heads, head_dim] and alike");
  check_device(K, V, "V");
  pa_kv_cache_t kv{};
  kv.k = ptr(K);
  kv.v = ptr(V);
  kv.dtype = pa_dtype(K.scalar_type());
  kv.num_blocks = static_cast<int32_t>(K.size(0));
  kv.block_size = static_cast<int32_t>(K.size(1));
  kv.num_kv_heads = static_cast<int32_t>(K.size(2));
  kv.head_dim = static_cast<int32_t>(K.size(3));
  TORCH_CHECK_VALUE(K.stride(3) == 1 && V.stride(3) == 1, "pie_b200: K/V pools need a contiguous head_dim");
  kv.k_stride_block = K.stride(0);
  kv.k_stride_slot = K.stride(1);
  kv.k_stride_head = K.stride(2);
  kv.v_stride_block = V.stride(0);
  kv.v_stride_slot = V.stride(1);
  kv.v_stride_head = V.stride(2);
  kv.scale_dtype = PA_DTYPE_F16;
  if (kv.dtype == PA_DTYPE_I8) {
    TORCH_CHECK_VALUE(ks.has_value() && vs.has_value(), "pie_b200: an int8 KV pool needs k_scale and v_scale");
    const at::Tensor* sc[2] = {&*ks, &*vs};
    int64_t st[2][3];
    for (int i = 0; i < 2; ++i) {
      const at::Tensor& s = *sc[i];
      check_device(K, s, i ? "v_scale" : "k_scale");
      if (s.dim() == 2) {
        TORCH_CHECK_VALUE(s.size(0) == K.size(0) && s.size(1) == K.size(2), "pie_b200: per-block scales must be [",
                    K.size(0), ", ", K.size(2), "]");
        st[i][0] = s.stride(0);
        st[i][1] = 0;
        st[i][2] = s.stride(1);
      } else {
        TORCH_CHECK_VALUE(s.dim() == 3 && s.size(0) == K.size(0) && s.size(1) == K.size(1) && s.size(2) == K.size(2),
                    "pie_b200: per-token scales must be [", K.size(0), ", ", K.size(1), ", ", K.size(2), "]");
        st[i][0] = s.stride(0);
        st[i][1] = s.stride(1);
        st[i][2] = s.stride(2);
      }
    }
    TORCH_CHECK_VALUE(ks->scalar_type() == vs->scalar_type() &&
                    (ks->scalar_type() == at::kHalf || ks->scalar_type() == at::kFloat),
                "pie_b200: k_scale / v_scale must share a float16 or float32 dtype");
    kv.scale_dtype = pa_dtype(ks->scalar_type());
    kv.k_scale = ptr(*ks);
    kv.v_scale = ptr(*vs);
    kv.ks_stride_block = st[0][0];
    kv.ks_stride_slot = st[0][1];
    kv.ks_stride_head = st[0][2];
    kv.vs_stride_block = st[1][0];
    kv.vs_stride_slot = st[1][1];
    kv.vs_stride_head = st[1][2];
  }
  return kv;
}

pa_paging_t paging(const at::Tensor& ref, const at::Tensor& block_table, const at::Tensor& num_blocks,
                   const at::Tensor& q_len, const at::Tensor& kv_len) {
  check_device(ref, block_table, "block_table");
  TORCH_CHECK_VALUE(block_table.scalar_type() == at::kInt && block_table.dim() == 2,
              "pie_b200: block_table must be int32 [num_seqs, max_blocks]");
  const int64_t B = block_table.size(0);
  check_i32(ref, num_blocks, "num_blocks_per_seq", B);
  check_i32(ref, q_len, "q_len_per_seq", B);
  check_i32(ref, kv_len, "kv_len_per_seq", B);
  pa_paging_t pg{};
  pg.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  pg.bt_stride_seq = block_table.stride(0);
  pg.bt_stride_col = block_table.stride(1);
  pg.bt_cols = static_cast<int32_t>(block_table.size(1));
  pg.num_seqs = static_cast<int32_t>(B);
  pg.num_blocks_per_seq = static_cast<const int32_t*>(num_blocks.data_ptr());
  pg.q_len_per_seq = static_cast<const int32_t*>(q_len.data_ptr());
  pg.kv_len_per_seq = static_cast<const int32_t*>(kv_len.data_ptr());
  return pg;
}

// One cached workspace per device (256-byte aligned by torch's allocator).
at::Tensor workspace(const at::Device& dev, size_t bytes) {
  static std::mutex mu;
  static std::vector<at::Tensor> cache;
  std::lock_guard<std::mutex> lk(mu);
  const size_t i = static_cast<size_t>(dev.index());
  if (cache.size() <= i) cache.resize(i + 1);
  at::Tensor& ws = cache[i];
  if (!ws.defined() || static_cast<size_t>(ws.numel()) < bytes) {
    const int64_t n = static_cast<int64_t>(bytes > (1u << 20) ? bytes : (1u << 20));
    ws = at::empty({n}, at::TensorOptions().dtype(at::kByte).device(dev));
  }
  return ws;
}

// An uninitialised tensor on the current device's allocator, without a dispatch.
at::Tensor fresh(at::IntArrayRef sizes, at::ScalarType t, const at::Device& dev) {
  return at::Tensor(at::detail::empty_cuda(sizes, t, dev, std::nullopt));
}

pa_attn_io_t io_desc(const at::Tensor& Q, const at::Tensor& O, const at::Tensor& L, bool ragged, int64_t max_q_len,
                     bool causal_top_left, double softmax_scale) {
  pa_attn_io_t io{};
  io.q = ptr(Q);
  io.q_dtype = pa_dtype(Q.scalar_type());
  io.num_q_heads = static_cast<int32_t>(Q.size(1));
  io.max_q_len = static_cast<int32_t>(max_q_len);
  io.causal_top_left = causal_top_left ? 1 : 0;
  if (ragged) {  // [T, Hq, D] / [T, Hq]
    io.q_stride_seq = 0;
    io.q_stride_head = Q.stride(1);
    io.q_stride_row = Q.stride(0);
    io.o_stride_seq = 0;
    io.o_stride_head = O.stride(1);
    io.o_stride_row = O.stride(0);
    io.l_stride_seq = 0;
    io.l_stride_head = L.stride(1);
    io.l_stride_row = L.stride(0);
  } else {  // [B, Hq, maxq, D] / [B, Hq, maxq]
    io.q_stride_seq = Q.stride(0);
    io.q_stride_head = Q.stride(1);
    io.q_stride_row = Q.stride(2);
    io.o_stride_seq = O.stride(0);
    io.o_stride_head = O.stride(1);
    io.o_stride_row = O.stride(2);
    io.l_stride_seq = L.stride(0);
    io.l_stride_head = L.stride(1);
    io.l_stride_row = L.stride(2);
  }
  io.o = ptr(O);
  io.lse = ptr(L);
  io.softmax_scale = static_cast<float>(softmax_scale);
  return io;
}

void check_q(const at::Tensor& Q, int64_t dims) {
  TORCH_CHECK_VALUE(Q.is_cuda() && Q.dim() == dims, "pie_b200: Q must be a ", dims, "-D CUDA tensor");
  TORCH_CHECK_VALUE(Q.scalar_type() == at::kHalf || Q.scalar_type() == at::kBFloat16, "pie_b200: Q must be fp16 or bf16");
  TORCH_CHECK_VALUE(Q.stride(dims - 1) == 1, "pie_b200: Q needs a contiguous head_dim");
}

void check_out(const at::Tensor& Q, const at::Tensor& O, const at::Tensor& L) {
  check_device(Q, O, "out");
  check_device(Q, L, "lse");
  TORCH_CHECK_VALUE(O.scalar_type() == at::kHalf && O.sizes() == Q.sizes(), "pie_b200: out must be float16 shaped like Q");
  TORCH_CHECK_VALUE(L.scalar_type() == at::kHalf && L.sizes() == Q.sizes().slice(0, Q.dim() - 1),
              "pie_b200: lse must be float16 shaped like Q without head_dim");
}

// mode: 0 = choose (paged_attn_forward), 1 = split-K decode, 2 = prefill kernel
void paged_attention_out(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V, const at::Tensor& q_len,
                         const at::Tensor& block_table, const at::Tensor& num_blocks, const at::Tensor& kv_len,
                         const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
                         bool causal_top_left, double softmax_scale, int64_t mode,
                         const std::optional<at::Tensor>& status, at::Tensor& out, at::Tensor& lse) {
  check_q(Q, 4);
  check_out(Q, out, lse);
  check_device(Q, K, "K");
  TORCH_CHECK_VALUE(block_table.size(0) == Q.size(0), "pie_b200: block_table has ", block_table.size(0), " rows for ",
              Q.size(0), " sequences");
  const c10::cuda::CUDAGuard guard(Q.device());
  pa_kv_cache_t kv = kv_desc(K, V, k_scale, v_scale);
  pa_paging_t pg = paging(Q, block_table, num_blocks, q_len, kv_len);
  pa_attn_io_t io = io_desc(Q, out, lse, false, Q.size(2), causal_top_left, softmax_scale);
  void* stream = c10::cuda::getCurrentCUDAStream(Q.device().index()).stream();
  int32_t* st = opt_ptr<int32_t>(status);
  if (mode == 2) {
    check_rc(paged_attn_prefill(&io, &kv, &pg, st, stream), "paged_attn_prefill");
    return;
  }
  size_t bytes = 0;
  check_rc(paged_attn_workspace_size(&io, &kv, &pg, &bytes), "paged_attn_workspace_size");
  at::Tensor ws;
  if (bytes) ws = workspace(Q.device(), bytes);
  void* wp = bytes ? ws.data_ptr() : nullptr;
  const size_t wb = bytes ? static_cast<size_t>(ws.numel()) : 0;
  if (mode == 1) check_rc(paged_attn_decode(&io, &kv, &pg, wp, wb, st, stream), "paged_attn_decode");
  else check_rc(paged_attn_forward(&io, &kv, &pg, wp, wb, st, stream), "paged_attn_forward");
}

std::tuple<at::Tensor, at::Tensor> paged_attention(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V,
                                                   const at::Tensor& q_len, const at::Tensor& block_table,
                                                   const at::Tensor& num_blocks, const at::Tensor& kv_len,
                                                   const std::optional<at::Tensor>& k_scale,
                                                   const std::optional<at::Tensor>& v_scale, bool causal_top_left,
                                                   double softmax_scale, int64_t mode,
                                                   const std::optional<at::Tensor>& status) {
  at::Tensor out = at::empty(Q.sizes(), Q.options().dtype(at::kHalf));
  at::Tensor lse = at::empty(Q.sizes().slice(0, 3), Q.options().dtype(at::kHalf));
  paged_attention_out(Q, K, V, q_len, block_table, num_blocks, kv_len, k_scale, v_scale, causal_top_left,
                      softmax_scale, mode, status, out, lse);
  return {out, lse};
}

void paged_attention_varlen_out(const at::Tensor& Q, const at::Tensor& q_start, const at::Tensor& q_len,
                                int64_t max_q_len, const at::Tensor& K, const at::Tensor& V,
                                const at::Tensor& block_table, const at::Tensor& num_blocks, const at::Tensor& kv_len,
                                const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
                                bool causal_top_left, double softmax_scale, const std::optional<at::Tensor>& status,
                                at::Tensor& out, at::Tensor& lse) {
  check_q(Q, 3);
  check_out(Q, out, lse);
  check_device(Q, K, "K");
  const c10::cuda::CUDAGuard guard(Q.device());
  pa_kv_cache_t kv = kv_desc(K, V, k_scale, v_scale);
  pa_paging_t pg = paging(Q, block_table, num_blocks, q_len, kv_len);
  check_i32(Q, q_start, "q_start", block_table.size(0));
  pa_attn_io_t io = io_desc(Q, out, lse, true, max_q_len, causal_top_left, softmax_scale);
  void* stream = c10::cuda::getCurrentCUDAStream(Q.device().index()).stream();
  size_t bytes = 0;
  check_rc(paged_attn_workspace_size(&io, &kv, &pg, &bytes), "paged_attn_workspace_size");
  at::Tensor ws;
  if (bytes) ws = workspace(Q.device(), bytes);
  check_rc(paged_attn_varlen(&io, &kv, &pg, static_cast<const int32_t*>(q_start.data_ptr()),
                             static_cast<int32_t>(Q.size(0)), bytes ? ws.data_ptr() : nullptr,
                             bytes ? static_cast<size_t>(ws.numel()) : 0, opt_ptr<int32_t>(status), stream),
           "paged_attn_varlen");
}

std::tuple<at::Tensor, at::Tensor> paged_attention_varlen(
    const at::Tensor& Q, const at::Tensor& q_start, const at::Tensor& q_len, int64_t max_q_len, const at::Tensor& K,
    const at::Tensor& V, const at::Tensor& block_table, const at::Tensor& num_blocks, const at::Tensor& kv_len,
    const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale, bool causal_top_left,
    double softmax_scale, const std::optional<at::Tensor>& status) {
  at::Tensor out = at::empty(Q.sizes(), Q.options().dtype(at::kHalf));
  at::Tensor lse = at::empty(Q.sizes().slice(0, 2), Q.options().dtype(at::kHalf));
  paged_attention_varlen_out(Q, q_start, q_len, max_q_len, K, V, block_table, num_blocks, kv_len, k_scale, v_scale,
                             causal_top_left, softmax_scale, status, out, lse);
  return {out, lse};
}

// As the Python front end hands them on: int32, contiguous.
at::Tensor as_i32(const at::Tensor& t) {
  return t.scalar_type() == at::kInt && t.is_contiguous() ? t : t.to(at::kInt).contiguous();
}
at::Tensor flat_i32(const at::Tensor& t) {
  at::Tensor v = as_i32(t);
  return v.dim() == 1 ? v : v.view({-1});
}

void shared_prefix_attention_out(const at::Tensor& Q, const at::Tensor& K, const at::Tensor& V, const at::Tensor& q_len,
                                 const at::Tensor& block_table, const at::Tensor& num_blocks, const at::Tensor& kv_len,
                                 const at::Tensor& group_start, const at::Tensor& prefix_len,
                                 const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
                                 double softmax_scale, const std::optional<at::Tensor>& status, at::Tensor& out,
                                 at::Tensor& lse) {
  check_q(Q, 4);
  check_out(Q, out, lse);
  TORCH_CHECK_VALUE(Q.size(3) < 2 || out.stride(3) == 1, "pie_b200: out needs a contiguous head_dim");
  check_device(Q, K, "K");
  TORCH_CHECK_VALUE(K.dim() == 4 && K.size(3) == Q.size(3), "pie_b200: head_dim of Q and of the pool differ");
  TORCH_CHECK_VALUE(block_table.dim() == 2 && block_table.size(0) == Q.size(0), "pie_b200: block_table needs ", Q.size(0),
                    " rows");
  TORCH_CHECK_VALUE(group_start.numel() >= 1, "pie_b200: group_start holds num_groups + 1 entries");
  const int64_t G = group_start.numel() - 1;
  check_i32(Q, group_start, "group_start", G + 1);
  check_i32(Q, prefix_len, "prefix_len", G);
  check_status(Q, status);
  const c10::cuda::CUDAGuard guard(Q.device());
  pa_kv_cache_t kv = kv_desc(K, V, k_scale, v_scale);
  pa_paging_t pg = paging(Q, block_table, num_blocks, q_len, kv_len);
  pa_attn_io_t io = io_desc(Q, out, lse, false, Q.size(2), false, softmax_scale);
  pa_groups_t gr{};
  gr.group_start = static_cast<const int32_t*>(group_start.data_ptr());
  gr.prefix_len = static_cast<const int32_t*>(prefix_len.data_ptr());
  gr.num_groups = static_cast<int32_t>(G);
  size_t bytes = 0;
  check_rc(shared_prefix_workspace_size(&io, &kv, &pg, &gr, &bytes), "shared_prefix_attn");
  // a workspace of this call's own: calls on other streams and captured graphs do not share it
  at::Tensor ws = fresh({static_cast<int64_t>(bytes > 0 ? bytes : 1)}, at::kByte, Q.device());
  void* stream = c10::cuda::getCurrentCUDAStream(Q.device().index()).stream();
  check_rc(shared_prefix_attn(&io, &kv, &pg, &gr, ws.data_ptr(), bytes, opt_ptr<int32_t>(status), stream),
           "shared_prefix_attn");
}

// Makes O and L, and takes what the Python front end would convert: the whole call without Python's checks (a small
// call is bound by the host: 26 us with them, 14 without).
std::tuple<at::Tensor, at::Tensor> shared_prefix_attention(
    const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& q_len, const at::Tensor& block_table,
    const at::Tensor& num_blocks, int64_t block_size, const at::Tensor& kv_len, const at::Tensor& group_start,
    const at::Tensor& prefix_len, const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
    double softmax_scale, const std::optional<at::Tensor>& status) {
  TORCH_CHECK_VALUE(q.dim() == 4 && k.dim() == 4 && v.dim() == 4,
                    "pie_b200: Q must be [num_seqs, num_q_heads, max_q_len, head_dim], K and V 4-D pools");
  const bool swapped = k.size(1) != block_size && k.size(2) == block_size;
  const at::Tensor K = swapped ? k.transpose(1, 2) : k, V = swapped ? v.transpose(1, 2) : v;
  TORCH_CHECK_VALUE(K.size(1) == block_size, "pie_b200: block_size ", block_size, " does not match the pool");
  const auto small = [](const at::Tensor& t) { return t.scalar_type() == at::kHalf || t.scalar_type() == at::kBFloat16; };
  at::Tensor Q = small(q) ? q : q.to(small(K) ? K.scalar_type() : at::kHalf);
  if (Q.stride(3) != 1) Q = Q.contiguous();
  TORCH_CHECK_VALUE(group_start.dim() == 1 && group_start.numel() >= 1 && prefix_len.dim() == 1,
                    "pie_b200: group_start must hold num_groups + 1 offsets, prefix_len num_groups lengths");
  check_q(Q, 4);
  at::Tensor out = fresh(Q.sizes(), at::kHalf, Q.device()), lse = fresh(Q.sizes().slice(0, 3), at::kHalf, Q.device());
  shared_prefix_attention_out(Q, K, V, as_i32(q_len),
                              block_table.scalar_type() == at::kInt ? block_table : block_table.to(at::kInt),
                              as_i32(num_blocks), as_i32(kv_len), as_i32(group_start), as_i32(prefix_len), k_scale, v_scale,
                              softmax_scale, status, out, lse);
  return {out, lse};
}

void write_kv(const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& block_table,
              const at::Tensor& seq_index, const at::Tensor& positions, at::Tensor& k_cache, at::Tensor& v_cache,
              const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
              const std::optional<at::Tensor>& status) {
  TORCH_CHECK_VALUE(k_new.dim() == 3 && v_new.sizes() == k_new.sizes() && v_new.scalar_type() == k_new.scalar_type(),
              "pie_b200: k_new / v_new must be [num_tokens, num_kv_heads, head_dim] of equal shape and dtype");
  TORCH_CHECK_VALUE(k_new.stride(2) == 1 && v_new.stride(2) == 1, "pie_b200: new rows need a contiguous head_dim");
  check_device(k_cache, k_new, "k_new");
  check_device(k_cache, v_new, "v_new");
  check_device(k_cache, block_table, "block_table");
  TORCH_CHECK_VALUE(block_table.scalar_type() == at::kInt && block_table.dim() == 2, "pie_b200: block_table must be int32 2-D");
  const int64_t T = k_new.size(0);
  check_i32(k_cache, seq_index, "seq_index", T);
  check_i32(k_cache, positions, "positions", T);
  const c10::cuda::CUDAGuard guard(k_cache.device());
  pa_kv_cache_t kv = kv_desc(k_cache, v_cache, k_scale, v_scale);
  pa_paging_t pg{};
  pg.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  pg.bt_stride_seq = block_table.stride(0);
  pg.bt_stride_col = block_table.stride(1);
  pg.bt_cols = static_cast<int32_t>(block_table.size(1));
  pg.num_seqs = static_cast<int32_t>(block_table.size(0));
  pa_kv_new_t nw{};
  nw.k_new = ptr(k_new);
  nw.v_new = ptr(v_new);
  nw.dtype = pa_dtype(k_new.scalar_type());
  nw.num_tokens = static_cast<int32_t>(T);
  nw.k_stride_token = k_new.stride(0);
  nw.k_stride_head = k_new.stride(1);
  nw.v_stride_token = v_new.stride(0);
  nw.v_stride_head = v_new.stride(1);
  nw.seq_index = static_cast<const int32_t*>(seq_index.data_ptr());
  nw.positions = static_cast<const int32_t*>(positions.data_ptr());
  void* stream = c10::cuda::getCurrentCUDAStream(k_cache.device().index()).stream();
  int32_t* st = opt_ptr<int32_t>(status);
  if (kv.dtype == PA_DTYPE_I8) check_rc(kv_write_quant(&nw, &kv, &pg, st, stream), "kv_write_quant");
  else check_rc(kv_write_copy(&nw, &kv, &pg, st, stream), "kv_write_copy");
}

void project_write_kv(const at::Tensor& x, const at::Tensor& w, const std::optional<at::Tensor>& bias,
                      const at::Tensor& block_table, const at::Tensor& seq_index, const at::Tensor& positions,
                      at::Tensor& k_cache, at::Tensor& v_cache, const std::optional<at::Tensor>& k_scale,
                      const std::optional<at::Tensor>& v_scale, const std::optional<at::Tensor>& status) {
  TORCH_CHECK_VALUE(x.dim() == 2 && w.dim() == 2 && x.size(1) == w.size(1) && x.scalar_type() == w.scalar_type(),
                    "pie_b200: x [T, d_model] and w [2 * Hkv * D, d_model] must share d_model and dtype");
  TORCH_CHECK_VALUE(x.stride(1) == 1 && w.stride(1) == 1, "pie_b200: x / w need contiguous rows");
  TORCH_CHECK_VALUE(w.size(0) == 2 * k_cache.size(2) * k_cache.size(3),
                    "pie_b200: w must hold 2 * num_kv_heads * head_dim rows (W_k then W_v)");
  check_device(k_cache, x, "x");
  check_device(k_cache, w, "w");
  check_device(k_cache, block_table, "block_table");
  TORCH_CHECK_VALUE(block_table.scalar_type() == at::kInt && block_table.dim() == 2,
                    "pie_b200: block_table must be int32 2-D");
  const int64_t T = x.size(0);
  check_i32(k_cache, seq_index, "seq_index", T);
  check_i32(k_cache, positions, "positions", T);
  if (bias.has_value()) {
    check_device(k_cache, *bias, "bias");
    TORCH_CHECK_VALUE(bias->scalar_type() == at::kFloat && bias->is_contiguous() && bias->numel() == w.size(0),
                      "pie_b200: bias must be a contiguous float32 vector of w's rows");
  }
  const c10::cuda::CUDAGuard guard(k_cache.device());
  pa_kv_cache_t kv = kv_desc(k_cache, v_cache, k_scale, v_scale);
  pa_paging_t pg{};
  pg.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  pg.bt_stride_seq = block_table.stride(0);
  pg.bt_stride_col = block_table.stride(1);
  pg.bt_cols = static_cast<int32_t>(block_table.size(1));
  pg.num_seqs = static_cast<int32_t>(block_table.size(0));
  pa_kv_proj_t pj{};
  pj.x = ptr(x);
  pj.w = ptr(w);
  pj.bias = bias.has_value() ? static_cast<const float*>(bias->data_ptr()) : nullptr;
  pj.x_stride = x.stride(0);
  pj.w_stride = w.stride(0);
  pj.dtype = pa_dtype(x.scalar_type());
  pj.num_tokens = static_cast<int32_t>(T);
  pj.d_model = static_cast<int32_t>(x.size(1));
  pj.seq_index = static_cast<const int32_t*>(seq_index.data_ptr());
  pj.positions = static_cast<const int32_t*>(positions.data_ptr());
  void* stream = c10::cuda::getCurrentCUDAStream(k_cache.device().index()).stream();
  check_rc(kv_project_write(&pj, &kv, &pg, opt_ptr<int32_t>(status), stream), "kv_project_write");
}

pa_kv_new_t new_rows(const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& seq_index,
                     const at::Tensor& positions) {
  pa_kv_new_t nw{};
  nw.k_new = ptr(k_new);
  nw.v_new = ptr(v_new);
  nw.dtype = pa_dtype(k_new.scalar_type());
  nw.num_tokens = static_cast<int32_t>(k_new.size(0));
  nw.k_stride_token = k_new.stride(0);
  nw.k_stride_head = k_new.stride(1);
  nw.v_stride_token = v_new.stride(0);
  nw.v_stride_head = v_new.stride(1);
  nw.seq_index = static_cast<const int32_t*>(seq_index.data_ptr());
  nw.positions = static_cast<const int32_t*>(positions.data_ptr());
  return nw;
}

void rotate_write_kv_out(const std::optional<at::Tensor>& q, const at::Tensor& k_new, const at::Tensor& v_new,
                         const at::Tensor& cos_sin, bool interleaved, const at::Tensor& block_table,
                         const at::Tensor& seq_index, const at::Tensor& positions, at::Tensor& k_cache, at::Tensor& v_cache,
                         const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
                         const std::optional<at::Tensor>& status, const std::optional<at::Tensor>& q_out) {
  TORCH_CHECK_VALUE(k_new.dim() == 3 && v_new.sizes() == k_new.sizes() && v_new.scalar_type() == k_new.scalar_type(),
                    "pie_b200: k_new / v_new must be [num_tokens, num_kv_heads, head_dim] of equal shape and dtype");
  TORCH_CHECK_VALUE(k_new.stride(2) == 1 && v_new.stride(2) == 1, "pie_b200: new rows need a contiguous head_dim");
  TORCH_CHECK_VALUE(k_cache.dim() == 4 && k_new.size(1) == k_cache.size(2) && k_new.size(2) == k_cache.size(3),
                    "pie_b200: new rows do not match the pool's heads");
  check_device(k_cache, k_new, "k_new");
  check_device(k_cache, v_new, "v_new");
  check_device(k_cache, cos_sin, "cos_sin");
  check_device(k_cache, block_table, "block_table");
  TORCH_CHECK_VALUE(block_table.scalar_type() == at::kInt && block_table.dim() == 2, "pie_b200: block_table must be int32 2-D");
  TORCH_CHECK_VALUE(cos_sin.scalar_type() == at::kFloat && cos_sin.dim() == 2 && cos_sin.stride(1) == 1,
                    "pie_b200: cos_sin must be float32 [num_positions, rot_dim] with contiguous rows");
  const int64_t T = k_new.size(0);
  check_i32(k_cache, seq_index, "seq_index", T);
  check_i32(k_cache, positions, "positions", T);
  check_status(k_cache, status);
  TORCH_CHECK_VALUE(q.has_value() == q_out.has_value(), "pie_b200: q and q_out come together");
  pa_rotate_t r{};
  if (q.has_value()) {
    check_device(k_cache, *q, "q");
    check_device(k_cache, *q_out, "q_out");
    TORCH_CHECK_VALUE(q->dim() == 3 && q->size(0) == T && q->size(2) == k_new.size(2) &&
                          q->scalar_type() == k_new.scalar_type() && q->stride(2) == 1,
                      "pie_b200: q must be [num_tokens, num_q_heads, head_dim] in the new rows' dtype");
    TORCH_CHECK_VALUE(q_out->sizes() == q->sizes() && q_out->scalar_type() == q->scalar_type() && q_out->stride(2) == 1,
                      "pie_b200: q_out must be shaped and typed like q");
    r.q = ptr(*q);
    r.q_out = ptr(*q_out);
    r.q_stride_token = q->stride(0);
    r.q_stride_head = q->stride(1);
    r.qo_stride_token = q_out->stride(0);
    r.qo_stride_head = q_out->stride(1);
    r.num_q_heads = static_cast<int32_t>(q->size(1));
  }
  r.cos_sin = static_cast<const float*>(cos_sin.data_ptr());
  r.cs_stride = cos_sin.size(0) > 1 ? cos_sin.stride(0) : cos_sin.size(1);
  r.rot_dim = static_cast<int32_t>(cos_sin.size(1));
  r.num_positions = static_cast<int32_t>(cos_sin.size(0));
  r.interleaved = interleaved ? 1 : 0;
  const c10::cuda::CUDAGuard guard(k_cache.device());
  pa_kv_cache_t kv = kv_desc(k_cache, v_cache, k_scale, v_scale);
  TORCH_CHECK_VALUE(kv.dtype != PA_DTYPE_I8 || (k_scale->dim() == 3 && v_scale->dim() == 3),
                    "pie_b200: an int8 pool written per token needs per-token scales [NB, BS, H]");
  pa_paging_t pg{};
  pg.block_table = static_cast<const int32_t*>(block_table.data_ptr());
  pg.bt_stride_seq = block_table.stride(0);
  pg.bt_stride_col = block_table.stride(1);
  pg.bt_cols = static_cast<int32_t>(block_table.size(1));
  pg.num_seqs = static_cast<int32_t>(block_table.size(0));
  const pa_kv_new_t nw = new_rows(k_new, v_new, seq_index, positions);
  void* stream = c10::cuda::getCurrentCUDAStream(k_cache.device().index()).stream();
  check_rc(kv_rotate_write(&nw, &r, &kv, &pg, opt_ptr<int32_t>(status), stream), "kv_rotate_write");
}

// Makes the rotated queries, and takes what the Python front end would convert (one token: 17 us a call with its checks,
// 8 without).
at::Tensor rotate_write_kv(const at::Tensor& q, const at::Tensor& k_new, const at::Tensor& v_new, const at::Tensor& cos_sin,
                           bool interleaved, const at::Tensor& block_table, const at::Tensor& seq_index,
                           const at::Tensor& positions, at::Tensor& k_cache, at::Tensor& v_cache,
                           const std::optional<at::Tensor>& k_scale, const std::optional<at::Tensor>& v_scale,
                           const std::optional<at::Tensor>& status) {
  TORCH_CHECK_VALUE(k_new.dim() == 3 && v_new.dim() == 3 && q.dim() == 3 && q.is_cuda(),
                    "pie_b200: q, k_new and v_new must be CUDA tensors [num_tokens, heads, head_dim]");
  TORCH_CHECK_VALUE(k_new.scalar_type() == at::kHalf || k_new.scalar_type() == at::kBFloat16 || k_new.scalar_type() == at::kFloat,
                    "pie_b200: k_new / v_new must share a float16, bfloat16 or float32 dtype");
  TORCH_CHECK_VALUE(cos_sin.dim() == 2 && cos_sin.size(1) >= 16 && cos_sin.size(1) <= k_new.size(2) && cos_sin.size(1) % 16 == 0,
                    "pie_b200: cos_sin must be float32 [num_positions, rot_dim], rot_dim a multiple of 16 up to head_dim");
  const auto rows = [](const at::Tensor& t) { return t.stride(2) == 1 ? t : t.contiguous(); };
  const std::optional<at::Tensor> out = fresh(q.sizes(), q.scalar_type(), q.device());
  rotate_write_kv_out(rows(q), rows(k_new), rows(v_new), cos_sin.stride(1) == 1 ? cos_sin : cos_sin.contiguous(), interleaved,
                      block_table.scalar_type() == at::kInt ? block_table : block_table.to(at::kInt), flat_i32(seq_index),
                      flat_i32(positions), k_cache, v_cache, k_scale, v_scale, status, out);
  return *out;
}

void check_rows(const at::Tensor& ref, const std::optional<at::Tensor>& t, const char* name, at::ScalarType type,
                int64_t rows) {
  if (!t.has_value()) return;
  check_device(ref, *t, name);
  TORCH_CHECK_VALUE(t->scalar_type() == type && t->dim() == 1 && t->is_contiguous() && t->size(0) == rows, "pie_b200: ",
                    name, " must be a contiguous vector of ", rows, type == at::kInt ? " int32" : " float32", " values");
}

void adjust_logits_out(const at::Tensor& logits, const std::optional<at::Tensor>& tokens,
                       const std::optional<at::Tensor>& num_tokens, const std::optional<at::Tensor>& prompt_len,
                       const std::optional<at::Tensor>& repetition, double repetition_value,
                       const std::optional<at::Tensor>& presence, double presence_value,
                       const std::optional<at::Tensor>& frequency, double frequency_value,
                       const std::optional<at::Tensor>& bias, const std::optional<at::Tensor>& bias_row,
                       const std::optional<at::Tensor>& mask, const std::optional<at::Tensor>& mask_row,
                       const std::optional<at::Tensor>& status, at::Tensor& out) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 2 && (logits.size(1) < 2 || logits.stride(1) == 1),
                    "pie_b200: logits must be a CUDA tensor [rows, vocab] with a contiguous vocabulary");
  check_device(logits, out, "out");
  TORCH_CHECK_VALUE(out.sizes() == logits.sizes() && (out.size(1) < 2 || out.stride(1) == 1),
                    "pie_b200: out must be shaped like logits, with a contiguous vocabulary");
  const int64_t R = logits.size(0), V = logits.size(1);
  constexpr int64_t kMost = int64_t{1} << 31;
  TORCH_CHECK_VALUE(R < kMost && V >= 1 && V <= (int64_t{1} << 30), "pie_b200: logits sizes out of range");
  check_rows(logits, num_tokens, "num_tokens", at::kInt, R);
  check_rows(logits, prompt_len, "prompt_len", at::kInt, R);
  check_rows(logits, repetition, "repetition_penalty", at::kFloat, R);
  check_rows(logits, presence, "presence_penalty", at::kFloat, R);
  check_rows(logits, frequency, "frequency_penalty", at::kFloat, R);
  check_rows(logits, bias_row, "bias_row", at::kInt, R);
  check_rows(logits, mask_row, "mask_row", at::kInt, R);
  check_status(logits, status);
  pa_logits_t a{};
  a.logits = logits.data_ptr();
  a.out = out.data_ptr();
  a.stride_row = logits.stride(0);
  a.out_stride_row = out.stride(0);
  a.dtype = pa_dtype(logits.scalar_type());
  a.out_dtype = pa_dtype(out.scalar_type());
  a.rows = static_cast<int32_t>(R);
  a.vocab = static_cast<int32_t>(V);
  if (tokens.has_value()) {
    check_device(logits, *tokens, "tokens");
    TORCH_CHECK_VALUE(tokens->scalar_type() == at::kInt && tokens->dim() == 2 && tokens->size(0) == R &&
                          tokens->size(1) < kMost && (tokens->size(1) < 2 || tokens->stride(1) == 1),
                      "pie_b200: tokens must be int32 [", R, ", max_tokens] with contiguous rows");
    a.tokens = static_cast<const int32_t*>(tokens->data_ptr());
    a.tokens_stride = tokens->stride(0);
    a.max_tokens = static_cast<int32_t>(tokens->size(1));
  }
  a.num_tokens = opt_ptr<const int32_t>(num_tokens);
  a.prompt_len = opt_ptr<const int32_t>(prompt_len);
  a.repetition = opt_ptr<const float>(repetition);
  a.presence = opt_ptr<const float>(presence);
  a.frequency = opt_ptr<const float>(frequency);
  a.repetition_value = static_cast<float>(repetition_value);
  a.presence_value = static_cast<float>(presence_value);
  a.frequency_value = static_cast<float>(frequency_value);
  if (bias.has_value()) {
    check_device(logits, *bias, "bias");
    TORCH_CHECK_VALUE(bias->scalar_type() == at::kFloat && bias->dim() == 2 && bias->size(1) == V && bias->size(0) < kMost &&
                          (V < 2 || bias->stride(1) == 1),
                      "pie_b200: bias must be float32 [bias rows, ", V, "] with contiguous rows");
    a.bias = static_cast<const float*>(bias->data_ptr());
    a.bias_stride = bias->stride(0);
    a.bias_rows = static_cast<int32_t>(bias->size(0));
    a.bias_row = opt_ptr<const int32_t>(bias_row);
  }
  if (mask.has_value()) {
    check_device(logits, *mask, "mask");
    TORCH_CHECK_VALUE(mask->scalar_type() == at::kInt && mask->dim() == 2 && mask->size(1) == (V + 31) / 32 &&
                          mask->size(0) < kMost && (mask->size(1) < 2 || mask->stride(1) == 1),
                      "pie_b200: mask must be int32 [mask rows, ", (V + 31) / 32, "] with contiguous rows");
    a.mask = static_cast<const int32_t*>(mask->data_ptr());
    a.mask_stride = mask->stride(0);
    a.mask_rows = static_cast<int32_t>(mask->size(0));
    a.mask_row = opt_ptr<const int32_t>(mask_row);
  }
  const c10::cuda::CUDAGuard guard(logits.device());
  void* stream = c10::cuda::getCurrentCUDAStream(logits.device().index()).stream();
  check_rc(logits_adjust(&a, opt_ptr<int32_t>(status), stream), "logits_adjust");
}

// Makes the new logits, and takes what the Python front end would convert (one row: 23 us a call with its checks, 8
// without).
at::Tensor adjust_logits(const at::Tensor& logits, const std::optional<at::Tensor>& tokens,
                         const std::optional<at::Tensor>& num_tokens, const std::optional<at::Tensor>& prompt_len,
                         const std::optional<at::Tensor>& repetition, double repetition_value,
                         const std::optional<at::Tensor>& presence, double presence_value,
                         const std::optional<at::Tensor>& frequency, double frequency_value,
                         const std::optional<at::Tensor>& bias, const std::optional<at::Tensor>& bias_row,
                         const std::optional<at::Tensor>& mask, const std::optional<at::Tensor>& mask_row,
                         const std::optional<at::Tensor>& status) {
  const auto type = logits.scalar_type();
  TORCH_CHECK_VALUE(logits.dim() >= 1 && (type == at::kFloat || type == at::kHalf || type == at::kBFloat16) && logits.is_cuda(),
                    "pie_b200: logits must be float32, float16 or bfloat16 [..., vocab] on a CUDA device");
  const int64_t V = logits.size(-1);
  TORCH_CHECK_VALUE(V >= 1, "pie_b200: logits need a vocabulary");
  TORCH_CHECK_VALUE(repetition.has_value() || repetition_value > 0, "pie_b200: repetition_penalty must be positive");
  TORCH_CHECK_VALUE(tokens.has_value() || (!num_tokens.has_value() && !prompt_len.has_value()),
                    "pie_b200: num_tokens and prompt_len come with tokens");
  using Opt = std::optional<at::Tensor>;
  const auto matrix = [](const at::Tensor& t, int64_t cols) {  // [..., cols] as rows
    at::Tensor m = t.dim() == 2 ? t : t.reshape({t.numel() / (cols > 0 ? cols : 1), cols});
    return m.size(1) < 2 || m.stride(1) == 1 ? m : m.contiguous();
  };
  const auto ints = [](const Opt& t) { return t.has_value() ? Opt(flat_i32(*t)) : t; };
  const at::Tensor x = matrix(logits, V);
  const int64_t R = x.size(0);
  const auto values = [R](const Opt& t) {
    if (!t.has_value() || (t->scalar_type() == at::kFloat && t->dim() == 1 && t->is_contiguous())) return t;
    TORCH_CHECK_VALUE(t->numel() == R, "pie_b200: a penalty must be a number or ", R, " values");
    return Opt(t->to(at::kFloat).reshape({R}).contiguous());
  };
  Opt seen = tokens, add = bias, bits = mask;
  if (seen.has_value()) {
    TORCH_CHECK_VALUE(seen->dim() == logits.dim() && seen->sizes().slice(0, seen->dim() - 1) == logits.sizes().slice(0, logits.dim() - 1),
                      "pie_b200: tokens must be shaped like logits, with their own last dimension");
    at::Tensor i = seen->scalar_type() == at::kInt ? *seen : seen->to(at::kInt);
    const int64_t L = i.size(-1);
    if (i.dim() != 2) i = i.reshape({R, L});
    seen = L < 2 || i.stride(1) == 1 ? i : i.contiguous();
  }
  const auto rows_of = [R](const Opt& t, const Opt& by, const char* name) {
    TORCH_CHECK_VALUE(t.has_value() || !by.has_value(), "pie_b200: ", name, "_row without ", name);
    TORCH_CHECK_VALUE(!t.has_value() || by.has_value() || t->size(0) == 1 || t->size(0) == R, "pie_b200: ", name, " has ",
                      t.has_value() ? t->size(0) : 0, " rows for ", R, " rows of logits: pass ", name, "_row");
  };
  if (add.has_value()) {
    at::Tensor b = add->scalar_type() == at::kFloat ? *add : add->to(at::kFloat);
    TORCH_CHECK_VALUE((b.dim() == 1 || b.dim() == 2) && b.size(-1) == V, "pie_b200: bias must be [N, ", V, "] or [", V, "]");
    add = matrix(b, V);
  }
  if (bits.has_value()) {
    const int64_t W = (V + 31) / 32;
    TORCH_CHECK_VALUE((bits->dim() == 1 || bits->dim() == 2) && bits->size(-1) == W && bits->scalar_type() == at::kInt,
                      "pie_b200: mask must be int32 [M, ", W, "] or [", W, "]");
    bits = matrix(*bits, W);
  }
  rows_of(add, bias_row, "bias");
  rows_of(bits, mask_row, "mask");
  at::Tensor out = fresh(logits.sizes(), type, logits.device());
  at::Tensor o = out.dim() == 2 ? out : out.view({R, V});
  adjust_logits_out(x, seen, ints(num_tokens), ints(prompt_len), values(repetition), repetition_value, values(presence),
                    presence_value, values(frequency), frequency_value, add, ints(bias_row), bits, ints(mask_row), status, o);
  return out;
}

// ---- shared blocks, page copies, beams ---------------------------------------
// One descriptor per layer; the scale lists are empty but for int8 pools.
std::vector<pa_kv_cache_t> layer_descs(at::TensorList k, at::TensorList v, at::TensorList ks, at::TensorList vs) {
  TORCH_CHECK_VALUE(!k.empty() && k.size() == v.size(), "pie_b200: as many K as V pools are needed, one at least (got ",
                    k.size(), " and ", v.size(), ")");
  const bool i8 = k[0].scalar_type() == at::kChar;
  TORCH_CHECK_VALUE(!i8 || (ks.size() == k.size() && vs.size() == k.size()),
                    "pie_b200: int8 KV pools need k_scale and v_scale for every layer");
  TORCH_CHECK_VALUE(k[0].is_cuda(), "pie_b200: the pools must be CUDA tensors");
  std::vector<pa_kv_cache_t> d;
  d.reserve(k.size());
  d.push_back(i8 ? kv_desc(k[0], v[0], ks[0], vs[0]) : kv_desc(k[0], v[0], std::nullopt, std::nullopt));
  // further layers: like layer 0 but for their pointers
  const auto like = [](const at::Tensor& a, const at::Tensor& b) {
    return a.scalar_type() == b.scalar_type() && a.device() == b.device() && a.sizes() == b.sizes() &&
           a.strides() == b.strides();
  };
  for (size_t i = 1; i < k.size(); ++i) {
    TORCH_CHECK_VALUE(like(k[i], k[0]) && like(v[i], v[0]) && (!i8 || (like(ks[i], ks[0]) && like(vs[i], vs[0]))),
                      "pie_b200: layer ", i, "'s pools or scales differ from layer 0's in type, device, shape or strides");
    d.push_back(d[0]);
    d[i].k = ptr(k[i]);
    d[i].v = ptr(v[i]);
    if (i8) {
      d[i].k_scale = ptr(ks[i]);
      d[i].v_scale = ptr(vs[i]);
    }
  }
  return d;
}

void copy_blocks(at::TensorList k, at::TensorList v, at::TensorList ks, at::TensorList vs, const at::Tensor& src,
                 const at::Tensor& dst, const std::optional<at::Tensor>& num_slots,
                 const std::optional<at::Tensor>& status) {
  const std::vector<pa_kv_cache_t> d = layer_descs(k, v, ks, vs);
  const int64_t n = src.numel();
  check_i32(k[0], src, "src", n);
  check_i32(k[0], dst, "dst", n);
  if (num_slots.has_value()) check_i32(k[0], *num_slots, "num_slots", n);
  check_status(k[0], status);
  const c10::cuda::CUDAGuard guard(k[0].device());
  void* stream = c10::cuda::getCurrentCUDAStream(k[0].device().index()).stream();
  check_rc(kv_copy_blocks(d.data(), static_cast<int32_t>(d.size()), static_cast<const int32_t*>(src.data_ptr()),
                          static_cast<const int32_t*>(dst.data_ptr()), opt_ptr<const int32_t>(num_slots),
                          static_cast<int32_t>(n), opt_ptr<int32_t>(status), stream),
           "kv_copy_blocks");
}

struct SharedPool {
  pa_block_pool_t pool{};
  pa_block_share_t share{};
};

SharedPool pool_desc(const at::Tensor& ref, const at::Tensor& free_stack, const at::Tensor& free_top,
                     const at::Tensor& table, const at::Tensor& count, const at::Tensor& ref_count,
                     const at::Tensor& scratch) {
  check_vec(ref, free_stack, "free_stack");
  check_vec(ref, free_top, "free_top");
  check_vec(ref, count, "count");
  check_vec(ref, ref_count, "ref_count");
  check_vec(ref, scratch, "scratch");
  check_device(ref, table, "table");
  TORCH_CHECK_VALUE(table.scalar_type() == at::kInt && table.dim() == 2 && (table.size(1) < 2 || table.stride(1) == 1),
                    "pie_b200: table must be int32 [max_seqs, max_blocks_per_seq] with contiguous rows");
  TORCH_CHECK_VALUE(free_top.numel() >= 1 && count.numel() == table.size(0),
                    "pie_b200: count needs one entry per table row, free_top one entry");
  TORCH_CHECK_VALUE(free_stack.numel() >= ref_count.numel(), "pie_b200: free_stack needs an entry per block");
  SharedPool s;
  s.pool.free_stack = static_cast<int32_t*>(free_stack.data_ptr());
  s.pool.free_top = static_cast<int32_t*>(free_top.data_ptr());
  s.pool.table = static_cast<int32_t*>(table.data_ptr());
  s.pool.count = static_cast<int32_t*>(count.data_ptr());
  s.pool.table_stride = table.size(0) > 1 ? table.stride(0) : table.size(1);
  s.pool.num_blocks = static_cast<int32_t>(ref_count.numel());
  s.pool.max_seqs = static_cast<int32_t>(table.size(0));
  s.pool.max_blocks_per_seq = static_cast<int32_t>(table.size(1));
  s.share.ref_count = static_cast<int32_t*>(ref_count.data_ptr());
  s.share.scratch = static_cast<int32_t*>(scratch.data_ptr());
  s.share.scratch_words = scratch.numel();
  return s;
}

at::Tensor reorder_beams(const at::Tensor& free_stack, const at::Tensor& free_top, const at::Tensor& table,
                         const at::Tensor& count, const at::Tensor& ref_count, const at::Tensor& scratch,
                         const at::Tensor& slots, const at::Tensor& parents, const at::Tensor& num_tokens,
                         at::TensorList k, at::TensorList v, at::TensorList ks, at::TensorList vs,
                         const std::optional<at::Tensor>& status) {
  const std::vector<pa_kv_cache_t> d = layer_descs(k, v, ks, vs);
  SharedPool s = pool_desc(k[0], free_stack, free_top, table, count, ref_count, scratch);
  check_vec(k[0], slots, "slots");
  check_vec(k[0], parents, "parents");
  TORCH_CHECK_VALUE(slots.dim() == 2 && parents.sizes() == slots.sizes(),
                    "pie_b200: slots and parents must be [num_groups, num_beams]");
  check_i32(k[0], num_tokens, "num_tokens", slots.size(0));
  check_status(k[0], status);
  const c10::cuda::CUDAGuard guard(k[0].device());
  at::Tensor out = fresh(slots.sizes(), at::kInt, k[0].device());
  void* stream = c10::cuda::getCurrentCUDAStream(k[0].device().index()).stream();
  check_rc(block_pool_reorder(&s.pool, &s.share, static_cast<const int32_t*>(slots.data_ptr()),
                              static_cast<const int32_t*>(parents.data_ptr()),
                              static_cast<const int32_t*>(num_tokens.data_ptr()), static_cast<int32_t>(slots.size(0)),
                              static_cast<int32_t>(slots.size(1)), static_cast<int32_t*>(out.data_ptr()), d.data(),
                              static_cast<int32_t>(d.size()), opt_ptr<int32_t>(status), stream),
           "block_pool_reorder");
  return out;
}

at::Tensor compact_blocks(const at::Tensor& free_stack, const at::Tensor& free_top, const at::Tensor& table,
                          const at::Tensor& count, const at::Tensor& ref_count, const at::Tensor& scratch,
                          int64_t num_blocks_after, at::TensorList k, at::TensorList v, at::TensorList ks,
                          at::TensorList vs, const std::optional<at::Tensor>& status) {
  const std::vector<pa_kv_cache_t> d = layer_descs(k, v, ks, vs);
  SharedPool s = pool_desc(k[0], free_stack, free_top, table, count, ref_count, scratch);
  check_status(k[0], status);
  TORCH_CHECK_VALUE(num_blocks_after <= s.pool.num_blocks, "pie_b200: num_blocks ", num_blocks_after, " exceeds the pool's ",
                    s.pool.num_blocks);
  const c10::cuda::CUDAGuard guard(k[0].device());
  at::Tensor live = fresh({1}, at::kInt, k[0].device());
  void* stream = c10::cuda::getCurrentCUDAStream(k[0].device().index()).stream();
  check_rc(block_pool_compact(&s.pool, &s.share,
                              num_blocks_after < 0 ? s.pool.num_blocks : static_cast<int32_t>(num_blocks_after),
                              static_cast<int32_t*>(live.data_ptr()), d.data(), static_cast<int32_t>(d.size()),
                              opt_ptr<int32_t>(status), stream),
           "block_pool_compact");
  return live;
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> beam_select_op(const at::Tensor& logits, const at::Tensor& scores,
                                                              int64_t num_out,
                                                              const std::optional<at::Tensor>& finished,
                                                              int64_t eos_id) {
  TORCH_CHECK_VALUE(logits.is_cuda() && logits.dim() == 3 && (logits.size(2) < 2 || logits.stride(2) == 1),
                    "pie_b200: logits must be a CUDA tensor [num_seqs, num_beams, vocab] with a contiguous vocabulary");
  check_device(logits, scores, "beam_scores");
  TORCH_CHECK_VALUE(scores.scalar_type() == at::kFloat && scores.is_contiguous() && scores.dim() == 2 &&
                        scores.size(0) == logits.size(0) && scores.size(1) == logits.size(1),
                    "pie_b200: beam_scores must be contiguous float32 [num_seqs, num_beams]");
  if (finished.has_value()) {
    check_device(logits, *finished, "finished");
    TORCH_CHECK_VALUE((finished->scalar_type() == at::kBool || finished->scalar_type() == at::kByte) &&
                          finished->is_contiguous() && finished->sizes() == scores.sizes(),
                      "pie_b200: finished must be contiguous bool [num_seqs, num_beams]");
  }
  const c10::cuda::CUDAGuard guard(logits.device());
  pa_beam_select_t a{};
  a.logits = logits.data_ptr();
  a.scores = static_cast<const float*>(scores.data_ptr());
  a.finished = opt_ptr<const uint8_t>(finished);
  a.stride_seq = logits.stride(0);
  a.stride_beam = logits.stride(1);
  a.dtype = pa_dtype(logits.scalar_type());
  TORCH_CHECK_VALUE(logits.size(2) >= 1 && logits.size(2) < (int64_t{1} << 31) && logits.size(0) < (int64_t{1} << 31) &&
                        logits.size(1) < (int64_t{1} << 31) && num_out < (int64_t{1} << 31) && eos_id < (int64_t{1} << 31),
                    "pie_b200: beam_select sizes out of range");
  a.num_seqs = static_cast<int32_t>(logits.size(0));
  a.num_beams = static_cast<int32_t>(logits.size(1));
  a.vocab = static_cast<int32_t>(logits.size(2));
  a.eos_id = static_cast<int32_t>(eos_id);
  a.num_out = static_cast<int32_t>(num_out);
  size_t bytes = 0;
  check_rc(beam_select_workspace_size(&a, &bytes), "beam_select");
  // a workspace of this call's own: calls on other streams and captured graphs do not share it
  at::Tensor ws = fresh({static_cast<int64_t>(bytes > 0 ? bytes : 1)}, at::kByte, logits.device());
  // three tensors of their own, as the schema says: compiled code takes them to start on 16 bytes, and two types
  // over one storage could not be saved together
  std::tuple<at::Tensor, at::Tensor, at::Tensor> out{fresh({logits.size(0), num_out}, at::kFloat, logits.device()),
                                                     fresh({logits.size(0), num_out}, at::kInt, logits.device()),
                                                     fresh({logits.size(0), num_out}, at::kInt, logits.device())};
  a.out_scores = static_cast<float*>(std::get<0>(out).data_ptr());
  a.out_tokens = static_cast<int32_t*>(std::get<1>(out).data_ptr());
  a.out_parents = static_cast<int32_t*>(std::get<2>(out).data_ptr());
  void* stream = c10::cuda::getCurrentCUDAStream(logits.device().index()).stream();
  check_rc(beam_select(&a, ws.data_ptr(), bytes, stream), "beam_select");
  return out;
}

// ---- shapes only (fake / meta tensors) ------------------------------------
// Of every op that writes into its arguments and returns nothing.
void write_only_meta(const c10::OperatorHandle& op, c10::DispatchKeySet, torch::jit::Stack* stack) {
  torch::jit::drop(*stack, op.schema().arguments().size());
}

at::Tensor reorder_beams_meta(const at::Tensor&, const at::Tensor&, const at::Tensor&, const at::Tensor&,
                              const at::Tensor&, const at::Tensor&, const at::Tensor& slots, const at::Tensor&,
                              const at::Tensor&, at::TensorList, at::TensorList, at::TensorList, at::TensorList,
                              const std::optional<at::Tensor>&) {
  return at::empty(slots.sizes(), slots.options());
}

at::Tensor compact_blocks_meta(const at::Tensor&, const at::Tensor& free_top, const at::Tensor&, const at::Tensor&,
                               const at::Tensor&, const at::Tensor&, int64_t, at::TensorList, at::TensorList,
                               at::TensorList, at::TensorList, const std::optional<at::Tensor>&) {
  return at::empty({1}, free_top.options());
}

std::tuple<at::Tensor, at::Tensor, at::Tensor> beam_select_meta(const at::Tensor&, const at::Tensor& scores,
                                                                int64_t num_out, const std::optional<at::Tensor>&,
                                                                int64_t) {
  const auto i32 = scores.options().dtype(at::kInt);
  const int64_t B = scores.size(0);
  return {at::empty({B, num_out}, scores.options()), at::empty({B, num_out}, i32), at::empty({B, num_out}, i32)};
}

std::tuple<at::Tensor, at::Tensor> paged_attention_meta(const at::Tensor& Q, const at::Tensor&, const at::Tensor&,
                                                        const at::Tensor&, const at::Tensor&, const at::Tensor&,
                                                        const at::Tensor&, const std::optional<at::Tensor>&,
                                                        const std::optional<at::Tensor>&, bool, double, int64_t,
                                                        const std::optional<at::Tensor>&) {
  return {at::empty(Q.sizes(), Q.options().dtype(at::kHalf)),
          at::empty(Q.sizes().slice(0, 3), Q.options().dtype(at::kHalf))};
}

using Opt = std::optional<at::Tensor>;
std::tuple<at::Tensor, at::Tensor> shared_prefix_meta(const at::Tensor& Q, const at::Tensor&, const at::Tensor&,
                                                      const at::Tensor&, const at::Tensor&, const at::Tensor&, int64_t,
                                                      const at::Tensor&, const at::Tensor&, const at::Tensor&, const Opt&,
                                                      const Opt&, double, const Opt&) {
  return {at::empty_symint(Q.sym_sizes(), Q.options().dtype(at::kHalf)),
          at::empty_symint(Q.sym_sizes().slice(0, 3), Q.options().dtype(at::kHalf))};
}

at::Tensor rotate_write_meta(const at::Tensor& q, const at::Tensor&, const at::Tensor&, const at::Tensor&, bool,
                             const at::Tensor&, const at::Tensor&, const at::Tensor&, at::Tensor&, at::Tensor&, const Opt&,
                             const Opt&, const Opt&) {
  return at::empty_symint(q.sym_sizes(), q.options());
}

at::Tensor adjust_logits_meta(const at::Tensor& logits, const Opt&, const Opt&, const Opt&, const Opt&, double, const Opt&,
                              double, const Opt&, double, const Opt&, const Opt&, const Opt&, const Opt&, const Opt&) {
  return at::empty_symint(logits.sym_sizes(), logits.options());
}

std::tuple<at::Tensor, at::Tensor> paged_attention_varlen_meta(
    const at::Tensor& Q, const at::Tensor&, const at::Tensor&, int64_t, const at::Tensor&, const at::Tensor&,
    const at::Tensor&, const at::Tensor&, const at::Tensor&, const std::optional<at::Tensor>&,
    const std::optional<at::Tensor>&, bool, double, const std::optional<at::Tensor>&) {
  return {at::empty(Q.sizes(), Q.options().dtype(at::kHalf)),
          at::empty(Q.sizes().slice(0, 2), Q.options().dtype(at::kHalf))};
}

}  // namespace

TORCH_LIBRARY(pie_b200, m) {
  m.def("paged_attention(Tensor Q, Tensor K, Tensor V, Tensor q_len, Tensor block_table, Tensor num_blocks, "
        "Tensor kv_len, Tensor? k_scale, Tensor? v_scale, bool causal_top_left, float softmax_scale, int mode, "
        "Tensor(s!)? status) -> (Tensor, Tensor)");
  m.def("paged_attention_out(Tensor Q, Tensor K, Tensor V, Tensor q_len, Tensor block_table, Tensor num_blocks, "
        "Tensor kv_len, Tensor? k_scale, Tensor? v_scale, bool causal_top_left, float softmax_scale, int mode, "
        "Tensor(s!)? status, Tensor(a!) out, Tensor(b!) lse) -> ()");
  m.def("paged_attention_varlen(Tensor Q, Tensor q_start, Tensor q_len, int max_q_len, Tensor K, Tensor V, "
        "Tensor block_table, Tensor num_blocks, Tensor kv_len, Tensor? k_scale, Tensor? v_scale, "
        "bool causal_top_left, float softmax_scale, Tensor(s!)? status) -> (Tensor, Tensor)");
  m.def("paged_attention_varlen_out(Tensor Q, Tensor q_start, Tensor q_len, int max_q_len, Tensor K, Tensor V, "
        "Tensor block_table, Tensor num_blocks, Tensor kv_len, Tensor? k_scale, Tensor? v_scale, "
        "bool causal_top_left, float softmax_scale, Tensor(s!)? status, Tensor(a!) out, Tensor(b!) lse) -> ()");
  m.def("write_kv(Tensor k_new, Tensor v_new, Tensor block_table, Tensor seq_index, Tensor positions, "
        "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale, Tensor(d!)? v_scale, Tensor(s!)? status) -> ()");
  m.def("project_write_kv(Tensor x, Tensor w, Tensor? bias, Tensor block_table, Tensor seq_index, Tensor positions, "
        "Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale, Tensor(d!)? v_scale, Tensor(s!)? status) -> ()");
  m.def("shared_prefix_attention(Tensor Q, Tensor K, Tensor V, Tensor q_len, Tensor block_table, Tensor num_blocks, "
        "int block_size, Tensor kv_len, Tensor group_start, Tensor prefix_len, Tensor? k_scale, Tensor? v_scale, "
        "float softmax_scale, Tensor(s!)? status) -> (Tensor, Tensor)");
  m.def("shared_prefix_attention_out(Tensor Q, Tensor K, Tensor V, Tensor q_len, Tensor block_table, Tensor num_blocks, "
        "Tensor kv_len, Tensor group_start, Tensor prefix_len, Tensor? k_scale, Tensor? v_scale, float softmax_scale, "
        "Tensor(s!)? status, Tensor(a!) out, Tensor(b!) lse) -> ()");
  m.def("rotate_write_kv(Tensor q, Tensor k_new, Tensor v_new, Tensor cos_sin, bool interleaved, Tensor block_table, "
        "Tensor seq_index, Tensor positions, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale, "
        "Tensor(d!)? v_scale, Tensor(s!)? status) -> Tensor");
  m.def("rotate_write_kv_out(Tensor? q, Tensor k_new, Tensor v_new, Tensor cos_sin, bool interleaved, Tensor block_table, "
        "Tensor seq_index, Tensor positions, Tensor(a!) k_cache, Tensor(b!) v_cache, Tensor(c!)? k_scale, "
        "Tensor(d!)? v_scale, Tensor(s!)? status, Tensor(e!)? q_out) -> ()");
  m.def("adjust_logits(Tensor logits, Tensor? tokens, Tensor? num_tokens, Tensor? prompt_len, Tensor? repetition, "
        "float repetition_value, Tensor? presence, float presence_value, Tensor? frequency, float frequency_value, "
        "Tensor? bias, Tensor? bias_row, Tensor? mask, Tensor? mask_row, Tensor(s!)? status) -> Tensor");
  m.def("adjust_logits_out(Tensor logits, Tensor? tokens, Tensor? num_tokens, Tensor? prompt_len, Tensor? repetition, "
        "float repetition_value, Tensor? presence, float presence_value, Tensor? frequency, float frequency_value, "
        "Tensor? bias, Tensor? bias_row, Tensor? mask, Tensor? mask_row, Tensor(s!)? status, Tensor(a!) out) -> ()");
  m.def("copy_blocks(Tensor(a!)[] k_caches, Tensor(b!)[] v_caches, Tensor(c!)[] k_scales, Tensor(d!)[] v_scales, "
        "Tensor src, Tensor dst, Tensor? num_slots, Tensor(s!)? status) -> ()");
  m.def("reorder_beams(Tensor(a!) free_stack, Tensor(b!) free_top, Tensor(c!) table, Tensor(d!) count, "
        "Tensor(e!) ref_count, Tensor(f!) scratch, Tensor slots, Tensor parents, Tensor num_tokens, "
        "Tensor(g!)[] k_caches, Tensor(h!)[] v_caches, Tensor(i!)[] k_scales, Tensor(j!)[] v_scales, "
        "Tensor(s!)? status) -> Tensor");
  m.def("compact_blocks(Tensor(a!) free_stack, Tensor(b!) free_top, Tensor(c!) table, Tensor(d!) count, "
        "Tensor(e!) ref_count, Tensor(f!) scratch, int num_blocks_after, Tensor(g!)[] k_caches, "
        "Tensor(h!)[] v_caches, Tensor(i!)[] k_scales, Tensor(j!)[] v_scales, Tensor(s!)? status) -> Tensor");
  m.def("beam_select(Tensor logits, Tensor beam_scores, int num_out, Tensor? finished, int eos_id) -> "
        "(Tensor, Tensor, Tensor)");
}

TORCH_LIBRARY_IMPL(pie_b200, CUDA, m) {
  m.impl("paged_attention", &paged_attention);
  m.impl("paged_attention_out", &paged_attention_out);
  m.impl("paged_attention_varlen", &paged_attention_varlen);
  m.impl("paged_attention_varlen_out", &paged_attention_varlen_out);
  m.impl("write_kv", &write_kv);
  m.impl("project_write_kv", &project_write_kv);
  m.impl("shared_prefix_attention", &shared_prefix_attention);
  m.impl("shared_prefix_attention_out", &shared_prefix_attention_out);
  m.impl("rotate_write_kv", &rotate_write_kv);
  m.impl("rotate_write_kv_out", &rotate_write_kv_out);
  m.impl("adjust_logits", &adjust_logits);
  m.impl("adjust_logits_out", &adjust_logits_out);
  m.impl("copy_blocks", &copy_blocks);
  m.impl("reorder_beams", &reorder_beams);
  m.impl("compact_blocks", &compact_blocks);
  m.impl("beam_select", &beam_select_op);
}

TORCH_LIBRARY_IMPL(pie_b200, Meta, m) {
  m.impl("paged_attention", &paged_attention_meta);
  m.impl("paged_attention_varlen", &paged_attention_varlen_meta);
  m.impl("reorder_beams", &reorder_beams_meta);
  m.impl("compact_blocks", &compact_blocks_meta);
  m.impl("beam_select", &beam_select_meta);
  m.impl("shared_prefix_attention", &shared_prefix_meta);
  m.impl("rotate_write_kv", &rotate_write_meta);
  m.impl("adjust_logits", &adjust_logits_meta);
  for (const char* op : {"paged_attention_out", "paged_attention_varlen_out", "write_kv", "project_write_kv",
                         "shared_prefix_attention_out", "rotate_write_kv_out", "adjust_logits_out", "copy_blocks"})
    m.impl(op, torch::CppFunction::makeFromBoxedFunction<&write_only_meta>());
}
