"""Torch-tensor front end of the C ABI: argument checks, then the registered torch ops.

All tensors live on one CUDA device; every launch goes to torch's current
stream on that device, so calls compose with torch ops and CUDA graphs.
Nothing here computes on the host and there is no fallback path: a missing
library or a non-CUDA tensor raises.

The calls go through the torch.library ops of the extension
(``torch.ops.pie_b200.*``, csrc/torch_ops.cpp), which fill the C structs and
call libpaged_attn_b200.so in C++.  ``PIE_B200_BACKEND=ctypes`` routes the
same calls through the ctypes binding of the C ABI instead (``_lib``): the
two paths launch the same kernels with the same arguments.
"""
from __future__ import annotations

import ctypes
import math
import os
from typing import NamedTuple, Optional, Sequence, Union

import torch

from . import _lib
from ._lib import PaAttnIO, PaKvCache, PaKvNew, PaPaging

_TORCH2PA = {
    torch.float16: _lib.PA_DTYPE_F16,
    torch.bfloat16: _lib.PA_DTYPE_BF16,
    torch.int8: _lib.PA_DTYPE_I8,
    torch.float32: _lib.PA_DTYPE_F32,
}

_CHECK = os.environ.get("PIE_B200_CHECK", "0") not in ("", "0")
BACKEND = os.environ.get("PIE_B200_BACKEND", "torch")
if BACKEND not in ("torch", "ctypes"):
    raise ValueError(f"PIE_B200_BACKEND must be 'torch' or 'ctypes', not {BACKEND!r}")
_MODES = {"auto": 0, "decode": 1, "prefill": 2}


def _torch_ops():
    from . import _torch_ext

    return _torch_ext.ops()


_OPS: dict = {}


def _op(name: str):
    """The registered op's default overload, looked up once (a direct call skips the packet dispatch)."""
    op = _OPS.get(name)
    if op is None:
        op = getattr(_torch_ops(), name).default
        _OPS[name] = op
    return op


def _out_and_lse(shape: tuple, device) -> tuple[torch.Tensor, torch.Tensor]:
    """O (shape) and LSE (shape without head_dim), float16, from one allocation (O first, 256-byte aligned)."""
    n_o = math.prod(shape)
    buf = torch.empty(n_o + math.prod(shape[:-1]), dtype=torch.float16, device=device)
    return buf[:n_o].view(shape), buf[n_o:].view(shape[:-1])


def _i32(t: torch.Tensor) -> torch.Tensor:
    if t.dtype == torch.int32 and t.is_contiguous():
        return t
    return t.to(torch.int32).contiguous()


def _ptr(t: Optional[torch.Tensor]) -> Optional[int]:
    return None if t is None else t.data_ptr()


def kv_cache_desc(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                  v_scale: Optional[torch.Tensor] = None) -> PaKvCache:
    """Descriptor of a pool whose dims are read as [block, slot, head, d].

    Scales: [num_blocks, num_kv_heads] (one per block and head, the reference
    layout) or [num_blocks, block_size, num_kv_heads] (one per token and head).
    """
    check_cache(k_cache, v_cache, k_scale, v_scale)
    nb, bs, h, d = k_cache.shape
    kc = PaKvCache()
    kc.k = k_cache.data_ptr()
    kc.v = v_cache.data_ptr()
    kc.dtype = _TORCH2PA[k_cache.dtype]
    kc.num_blocks, kc.block_size, kc.num_kv_heads, kc.head_dim = nb, bs, h, d
    kc.k_stride_block, kc.k_stride_slot, kc.k_stride_head = k_cache.stride(0), k_cache.stride(1), k_cache.stride(2)
    kc.v_stride_block, kc.v_stride_slot, kc.v_stride_head = v_cache.stride(0), v_cache.stride(1), v_cache.stride(2)
    kc.scale_dtype = _lib.PA_DTYPE_F16
    if k_cache.dtype == torch.int8:
        kc.scale_dtype = _TORCH2PA[k_scale.dtype]
        kc.k_scale = k_scale.data_ptr()
        kc.v_scale = v_scale.data_ptr()
        kc.ks_stride_block, kc.ks_stride_slot, kc.ks_stride_head = _scale_strides(k_scale, nb, bs, h)
        kc.vs_stride_block, kc.vs_stride_slot, kc.vs_stride_head = _scale_strides(v_scale, nb, bs, h)
    return kc


def check_cache(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                v_scale: Optional[torch.Tensor] = None) -> None:
    """Raise ValueError unless the pools (and an INT8 pool's scales) are well formed."""
    if k_cache.dim() != 4 or v_cache.dim() != 4:
        raise ValueError("K/V pools must be 4-D [num_blocks, block_size, num_kv_heads, head_dim]")
    if k_cache.shape != v_cache.shape or k_cache.dtype != v_cache.dtype:
        raise ValueError(f"K and V pools differ: {tuple(k_cache.shape)}/{k_cache.dtype} vs "
                         f"{tuple(v_cache.shape)}/{v_cache.dtype}")
    if k_cache.dtype not in (torch.float16, torch.bfloat16, torch.int8, torch.float32):
        raise ValueError(f"KV pool dtype {k_cache.dtype} unsupported (float16, bfloat16, int8 or float32)")
    if k_cache.stride(3) != 1 or v_cache.stride(3) != 1:
        raise ValueError("KV pools need a contiguous head_dim")
    nb, bs, h, d = k_cache.shape
    if k_cache.dtype == torch.int8:
        if k_scale is None or v_scale is None:
            raise ValueError("an int8 KV pool needs k_scale and v_scale")
        for name, s in (("k_scale", k_scale), ("v_scale", v_scale)):
            if s.dtype not in (torch.float16, torch.float32):
                raise ValueError(f"{name} must be float16 or float32, got {s.dtype}")
            if s.device != k_cache.device:
                raise ValueError(f"{name} is on {s.device}, the pool on {k_cache.device}")
        if k_scale.dtype != v_scale.dtype:
            raise ValueError("k_scale and v_scale dtypes differ")
        _scale_strides(k_scale, nb, bs, h)
        _scale_strides(v_scale, nb, bs, h)


def _scale_strides(s: torch.Tensor, nb: int, bs: int, h: int) -> tuple[int, int, int]:
    if s.dim() == 2:
        if tuple(s.shape) != (nb, h):
            raise ValueError(f"per-block scales must be [{nb}, {h}], got {tuple(s.shape)}")
        return s.stride(0), 0, s.stride(1)
    if s.dim() == 3:
        if tuple(s.shape) != (nb, bs, h):
            raise ValueError(f"per-token scales must be [{nb}, {bs}, {h}], got {tuple(s.shape)}")
        return s.stride(0), s.stride(1), s.stride(2)
    raise ValueError("scales must be 2-D [NB, H] or 3-D [NB, BS, H]")


def pool_layout(K: torch.Tensor, V: torch.Tensor, block_size: int) -> tuple[torch.Tensor, torch.Tensor]:
    """The pools as [block, slot, head, d] views.

    The reference launcher reads dims 1 and 2 as (slot, head)
    (kernels/flash_attention.py:158-159) while the reference model allocates
    its caches as [num_blocks, heads, block_size, d_k]
    (transformer/model.py:64-65) and passes them unchanged
    (transformer/model.py:156-160).  A pool whose dim 1 is not ``block_size``
    but whose dim 2 is can only be the model's layout, so it is read through
    the transposed view; a pool that fits the launcher's layout is read as is.
    """
    if K.dim() == 4 and K.shape[1] != block_size and K.shape[2] == block_size:
        return K.transpose(1, 2), V.transpose(1, 2)
    return K, V


def _paging_tensors(block_table: torch.Tensor, num_blocks: torch.Tensor, q_len: torch.Tensor,
                    kv_len: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, torch.Tensor]:
    """int32 block table (any strides) and contiguous int32 metadata with one entry per sequence."""
    bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    if bt.dim() != 2:
        raise ValueError("block_table must be 2-D [num_seqs, max_blocks]")
    nbk, ql, kl = _i32(num_blocks), _i32(q_len), _i32(kv_len)
    for name, t in (("num_blocks_per_seq", nbk), ("q_len_per_seq", ql), ("kv_len_per_seq", kl)):
        if t.numel() != bt.shape[0]:
            raise ValueError(f"{name} has {t.numel()} entries for {bt.shape[0]} sequences")
    return bt, nbk, ql, kl


def paging_desc(block_table: torch.Tensor, num_blocks: torch.Tensor, q_len: torch.Tensor,
                kv_len: torch.Tensor, keep: list) -> PaPaging:
    bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    if bt.dim() != 2:
        raise ValueError("block_table must be 2-D [num_seqs, max_blocks]")
    nbk, ql, kl = _i32(num_blocks), _i32(q_len), _i32(kv_len)
    keep.extend((bt, nbk, ql, kl))
    pg = PaPaging()
    pg.block_table = bt.data_ptr()
    pg.bt_stride_seq, pg.bt_stride_col = bt.stride(0), bt.stride(1)
    pg.bt_cols = bt.shape[1]
    pg.num_seqs = bt.shape[0]
    pg.num_blocks_per_seq, pg.q_len_per_seq, pg.kv_len_per_seq = nbk.data_ptr(), ql.data_ptr(), kl.data_ptr()
    for name, t in (("num_blocks_per_seq", nbk), ("q_len_per_seq", ql), ("kv_len_per_seq", kl)):
        if t.numel() != pg.num_seqs:
            raise ValueError(f"{name} has {t.numel()} entries for {pg.num_seqs} sequences")
    return pg


_workspaces: dict[int, torch.Tensor] = {}
_status: dict[int, torch.Tensor] = {}


def workspace(device: torch.device, nbytes: int) -> torch.Tensor:
    """Per-device split-K workspace, grown on demand (256-byte aligned)."""
    idx = device.index if device.index is not None else torch.cuda.current_device()
    ws = _workspaces.get(idx)
    if ws is None or ws.numel() < nbytes:
        ws = torch.empty(max(nbytes, 1 << 20), dtype=torch.uint8, device=device)
        _workspaces[idx] = ws
    return ws


def status_word(device: torch.device) -> torch.Tensor:
    idx = device.index if device.index is not None else torch.cuda.current_device()
    st = _status.get(idx)
    if st is None:
        st = torch.zeros(1, dtype=torch.int32, device=device)
        _status[idx] = st
    return st


def _raise_status(fn: str, st: torch.Tensor) -> None:
    v = int(st.item())
    if v:
        st.zero_()
        _raise_status_value(fn, v)


def _raise_status_value(fn: str, v: int) -> None:
    """Raise IndexError naming the bits of a nonzero device status word."""
    if v:
        bits = []
        if v & _lib.PA_STATUS_BAD_BLOCK_ID:
            bits.append("block id outside the pool")
        if v & _lib.PA_STATUS_BAD_POSITION:
            bits.append("position beyond the block table")
        if v & _lib.PA_STATUS_BAD_NUM_BLOCKS:
            bits.append("num_blocks_per_seq wider than the block table")
        if v & _lib.PA_STATUS_BAD_SEQ_INDEX:
            bits.append("sequence index outside the block table")
        if v & _lib.PA_STATUS_WAIT_TIMEOUT:
            bits.append("a wait inside a kernel gave up")
        if v & _lib.PA_STATUS_PEER_TIMEOUT:
            bits.append("a peer GPU never reached the output-exchange barrier")
        if v & _lib.PA_STATUS_COPY_OVERLAP:
            bits.append("a page copy into another copy's source or target")
        if v & _lib.PA_STATUS_BAD_POOL:
            bits.append("block pool arrays that contradict each other, or more blocks in use than may stay")
        raise IndexError(f"{fn}: device status {v:#x}: " + "; ".join(bits))


def paged_attention(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, q_len_per_seq: torch.Tensor,
                    block_table: torch.Tensor, num_blocks_per_seq: torch.Tensor, block_size: int,
                    kv_len_per_seq: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                    v_scale: Optional[torch.Tensor] = None, *, out: Optional[torch.Tensor] = None,
                    lse: Optional[torch.Tensor] = None, causal_top_left: bool = False,
                    softmax_scale: Optional[float] = None, mode: str = "auto",
                    status: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Paged causal attention through the C ABI; returns (O fp16, L fp16)."""
    if Q.dim() != 4:
        raise ValueError("Q must be [num_seqs, num_q_heads, max_q_len, head_dim]")
    B, Hq, maxq, D = Q.shape
    K, V = pool_layout(K, V, block_size)
    if K.shape[1] != block_size:
        raise ValueError(f"block_size {block_size} does not match the pool's slot dimension {K.shape[1]}")
    if K.shape[3] != D:
        raise ValueError(f"head_dim of Q ({D}) and of the pool ({K.shape[3]}) differ")
    if block_table.shape[0] != B:
        raise ValueError(f"block_table has {block_table.shape[0]} rows for {B} sequences")
    dev = Q.device
    if Q.dtype not in (torch.float16, torch.bfloat16):
        Q = Q.to(K.dtype if K.dtype in (torch.float16, torch.bfloat16) else torch.float16)
    if Q.stride(3) != 1:
        Q = Q.contiguous()
    if mode not in _MODES:
        raise ValueError(f"mode must be one of {sorted(_MODES)}, not {mode!r}")
    if out is None and lse is None:
        out, lse = _out_and_lse((B, Hq, maxq, D), dev)
    if out is None:
        out = torch.empty((B, Hq, maxq, D), dtype=torch.float16, device=dev)
    elif out.dtype != torch.float16 or tuple(out.shape) != (B, Hq, maxq, D):
        raise ValueError("out must be float16 with Q's shape")
    if lse is None:
        lse = torch.empty((B, Hq, maxq), dtype=torch.float16, device=dev)
    if status is None and _CHECK:
        status = status_word(dev)
    if BACKEND == "torch":
        # pools, scales, devices and metadata lengths are checked by the op (ValueError)
        bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
        _op("paged_attention_out")(Q, K, V, _i32(q_len_per_seq), bt, _i32(num_blocks_per_seq),
                                   _i32(kv_len_per_seq), k_scale, v_scale, bool(causal_top_left),
                                   float(softmax_scale) if softmax_scale else 0.0, _MODES[mode], status, out, lse)
        if _CHECK and status is not None:
            _raise_status("paged_attention", status)
        return out, lse
    for name, t in (("K", K), ("V", V), ("block_table", block_table), ("q_len_per_seq", q_len_per_seq),
                    ("kv_len_per_seq", kv_len_per_seq), ("num_blocks_per_seq", num_blocks_per_seq)):
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, Q on {dev}")
    keep: list = []
    kc = kv_cache_desc(K, V, k_scale, v_scale)
    pg = paging_desc(block_table, num_blocks_per_seq, q_len_per_seq, kv_len_per_seq, keep)
    io = PaAttnIO()
    io.q = Q.data_ptr()
    io.q_dtype = _TORCH2PA[Q.dtype]
    io.num_q_heads, io.max_q_len = Hq, maxq
    io.causal_top_left = 1 if causal_top_left else 0
    io.q_stride_seq, io.q_stride_head, io.q_stride_row = Q.stride(0), Q.stride(1), Q.stride(2)
    io.o = out.data_ptr()
    io.o_stride_seq, io.o_stride_head, io.o_stride_row = out.stride(0), out.stride(1), out.stride(2)
    io.lse = lse.data_ptr()
    io.l_stride_seq, io.l_stride_head, io.l_stride_row = lse.stride(0), lse.stride(1), lse.stride(2)
    io.softmax_scale = float(softmax_scale) if softmax_scale else 0.0

    lib = _lib.load()
    stream = torch.cuda.current_stream(dev).cuda_stream
    st_ptr = _ptr(status)
    with torch.cuda.device(dev):
        if mode == "prefill":
            _lib.check("paged_attn_prefill", lib.paged_attn_prefill(io, kc, pg, st_ptr, stream))
        else:
            nbytes = ctypes.c_size_t(0)
            _lib.check("paged_attn_workspace_size", lib.paged_attn_workspace_size(io, kc, pg, ctypes.byref(nbytes)))
            ws = workspace(dev, nbytes.value) if nbytes.value else None
            fn = lib.paged_attn_decode if mode == "decode" else lib.paged_attn_forward
            _lib.check(fn.__name__, fn(io, kc, pg, _ptr(ws), 0 if ws is None else ws.numel(), st_ptr, stream))
    if _CHECK and status is not None:
        _raise_status("paged_attention", status)
    return out, lse


def paged_attention_varlen(Q: torch.Tensor, cu_seqlens_q: torch.Tensor, K: torch.Tensor, V: torch.Tensor,
                           block_table: torch.Tensor, num_blocks_per_seq: torch.Tensor, block_size: int,
                           kv_len_per_seq: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                           v_scale: Optional[torch.Tensor] = None, *, max_q_len: Optional[int] = None,
                           out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                           causal_top_left: bool = False, softmax_scale: Optional[float] = None,
                           status: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """Paged causal attention over ragged query rows through paged_attn_varlen.

    Q is ``[T, Hq, D]`` with the rows of sequence b at
    ``cu_seqlens_q[b] : cu_seqlens_q[b + 1]``; returns O ``[T, Hq, D]`` and L
    ``[T, Hq]`` (fp16).  ``max_q_len`` (the longest sequence's row count) sizes
    the grid; without it one host read of ``cu_seqlens_q`` finds it.
    """
    if Q.dim() != 3:
        raise ValueError("Q must be [total_q_rows, num_q_heads, head_dim]")
    T, Hq, D = Q.shape
    B = block_table.shape[0]
    if cu_seqlens_q.dim() != 1 or cu_seqlens_q.shape[0] != B + 1:
        raise ValueError(f"cu_seqlens_q must hold {B + 1} offsets for {B} sequences")
    K, V = pool_layout(K, V, block_size)
    if K.shape[1] != block_size:
        raise ValueError(f"block_size {block_size} does not match the pool's slot dimension {K.shape[1]}")
    if K.shape[3] != D:
        raise ValueError(f"head_dim of Q ({D}) and of the pool ({K.shape[3]}) differ")
    dev = Q.device
    for name, t in (("K", K), ("V", V), ("block_table", block_table), ("cu_seqlens_q", cu_seqlens_q),
                    ("kv_len_per_seq", kv_len_per_seq), ("num_blocks_per_seq", num_blocks_per_seq)):
        if t.device != dev:
            raise ValueError(f"{name} is on {t.device}, Q on {dev}")
    cu = _i32(cu_seqlens_q)
    q_start = cu[:-1]
    q_len = (cu[1:] - cu[:-1]).contiguous()
    if max_q_len is None:
        max_q_len = int(q_len.max().item()) if B else 0
    mma_dtype = K.dtype if K.dtype in (torch.float16, torch.bfloat16) else torch.float16
    if Q.dtype not in (torch.float16, torch.bfloat16):
        Q = Q.to(mma_dtype)
    if Q.stride(2) != 1:
        Q = Q.contiguous()
    if out is None:
        out = torch.empty((T, Hq, D), dtype=torch.float16, device=dev)
    elif out.dtype != torch.float16 or tuple(out.shape) != (T, Hq, D):
        raise ValueError("out must be float16 with Q's shape")
    if lse is None:
        lse = torch.empty((T, Hq), dtype=torch.float16, device=dev)
    if status is None and _CHECK:
        status = status_word(dev)
    if BACKEND == "torch":
        check_cache(K, V, k_scale, v_scale)
        bt, nbk, ql, kl = _paging_tensors(block_table, num_blocks_per_seq, q_len, kv_len_per_seq)
        if T:
            _op("paged_attention_varlen_out")(Q, q_start, ql, int(max_q_len), K, V, bt, nbk, kl, k_scale,
                                                    v_scale, bool(causal_top_left),
                                                    float(softmax_scale) if softmax_scale else 0.0, status, out, lse)
        if _CHECK and status is not None:
            _raise_status("paged_attention_varlen", status)
        return out, lse
    keep: list = [cu, q_len]
    kc = kv_cache_desc(K, V, k_scale, v_scale)
    pg = paging_desc(block_table, num_blocks_per_seq, q_len, kv_len_per_seq, keep)
    io = PaAttnIO()
    io.q = Q.data_ptr()
    io.q_dtype = _TORCH2PA[Q.dtype]
    io.num_q_heads, io.max_q_len = Hq, int(max_q_len)
    io.causal_top_left = 1 if causal_top_left else 0
    io.q_stride_seq, io.q_stride_head, io.q_stride_row = 0, Q.stride(1), Q.stride(0)
    io.o = out.data_ptr()
    io.o_stride_seq, io.o_stride_head, io.o_stride_row = 0, out.stride(1), out.stride(0)
    io.lse = lse.data_ptr()
    io.l_stride_seq, io.l_stride_head, io.l_stride_row = 0, lse.stride(1), lse.stride(0)
    io.softmax_scale = float(softmax_scale) if softmax_scale else 0.0

    lib = _lib.load()
    stream = torch.cuda.current_stream(dev).cuda_stream
    st_ptr = _ptr(status)
    with torch.cuda.device(dev):
        nbytes = ctypes.c_size_t(0)
        _lib.check("paged_attn_workspace_size", lib.paged_attn_workspace_size(io, kc, pg, ctypes.byref(nbytes)))
        ws = workspace(dev, nbytes.value) if nbytes.value else None
        _lib.check("paged_attn_varlen", lib.paged_attn_varlen(io, kc, pg, q_start.data_ptr(), T, _ptr(ws),
                                                              0 if ws is None else ws.numel(), st_ptr, stream))
    if _CHECK and status is not None:
        _raise_status("paged_attention_varlen", status)
    return out, lse


def shared_prefix_attention(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, q_len_per_seq: torch.Tensor,
                            block_table: torch.Tensor, num_blocks_per_seq: torch.Tensor, block_size: int,
                            kv_len_per_seq: torch.Tensor, group_start: torch.Tensor, prefix_len: torch.Tensor,
                            k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, *,
                            out: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                            softmax_scale: Optional[float] = None,
                            status: Optional[torch.Tensor] = None) -> tuple[torch.Tensor, torch.Tensor]:
    """``paged_attention`` of decode rows where groups of sequences share a prefix, read once a group; (O, L) fp16.

    Sequences ``group_start[g] .. group_start[g + 1] - 1`` (int32 [G + 1], on the device, rising) form group g; their
    block tables name the same blocks for the first ``prefix_len[g]`` tokens (int32 [G]; cut to whole blocks, and to
    what every row sees).  ``DeviceBlockManager.shared_prefixes`` and ``BeamSearch.step_inputs`` give both.  At most
    16 query rows times heads of a KV head (``max_q_len * Hq / Hkv``); fp16, bf16 and int8 pools.
    """
    if BACKEND == "torch" and Q.is_cuda and out is None and lse is None and not _CHECK:  # the op checks and makes them
        return _op("shared_prefix_attention")(Q, K, V, q_len_per_seq, block_table, num_blocks_per_seq, block_size,
                                              kv_len_per_seq, group_start, prefix_len, k_scale, v_scale,
                                              softmax_scale or 0.0, status)
    if Q.dim() != 4:
        raise ValueError("Q must be [num_seqs, num_q_heads, max_q_len, head_dim]")
    B, Hq, maxq, D = Q.shape
    K, V = pool_layout(K, V, block_size)
    if K.dim() != 4 or K.shape[1] != block_size:
        raise ValueError(f"block_size {block_size} does not match the pool {tuple(K.shape)}")
    if K.shape[3] != D:
        raise ValueError(f"head_dim of Q ({D}) and of the pool ({K.shape[3]}) differ")
    if block_table.dim() != 2 or block_table.shape[0] != B:
        raise ValueError(f"block_table must be [{B}, max_blocks]")
    if group_start.dim() != 1 or group_start.numel() < 1 or tuple(prefix_len.shape) != (group_start.numel() - 1,):
        raise ValueError("group_start must hold num_groups + 1 offsets, prefix_len num_groups lengths")
    dev = Q.device
    if Q.dtype not in (torch.float16, torch.bfloat16):
        Q = Q.to(K.dtype if K.dtype in (torch.float16, torch.bfloat16) else torch.float16)
    if Q.stride(3) != 1:
        Q = Q.contiguous()
    if out is None and lse is None:
        out, lse = _out_and_lse((B, Hq, maxq, D), dev)
    if out is None:
        out = torch.empty((B, Hq, maxq, D), dtype=torch.float16, device=dev)
    elif out.dtype != torch.float16 or tuple(out.shape) != (B, Hq, maxq, D) or (D > 1 and out.stride(3) != 1):
        raise ValueError("out must be float16 with Q's shape and a contiguous head_dim")
    if lse is None:
        lse = torch.empty((B, Hq, maxq), dtype=torch.float16, device=dev)
    elif lse.dtype != torch.float16 or tuple(lse.shape) != (B, Hq, maxq):
        raise ValueError("lse must be float16 with Q's shape without head_dim")
    if status is None and _CHECK:
        status = status_word(dev)
    gs, pl = _i32(group_start), _i32(prefix_len)
    scale = float(softmax_scale) if softmax_scale else 0.0
    if BACKEND == "torch":
        bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
        _op("shared_prefix_attention_out")(Q, K, V, _i32(q_len_per_seq), bt, _i32(num_blocks_per_seq), _i32(kv_len_per_seq), gs,
                                                           pl, k_scale, v_scale, scale, status, out, lse)
    else:
        for name, t in (("K", K), ("V", V), ("block_table", block_table), ("q_len_per_seq", q_len_per_seq),
                        ("kv_len_per_seq", kv_len_per_seq), ("num_blocks_per_seq", num_blocks_per_seq),
                        ("group_start", gs), ("prefix_len", pl), ("out", out), ("lse", lse)):
            if t.device != dev:
                raise ValueError(f"{name} is on {t.device}, Q on {dev}")
        keep: list = []
        kc = kv_cache_desc(K, V, k_scale, v_scale)
        pg = paging_desc(block_table, num_blocks_per_seq, q_len_per_seq, kv_len_per_seq, keep)
        io = PaAttnIO()
        io.q, io.q_dtype, io.num_q_heads, io.max_q_len = Q.data_ptr(), _TORCH2PA[Q.dtype], Hq, maxq
        io.q_stride_seq, io.q_stride_head, io.q_stride_row = Q.stride(0), Q.stride(1), Q.stride(2)
        io.o = out.data_ptr()
        io.o_stride_seq, io.o_stride_head, io.o_stride_row = out.stride(0), out.stride(1), out.stride(2)
        io.lse = lse.data_ptr()
        io.l_stride_seq, io.l_stride_head, io.l_stride_row = lse.stride(0), lse.stride(1), lse.stride(2)
        io.softmax_scale = scale
        gr = _lib.PaGroups(gs.data_ptr(), pl.data_ptr(), pl.numel(), 0)
        lib = _lib.load()
        with torch.cuda.device(dev):
            nbytes = ctypes.c_size_t(0)
            _lib.check("shared_prefix_attn", lib.shared_prefix_workspace_size(io, kc, pg, gr, ctypes.byref(nbytes)))
            ws = torch.empty(max(1, nbytes.value), dtype=torch.uint8, device=dev)
            _lib.check("shared_prefix_attn", lib.shared_prefix_attn(io, kc, pg, gr, ws.data_ptr(), nbytes.value, _ptr(status),
                                                                    _stream(dev)))
    if _CHECK and status is not None:
        _raise_status("shared_prefix_attention", status)
    return out, lse


def paged_attention_peers(Q: torch.Tensor, K: torch.Tensor, V: torch.Tensor, q_len_per_seq: torch.Tensor,
                          block_table: torch.Tensor, num_blocks_per_seq: torch.Tensor, block_size: int,
                          kv_len_per_seq: torch.Tensor, k_scale: Optional[torch.Tensor], v_scale: Optional[torch.Tensor],
                          out: torch.Tensor, out_peer_ptrs: list[int], *,
                          status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Decode whose O rows go to every GPU of a peer exchange (paged_attn_decode_peers).

    ``out`` is this GPU's view of the destination (it fixes the layout);
    ``out_peer_ptrs[r]`` is the address of the same element 0 in GPU r's
    mapped buffer.  Returns the local LSE [B, Hq, q] (fp16).
    """
    B, Hq, maxq, D = Q.shape
    dev = Q.device
    if Q.stride(3) != 1:
        Q = Q.contiguous()
    keep: list = []
    kc = kv_cache_desc(K, V, k_scale, v_scale)
    pg = paging_desc(block_table, num_blocks_per_seq, q_len_per_seq, kv_len_per_seq, keep)
    if out.dtype != torch.float16 or tuple(out.shape) != (B, Hq, maxq, D):
        raise ValueError("out must be float16 with Q's shape")
    lse = torch.empty((B, Hq, maxq), dtype=torch.float16, device=dev)
    io = PaAttnIO()
    io.q = Q.data_ptr()
    io.q_dtype = _TORCH2PA[Q.dtype]
    io.num_q_heads, io.max_q_len = Hq, maxq
    io.q_stride_seq, io.q_stride_head, io.q_stride_row = Q.stride(0), Q.stride(1), Q.stride(2)
    io.o = out.data_ptr()
    io.o_stride_seq, io.o_stride_head, io.o_stride_row = out.stride(0), out.stride(1), out.stride(2)
    io.lse = lse.data_ptr()
    io.l_stride_seq, io.l_stride_head, io.l_stride_row = lse.stride(0), lse.stride(1), lse.stride(2)
    lib = _lib.load()
    stream = torch.cuda.current_stream(dev).cuda_stream
    if status is None and _CHECK:
        status = status_word(dev)
    peers = (ctypes.c_void_p * len(out_peer_ptrs))(*out_peer_ptrs)
    with torch.cuda.device(dev):
        nbytes = ctypes.c_size_t(0)
        _lib.check("paged_attn_workspace_size", lib.paged_attn_workspace_size(io, kc, pg, ctypes.byref(nbytes)))
        ws = workspace(dev, nbytes.value) if nbytes.value else None
        _lib.check("paged_attn_decode_peers",
                   lib.paged_attn_decode_peers(io, kc, pg, _ptr(ws), 0 if ws is None else ws.numel(), peers,
                                               len(out_peer_ptrs), _ptr(status), stream))
    if _CHECK and status is not None:
        _raise_status("paged_attention_peers", status)
    return lse


def write_kv(k_new: torch.Tensor, v_new: torch.Tensor, block_table: torch.Tensor, seq_index: torch.Tensor,
             positions: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
             k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, *,
             status: Optional[torch.Tensor] = None) -> None:
    """Append new rows [T, Hkv, D] at (seq_index[t], positions[t]) of the pool."""
    if k_new.dim() != 3 or v_new.shape != k_new.shape:
        raise ValueError("k_new / v_new must be [num_tokens, num_kv_heads, head_dim] of equal shape")
    T, H, D = k_new.shape
    if (H, D) != (k_cache.shape[2], k_cache.shape[3]):
        raise ValueError(f"new rows [*, {H}, {D}] do not match the pool [*, *, {k_cache.shape[2]}, {k_cache.shape[3]}]")
    if k_new.dtype not in (torch.float16, torch.bfloat16, torch.float32) or v_new.dtype != k_new.dtype:
        raise ValueError("k_new / v_new must share a float16, bfloat16 or float32 dtype")
    dev = k_cache.device
    if k_new.stride(2) != 1:
        k_new = k_new.contiguous()
    if v_new.stride(2) != 1:
        v_new = v_new.contiguous()
    if k_cache.dtype == torch.int8 and (k_scale is None or k_scale.dim() != 3):
        raise ValueError("quantise-on-write stores one scale per (token, head): scales must be [NB, BS, H]")
    if BACKEND != "torch":
        check_cache(k_cache, v_cache, k_scale, v_scale)  # the op checks them itself
    bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    si, ps = _i32(seq_index), _i32(positions)
    if si.numel() != T or ps.numel() != T:
        raise ValueError("seq_index / positions need one entry per token")
    if status is None and _CHECK:
        status = status_word(dev)
    if BACKEND == "torch":
        if bt.dim() != 2:
            raise ValueError("block_table must be 2-D [num_seqs, max_blocks]")
        _op("write_kv")(k_new, v_new, bt, si, ps, k_cache, v_cache, k_scale if k_cache.dtype == torch.int8 else None,
                        v_scale if k_cache.dtype == torch.int8 else None, status)
        if _CHECK and status is not None:
            _raise_status("write_kv_cache", status)
        return
    keep: list = []
    kc = kv_cache_desc(k_cache, v_cache, k_scale, v_scale)
    keep.extend((bt, si, ps))
    pg = _lib.PaPaging()
    pg.block_table = bt.data_ptr()
    pg.bt_stride_seq, pg.bt_stride_col = bt.stride(0), bt.stride(1)
    pg.bt_cols, pg.num_seqs = bt.shape[1], bt.shape[0]
    nw = PaKvNew()
    nw.k_new, nw.v_new = k_new.data_ptr(), v_new.data_ptr()
    nw.dtype = _TORCH2PA[k_new.dtype]
    nw.num_tokens = T
    nw.k_stride_token, nw.k_stride_head = k_new.stride(0), k_new.stride(1)
    nw.v_stride_token, nw.v_stride_head = v_new.stride(0), v_new.stride(1)
    nw.seq_index, nw.positions = si.data_ptr(), ps.data_ptr()
    lib = _lib.load()
    stream = torch.cuda.current_stream(dev).cuda_stream
    with torch.cuda.device(dev):
        if k_cache.dtype == torch.int8:
            _lib.check("kv_write_quant", lib.kv_write_quant(nw, kc, pg, _ptr(status), stream))
        else:
            _lib.check("kv_write_copy", lib.kv_write_copy(nw, kc, pg, _ptr(status), stream))
    if _CHECK and status is not None:
        _raise_status("write_kv_cache", status)


def project_write_kv(x: torch.Tensor, w_kv: torch.Tensor, bias: Optional[torch.Tensor], block_table: torch.Tensor,
                     seq_index: torch.Tensor, positions: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                     k_scale: Optional[torch.Tensor] = None, v_scale: Optional[torch.Tensor] = None, *,
                     status: Optional[torch.Tensor] = None) -> None:
    """K/V projection of x [T, d_model] with the cache write in its epilogue (kv_project_write).

    ``w_kv`` is [W_k; W_v] ([2 * Hkv * D, d_model], nn.Linear's weight layout)
    and ``bias`` the matching float32 [2 * Hkv * D] (or None): token t's K
    row of head h is ``x[t] @ W_k[h*D:(h+1)*D].T + b_k[h*D:(h+1)*D]``, written
    at (seq_index[t], positions[t]) of the pool like ``write_kv`` writes it.
    """
    if x.dim() != 2 or w_kv.dim() != 2 or x.shape[1] != w_kv.shape[1]:
        raise ValueError("x must be [T, d_model] and w_kv [2 * Hkv * D, d_model]")
    if x.dtype not in (torch.float16, torch.bfloat16) or w_kv.dtype != x.dtype:
        raise ValueError("x and w_kv must share a float16 or bfloat16 dtype")
    if k_cache.dtype == torch.int8 and (k_scale is None or k_scale.dim() != 3):
        raise ValueError("an int8 pool written per token needs per-token scales [NB, BS, H]")
    if w_kv.shape[0] != 2 * k_cache.shape[2] * k_cache.shape[3]:
        raise ValueError(f"w_kv has {w_kv.shape[0]} rows; the pool needs 2 * {k_cache.shape[2]} * {k_cache.shape[3]}")
    if seq_index.numel() != x.shape[0] or positions.numel() != x.shape[0]:
        raise ValueError("seq_index / positions need one entry per token")
    if x.stride(1) != 1:
        x = x.contiguous()
    if w_kv.stride(1) != 1:
        w_kv = w_kv.contiguous()
    dev = k_cache.device
    if bias is not None and (bias.dtype != torch.float32 or not bias.is_contiguous()):
        bias = bias.to(torch.float32).contiguous()
    bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    si, ps = _i32(seq_index), _i32(positions)
    if status is None and _CHECK:
        status = status_word(dev)
    int8 = k_cache.dtype == torch.int8
    if BACKEND == "torch":
        _op("project_write_kv")(x, w_kv, bias, bt, si, ps, k_cache, v_cache, k_scale if int8 else None,
                                v_scale if int8 else None, status)
    else:
        kc = kv_cache_desc(k_cache, v_cache, k_scale, v_scale)
        pg = _lib.PaPaging()
        pg.block_table = bt.data_ptr()
        pg.bt_stride_seq, pg.bt_stride_col = bt.stride(0), bt.stride(1)
        pg.bt_cols, pg.num_seqs = bt.shape[1], bt.shape[0]
        pj = _lib.PaKvProj()
        pj.x, pj.w = x.data_ptr(), w_kv.data_ptr()
        pj.bias = None if bias is None else bias.data_ptr()
        pj.x_stride, pj.w_stride = x.stride(0), w_kv.stride(0)
        pj.dtype = _TORCH2PA[x.dtype]
        pj.num_tokens, pj.d_model = x.shape[0], x.shape[1]
        pj.seq_index, pj.positions = si.data_ptr(), ps.data_ptr()
        lib = _lib.load()
        with torch.cuda.device(dev):
            _lib.check("kv_project_write", lib.kv_project_write(pj, kc, pg, _ptr(status),
                                                                torch.cuda.current_stream(dev).cuda_stream))
    if _CHECK and status is not None:
        _raise_status("project_write_kv", status)


def rope_table(num_positions: int, rot_dim: int, base: float = 10000.0, *, scaling: float = 1.0,
               device: torch.device | str = "cuda") -> torch.Tensor:
    """cos and sin of every position's angles, float32 [num_positions, rot_dim], for ``rotate_write_kv``.

    Pair i of position p turns by ``p / scaling * base ** (-2 i / rot_dim)`` (cos of the pairs, then sin; computed
    in 64 bits).  Any table of this layout will do: other schemes fill it themselves.
    """
    if rot_dim < 2 or rot_dim % 2 or num_positions < 0:
        raise ValueError(f"rot_dim {rot_dim} must be even and positive, num_positions {num_positions} >= 0")
    freq = float(base) ** (-torch.arange(0, rot_dim, 2, dtype=torch.float64) / rot_dim)
    angle = (torch.arange(num_positions, dtype=torch.float64) / scaling)[:, None] * freq
    return torch.cat([angle.cos(), angle.sin()], 1).float().to(device)


def rotate_write_kv(q: Optional[torch.Tensor], k_new: torch.Tensor, v_new: torch.Tensor, cos_sin: torch.Tensor,
                    block_table: torch.Tensor, seq_index: torch.Tensor, positions: torch.Tensor,
                    k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: Optional[torch.Tensor] = None,
                    v_scale: Optional[torch.Tensor] = None, *, interleaved: bool = False,
                    q_out: Optional[torch.Tensor] = None,
                    status: Optional[torch.Tensor] = None) -> Optional[torch.Tensor]:
    """``write_kv`` of keys rotated by their positions; returns ``q`` [T, Hq, D] rotated (None without q).

    ``cos_sin`` float32 [num_positions, rot_dim]: cos of each position's rot_dim / 2 pairs, then sin
    (``rope_table``).  Pairs are the dims i and i + rot_dim / 2, or with ``interleaved`` 2i and 2i + 1; dims from
    rot_dim on stay.  ``q``, ``k_new`` and ``v_new`` share a dtype; ``q_out`` may be ``q``.  A token whose position is
    outside ``cos_sin`` is left out (its row of the result too); see kv_rotate_write in the C header.
    """
    if BACKEND == "torch" and k_cache.is_cuda and q is not None and q_out is None and not _CHECK:  # the op checks
        return _op("rotate_write_kv")(q, k_new, v_new, cos_sin, interleaved, block_table, seq_index, positions, k_cache,
                                      v_cache, k_scale, v_scale, status)
    if k_new.dim() != 3 or v_new.shape != k_new.shape:
        raise ValueError("k_new / v_new must be [num_tokens, num_kv_heads, head_dim] of equal shape")
    T, H, D = k_new.shape
    if k_cache.dim() != 4 or (H, D) != (k_cache.shape[2], k_cache.shape[3]):
        raise ValueError(f"new rows [*, {H}, {D}] do not match the pool {tuple(k_cache.shape)}")
    if k_new.dtype not in (torch.float16, torch.bfloat16, torch.float32) or v_new.dtype != k_new.dtype:
        raise ValueError("k_new / v_new must share a float16, bfloat16 or float32 dtype")
    if cos_sin.dim() != 2 or cos_sin.dtype != torch.float32:
        raise ValueError("cos_sin must be float32 [num_positions, rot_dim]")
    if not 16 <= cos_sin.shape[1] <= D or cos_sin.shape[1] % 16:
        raise ValueError(f"rot_dim {cos_sin.shape[1]} must be a multiple of 16 up to head_dim {D}")
    if k_cache.dtype == torch.int8 and (k_scale is None or v_scale is None or k_scale.dim() != 3 or v_scale.dim() != 3):
        raise ValueError("quantise-on-write stores one scale per (token, head): scales must be [NB, BS, H]")
    if k_new.stride(2) != 1:
        k_new = k_new.contiguous()
    if v_new.stride(2) != 1:
        v_new = v_new.contiguous()
    if cos_sin.stride(1) != 1:
        cos_sin = cos_sin.contiguous()
    if q is None:
        if q_out is not None:
            raise ValueError("q_out without q")
    else:
        if q.dim() != 3 or q.shape[0] != T or q.shape[2] != D or q.dtype != k_new.dtype:
            raise ValueError(f"q must be [{T}, num_q_heads, {D}] in {k_new.dtype}")
        if q.stride(2) != 1:
            q = q.contiguous()
        if q_out is None:
            q_out = torch.empty(q.shape, dtype=q.dtype, device=q.device)
        elif q_out.shape != q.shape or q_out.dtype != q.dtype or q_out.stride(2) != 1:
            raise ValueError("q_out must be shaped and typed like q, with a contiguous head_dim")
    bt = block_table if block_table.dtype == torch.int32 else block_table.to(torch.int32)
    si, ps = _i32(seq_index), _i32(positions)
    if bt.dim() != 2 or si.numel() != T or ps.numel() != T:
        raise ValueError("block_table must be 2-D [num_seqs, max_blocks]; seq_index / positions need one entry per token")
    if status is None and _CHECK:
        status = status_word(k_cache.device)
    int8 = k_cache.dtype == torch.int8
    if BACKEND == "torch":
        _op("rotate_write_kv_out")(q, k_new, v_new, cos_sin, bool(interleaved), bt, si.view(-1), ps.view(-1), k_cache, v_cache,
                                   k_scale if int8 else None, v_scale if int8 else None, status, q_out)
    else:
        dev = k_cache.device
        for name, t in (("q", q), ("q_out", q_out), ("k_new", k_new), ("v_new", v_new), ("v_cache", v_cache),
                        ("cos_sin", cos_sin), ("block_table", bt), ("seq_index", si), ("positions", ps)):
            if t is not None and t.device != dev:
                raise ValueError(f"{name} is on {t.device}, the pool on {dev}")
        kc = kv_cache_desc(k_cache, v_cache, k_scale, v_scale)
        pg = _lib.PaPaging()
        pg.block_table = bt.data_ptr()
        pg.bt_stride_seq, pg.bt_stride_col = bt.stride(0), bt.stride(1)
        pg.bt_cols, pg.num_seqs = bt.shape[1], bt.shape[0]
        nw = PaKvNew()
        nw.k_new, nw.v_new = k_new.data_ptr(), v_new.data_ptr()
        nw.dtype, nw.num_tokens = _TORCH2PA[k_new.dtype], T
        nw.k_stride_token, nw.k_stride_head = k_new.stride(0), k_new.stride(1)
        nw.v_stride_token, nw.v_stride_head = v_new.stride(0), v_new.stride(1)
        nw.seq_index, nw.positions = si.data_ptr(), ps.data_ptr()
        r = _lib.PaRotate()
        if q is not None:
            r.q, r.q_out, r.num_q_heads = q.data_ptr(), q_out.data_ptr(), q.shape[1]
            r.q_stride_token, r.q_stride_head = q.stride(0), q.stride(1)
            r.qo_stride_token, r.qo_stride_head = q_out.stride(0), q_out.stride(1)
        r.cos_sin, r.num_positions, r.rot_dim = cos_sin.data_ptr(), cos_sin.shape[0], cos_sin.shape[1]
        r.cs_stride = cos_sin.stride(0) if cos_sin.shape[0] > 1 else cos_sin.shape[1]
        r.interleaved = int(bool(interleaved))
        with torch.cuda.device(dev):
            _lib.check("kv_rotate_write", _lib.load().kv_rotate_write(nw, r, kc, pg, _ptr(status), _stream(dev)))
    if _CHECK and status is not None:
        _raise_status("rotate_write_kv", status)
    return q_out


class PoolState(NamedTuple):
    """The device arrays of a block pool whose blocks sequences share (all int32, see pa_block_share_t).

    ``free_stack`` [num_blocks], ``free_top`` [1], ``table`` [max_seqs, max_blocks_per_seq], ``count`` [max_seqs]
    (-1: no entry), ``ref_count`` [num_blocks] holders of each block, ``scratch`` (``pool_scratch_words`` words,
    zero before its first use).
    """

    free_stack: torch.Tensor
    free_top: torch.Tensor
    table: torch.Tensor
    count: torch.Tensor
    ref_count: torch.Tensor
    scratch: torch.Tensor


def pool_scratch_words(num_blocks: int) -> int:
    """Words of a PoolState's ``scratch``: 16 + 3 * num_blocks + ceil(num_blocks / 32)."""
    return 16 + 3 * num_blocks + (num_blocks + 31) // 32


Caches = Union[torch.Tensor, Sequence[torch.Tensor]]


def _layers(t: Optional[Caches]) -> Sequence[torch.Tensor]:
    return () if t is None else (t,) if isinstance(t, torch.Tensor) else t


def layer_descs(k_cache: Caches, v_cache: Caches, k_scale: Optional[Caches] = None,
                v_scale: Optional[Caches] = None) -> ctypes.Array:
    """One descriptor per layer; layers differ in their pointers only."""
    k, v, ks, vs = _layers(k_cache), _layers(v_cache), _layers(k_scale), _layers(v_scale)
    if not k or len(k) != len(v):
        raise ValueError(f"as many K as V pools are needed, one at least (got {len(k)} and {len(v)})")
    if k[0].dtype == torch.int8 and not len(k) == len(ks) == len(vs):
        raise ValueError("int8 KV pools need k_scale and v_scale for every layer")
    if any(t.device != k[0].device for t in (*k, *v, *ks, *vs)):
        raise ValueError("the pools and scales of all layers must be on one device")
    descs = (PaKvCache * len(k))()
    for i in range(len(k)):
        if k[i].dtype == torch.int8:
            descs[i] = kv_cache_desc(k[i], v[i], ks[i], vs[i])
        else:
            descs[i] = kv_cache_desc(k[i], v[i])
    return descs


def _check_vectors(device: torch.device, **tensors: Optional[torch.Tensor]) -> None:
    for name, t in tensors.items():
        if t is None:
            continue
        if t.device != device:
            raise ValueError(f"{name} must be on {device}, got {t.device}")
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError(f"{name} must be contiguous int32")


def _stream(device: torch.device) -> int:
    return torch.cuda.current_stream(device).cuda_stream


def _copy_call(descs, dev: torch.device, src: torch.Tensor, dst: torch.Tensor, num_slots: Optional[torch.Tensor],
               status: Optional[torch.Tensor]) -> None:
    _check_vectors(dev, src=src, dst=dst, num_slots=num_slots, status=status)
    with torch.cuda.device(dev):
        _lib.check("kv_copy_blocks", _lib.load().kv_copy_blocks(
            descs, len(descs), src.data_ptr(), dst.data_ptr(), _ptr(num_slots), src.numel(), _ptr(status), _stream(dev)))


def copy_blocks(k_cache: Caches, v_cache: Caches, src: torch.Tensor, dst: torch.Tensor,
                k_scale: Optional[Caches] = None, v_scale: Optional[Caches] = None, *,
                num_slots: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> None:
    """Copy block ``src[i]`` to ``dst[i]`` in the pools of one layer (tensors) or of all layers (lists).

    ``src`` / ``dst`` int32 [n] on the device; ``num_slots`` int32 [n] copies only the first slots of each block.
    The copies act at once: a pair whose target another pair reads, or an earlier pair writes, is skipped (and
    reported in ``status``), as is one with an id outside the pool.
    """
    k, v = _layers(k_cache), _layers(v_cache)
    src, dst = _i32(src), _i32(dst)
    if num_slots is not None:
        num_slots = _i32(num_slots)
    if not k:
        raise ValueError("as many K as V pools are needed, one at least (got none)")
    if src.dim() != 1 or dst.shape != src.shape or (num_slots is not None and num_slots.shape != src.shape):
        raise ValueError("src, dst and num_slots must be vectors of one length")
    if BACKEND == "torch" and not _CHECK:  # the op checks the rest
        _op("copy_blocks")(k, v, _layers(k_scale), _layers(v_scale), src, dst, num_slots, status)
        return
    dev = k[0].device
    if status is None and _CHECK:
        status = status_word(dev)
    if BACKEND == "torch":
        _op("copy_blocks")(k, v, _layers(k_scale), _layers(v_scale), src, dst, num_slots, status)
    else:
        _copy_call(layer_descs(k_cache, v_cache, k_scale, v_scale), dev, src, dst, num_slots, status)
    if _CHECK and status is not None:
        _raise_status("copy_blocks", status)


def pool_descs(pool: PoolState):
    """The C descriptors (pa_block_pool_t, pa_block_share_t) of a pool's arrays."""
    from .block_pool import PaBlockPool

    dev = pool.ref_count.device
    _check_vectors(dev, free_stack=pool.free_stack, free_top=pool.free_top, count=pool.count, ref_count=pool.ref_count,
                   scratch=pool.scratch)
    t = pool.table
    if t.device != dev or t.dtype != torch.int32 or t.dim() != 2 or (t.shape[1] > 1 and t.stride(1) != 1):
        raise ValueError("table must be int32 [max_seqs, max_blocks_per_seq] with contiguous rows")
    if pool.count.numel() != t.shape[0] or pool.free_top.numel() < 1:
        raise ValueError("count needs one entry per table row, free_top one entry")
    if pool.free_stack.numel() < pool.ref_count.numel():
        raise ValueError("free_stack needs an entry per block")
    stride = t.stride(0) if t.shape[0] > 1 else t.shape[1]
    return (PaBlockPool(pool.free_stack.data_ptr(), pool.free_top.data_ptr(), t.data_ptr(), pool.count.data_ptr(), stride,
                        pool.ref_count.numel(), t.shape[0], t.shape[1], 0),
            _lib.PaBlockShare(pool.ref_count.data_ptr(), pool.scratch.data_ptr(), pool.scratch.numel()))


def _reorder_call(desc, share, descs, dev: torch.device, slots: torch.Tensor, parents: torch.Tensor,
                  num_tokens: torch.Tensor, status: Optional[torch.Tensor]) -> torch.Tensor:
    if slots.dim() != 2 or parents.shape != slots.shape or num_tokens.shape != slots.shape[:1]:
        raise ValueError("slots and parents must be [num_groups, num_beams], num_tokens [num_groups]")
    _check_vectors(dev, slots=slots, parents=parents, num_tokens=num_tokens, status=status)
    out = torch.empty_like(slots)
    with torch.cuda.device(dev):
        _lib.check("block_pool_reorder", _lib.load().block_pool_reorder(
            ctypes.byref(desc), ctypes.byref(share), slots.data_ptr(), parents.data_ptr(), num_tokens.data_ptr(),
            slots.shape[0], slots.shape[1], out.data_ptr(), descs, len(descs), _ptr(status), _stream(dev)))
    return out


def reorder_beams(pool: PoolState, slots: torch.Tensor, parents: torch.Tensor, num_tokens: torch.Tensor,
                  k_cache: Caches, v_cache: Caches, k_scale: Optional[Caches] = None,
                  v_scale: Optional[Caches] = None, *, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Beams take over their parents' state in the paged cache; returns the beams' pool rows afterwards.

    ``slots`` [G, K] are the pool rows of each group's beams, ``parents`` [G, K] the beam that beam j continues,
    ``num_tokens`` [G] the tokens in the cache (int32, on the device).  Full blocks are shared, a partly filled
    last block is copied in every layer, blocks that no beam continues are freed; see block_pool_reorder.
    """
    k, v = _layers(k_cache), _layers(v_cache)
    slots, parents, num_tokens = _i32(slots), _i32(parents), _i32(num_tokens)
    if not k:
        raise ValueError("as many K as V pools are needed, one at least (got none)")
    if BACKEND == "torch" and not _CHECK:  # the op checks the rest
        return _op("reorder_beams")(*pool, slots, parents, num_tokens, k, v, _layers(k_scale), _layers(v_scale), status)
    dev = k[0].device
    if status is None and _CHECK:
        status = status_word(dev)
    if BACKEND == "torch":
        out = _op("reorder_beams")(*pool, slots, parents, num_tokens, k, v, _layers(k_scale), _layers(v_scale), status)
    else:
        _check_vectors(dev, ref_count=pool.ref_count)
        out = _reorder_call(*pool_descs(pool), layer_descs(k_cache, v_cache, k_scale, v_scale), dev, slots, parents,
                            num_tokens, status)
    if _CHECK and status is not None:
        _raise_status("reorder_beams", status)
    return out


def _compact_call(desc, share, descs, dev: torch.device, num_blocks: int, status: Optional[torch.Tensor]) -> torch.Tensor:
    _check_vectors(dev, status=status)
    live = torch.empty(1, dtype=torch.int32, device=dev)
    with torch.cuda.device(dev):
        _lib.check("block_pool_compact", _lib.load().block_pool_compact(
            ctypes.byref(desc), ctypes.byref(share), num_blocks, live.data_ptr(), descs, len(descs), _ptr(status),
            _stream(dev)))
    return live


def compact_blocks(pool: PoolState, k_cache: Caches, v_cache: Caches, k_scale: Optional[Caches] = None,
                   v_scale: Optional[Caches] = None, *, num_blocks: Optional[int] = None,
                   status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Move the blocks in use to the lowest ids (pages, rows, holder counts, free list); see block_pool_compact.

    Afterwards only ids below ``num_blocks`` (default: all of the pool's) are in use or handed out.  Returns the
    number of blocks in use, int32 [1] on the device.
    """
    k, v = _layers(k_cache), _layers(v_cache)
    if not k:
        raise ValueError("as many K as V pools are needed, one at least (got none)")
    if num_blocks is not None and num_blocks < 0:
        raise ValueError("num_blocks must be >= 0")
    dev = k[0].device
    if status is None and _CHECK:
        status = status_word(dev)
    if BACKEND == "torch":
        live = _op("compact_blocks")(*pool, -1 if num_blocks is None else num_blocks, k, v, _layers(k_scale),
                                     _layers(v_scale), status)
    else:
        _check_vectors(dev, ref_count=pool.ref_count)
        desc, share = pool_descs(pool)
        live = _compact_call(desc, share, layer_descs(k_cache, v_cache, k_scale, v_scale), dev,
                             desc.num_blocks if num_blocks is None else num_blocks, status)
    if _CHECK and status is not None:
        _raise_status("compact_blocks", status)
    return live


def beam_select(logits: torch.Tensor, beam_scores: torch.Tensor, num_out: Optional[int] = None, *,
                finished: Optional[torch.Tensor] = None,
                eos_id: Optional[int] = None) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """The ``num_out`` best continuations of every sequence's beams; returns (scores, tokens, parents) [B, num_out].

    ``logits`` [B, K, V] (float32, float16 or bfloat16, any strides with a contiguous vocabulary), ``beam_scores``
    [B, K] float32: the candidate (k, v) scores ``beam_scores[k] + log_softmax(logits[k])[v]``.  Ordered by score, then
    lower beam, then larger logit, then lower token.  ``finished`` [B, K] (bool): such a beam is not read; it
    continues with ``eos_id`` at its own score.  ``num_out`` defaults to K; scores float32, tokens and
    parents int32.  See beam_select in the C header for NaN and infinities.
    """
    if logits.dim() != 3 or beam_scores.dim() != 2:
        raise ValueError("logits must be [num_seqs, num_beams, vocab] and beam_scores [num_seqs, num_beams]")
    if logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"logits must be float32, float16 or bfloat16, got {logits.dtype}")
    if finished is not None and eos_id is None:
        raise ValueError("finished beams need eos_id")
    B, K, V = logits.shape
    n = K if num_out is None else int(num_out)
    if V < 1 or not 1 <= n <= max(1, K) * V:
        raise ValueError(f"num_out {n} is outside 1..num_beams * vocab ({K} * {V})")
    if finished is not None and not 0 <= eos_id < V:
        raise ValueError(f"eos_id {eos_id} is outside the vocabulary of {V}")
    if logits.stride(2) != 1 and V > 1:
        logits = logits.contiguous()
    if not beam_scores.is_contiguous():
        beam_scores = beam_scores.contiguous()
    if finished is not None and not finished.is_contiguous():
        finished = finished.contiguous()
    if BACKEND == "torch":
        return _op("beam_select")(logits, beam_scores, n, finished, -1 if eos_id is None else int(eos_id))
    dev = logits.device
    if tuple(beam_scores.shape) != (B, K) or beam_scores.dtype != torch.float32 or beam_scores.device != dev:
        raise ValueError(f"beam_scores must be float32 [{B}, {K}] on {dev}")
    if finished is not None and (tuple(finished.shape) != (B, K) or finished.dtype not in (torch.bool, torch.uint8)
                                 or finished.device != dev):
        raise ValueError(f"finished must be bool [{B}, {K}] on {dev}")
    a = _lib.PaBeamSelect()
    a.logits, a.scores, a.finished = logits.data_ptr(), beam_scores.data_ptr(), _ptr(finished)
    a.stride_seq, a.stride_beam, a.dtype = logits.stride(0), logits.stride(1), _TORCH2PA[logits.dtype]
    a.num_seqs, a.num_beams, a.vocab, a.num_out = B, K, V, n
    a.eos_id = -1 if eos_id is None else int(eos_id)
    lib = _lib.load()
    with torch.cuda.device(dev):
        nbytes = ctypes.c_size_t(0)
        _lib.check("beam_select", lib.beam_select_workspace_size(a, ctypes.byref(nbytes)))
        ws = torch.empty(max(1, nbytes.value), dtype=torch.uint8, device=dev)
        scores = torch.empty(B, n, dtype=torch.float32, device=dev)
        tokens = torch.empty(B, n, dtype=torch.int32, device=dev)
        parents = torch.empty(B, n, dtype=torch.int32, device=dev)
        a.out_scores, a.out_tokens, a.out_parents = scores.data_ptr(), tokens.data_ptr(), parents.data_ptr()
        _lib.check("beam_select", lib.beam_select(a, ws.data_ptr(), nbytes.value, _stream(dev)))
    return scores, tokens, parents


Penalty = Union[float, torch.Tensor]


def _per_row(name: str, v: Penalty, rows: int, dev: torch.device) -> tuple[Optional[torch.Tensor], float]:
    if not isinstance(v, torch.Tensor):
        return None, float(v)
    if v.numel() != rows or v.device != dev:
        raise ValueError(f"{name} must be a number or {rows} values on {dev}")
    return v.to(torch.float32).reshape(rows).contiguous(), 0.0


def adjust_logits(logits: torch.Tensor, *, tokens: Optional[torch.Tensor] = None,
                  num_tokens: Optional[torch.Tensor] = None, prompt_len: Optional[torch.Tensor] = None,
                  repetition_penalty: Penalty = 1.0, presence_penalty: Penalty = 0.0, frequency_penalty: Penalty = 0.0,
                  bias: Optional[torch.Tensor] = None, bias_row: Optional[torch.Tensor] = None,
                  mask: Optional[torch.Tensor] = None, mask_row: Optional[torch.Tensor] = None,
                  out: Optional[torch.Tensor] = None, status: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Penalties for repeated tokens, biases and grammar masks on ``logits`` [..., V]; returns the new logits.

    Of a row, with n the times that token v was generated: ``x / repetition`` (``x * repetition`` below 0) where v was
    seen, then ``- frequency * n``, then ``- presence`` where n > 0, then ``+ bias``, then -inf where the mask's bit is
    clear, in float32 and rounded once to the dtype of ``out`` (by default the logits' own; float32 or ``logits``
    itself will do).

    ``tokens`` [..., L] (int32) are what each row has seen: the first ``prompt_len`` of them its prompt, which
    counts as seen but not as generated, those from ``num_tokens`` on nothing, ids outside the vocabulary nothing.
    A penalty is a number or one value per row.  ``bias`` float32 [N, V] (or [V]) and ``mask`` int32 [M, ceil(V / 32)]
    (token v: bit v % 32 of word v // 32, 1 = allowed) are one per row, one for all, or chosen by ``bias_row`` /
    ``mask_row`` (-1: none).  See logits_adjust in the C header.
    """
    if BACKEND == "torch" and logits.is_cuda and out is None and not _CHECK:  # the op checks and makes the new logits
        rep, rep_v = (repetition_penalty, 0.0) if isinstance(repetition_penalty, torch.Tensor) else (None, repetition_penalty)
        pres, pres_v = (presence_penalty, 0.0) if isinstance(presence_penalty, torch.Tensor) else (None, presence_penalty)
        freq, freq_v = (frequency_penalty, 0.0) if isinstance(frequency_penalty, torch.Tensor) else (None, frequency_penalty)
        return _op("adjust_logits")(logits, tokens, num_tokens, prompt_len, rep, rep_v, pres, pres_v, freq, freq_v, bias,
                                    bias_row, mask, mask_row, status)
    if logits.dim() < 1 or logits.dtype not in (torch.float32, torch.float16, torch.bfloat16):
        raise ValueError(f"logits must be float32, float16 or bfloat16 [..., vocab], got {logits.dtype} {tuple(logits.shape)}")
    V = logits.shape[-1]
    if V < 1:
        raise ValueError("logits need a vocabulary")
    if not isinstance(repetition_penalty, torch.Tensor) and not repetition_penalty > 0:
        raise ValueError(f"repetition_penalty {repetition_penalty} must be positive")
    x = logits if logits.dim() == 2 else logits.reshape(-1, V)
    if x.stride(1) != 1 and V > 1:
        x = x.contiguous()
    R, dev = x.shape[0], logits.device
    if out is None:
        out = torch.empty(logits.shape, dtype=logits.dtype, device=dev)
    elif out.shape != logits.shape or out.dtype not in (logits.dtype, torch.float32):
        raise ValueError("out must be shaped like logits, in their dtype or float32")
    o = out if out.dim() == 2 else out.view(-1, V)
    if o.stride(1) != 1 and V > 1:
        raise ValueError("out needs a contiguous vocabulary")
    if tokens is not None:
        if tokens.dim() != logits.dim() or tokens.shape[:-1] != logits.shape[:-1]:
            raise ValueError(f"tokens must be [{', '.join(map(str, logits.shape[:-1]))}, max_tokens]")
        tokens = tokens if tokens.dtype == torch.int32 else tokens.to(torch.int32)
        tokens = tokens if tokens.dim() == 2 else tokens.reshape(R, tokens.shape[-1])
        if tokens.stride(1) != 1 and tokens.shape[1] > 1:
            tokens = tokens.contiguous()
    elif num_tokens is not None or prompt_len is not None:
        raise ValueError("num_tokens and prompt_len come with tokens")
    num_tokens, prompt_len, bias_row, mask_row = (t if t is None else _i32(t).view(-1) for t in
                                                  (num_tokens, prompt_len, bias_row, mask_row))
    rep, rep_v = _per_row("repetition_penalty", repetition_penalty, R, dev)
    pres, pres_v = _per_row("presence_penalty", presence_penalty, R, dev)
    freq, freq_v = _per_row("frequency_penalty", frequency_penalty, R, dev)
    if bias is not None:
        bias = (bias if bias.dtype == torch.float32 else bias.float()).view(-1, V) if bias.dim() == 1 else bias.float()
        if bias.dim() != 2 or bias.shape[1] != V:
            raise ValueError(f"bias must be [N, {V}] or [{V}]")
        if bias.stride(1) != 1 and V > 1:
            bias = bias.contiguous()
    if mask is not None:
        mask = mask.view(1, -1) if mask.dim() == 1 else mask
        if mask.dim() != 2 or mask.dtype != torch.int32 or mask.shape[1] != (V + 31) // 32:
            raise ValueError(f"mask must be int32 [M, {(V + 31) // 32}] or [{(V + 31) // 32}]")
        if mask.stride(1) != 1 and mask.shape[1] > 1:
            mask = mask.contiguous()
    for name, t, by in (("bias", bias, bias_row), ("mask", mask, mask_row)):
        if t is None and by is not None:
            raise ValueError(f"{name}_row without {name}")
        if t is not None and by is None and t.shape[0] not in (1, R):
            raise ValueError(f"{name} has {t.shape[0]} rows for {R} rows of logits: pass {name}_row")
    if status is None and _CHECK:
        status = status_word(dev)
    if BACKEND == "torch":
        _op("adjust_logits_out")(x, tokens, num_tokens, prompt_len, rep, rep_v, pres, pres_v, freq, freq_v, bias, bias_row,
                                 mask, mask_row, status, o)
    else:
        for name, t in (("tokens", tokens), ("num_tokens", num_tokens), ("prompt_len", prompt_len), ("bias", bias),
                        ("bias_row", bias_row), ("mask", mask), ("mask_row", mask_row), ("out", o), ("status", status)):
            if t is not None and t.device != dev:
                raise ValueError(f"{name} is on {t.device}, logits on {dev}")
        if dev.type != "cuda":
            raise ValueError("logits must be a CUDA tensor")
        for name, t in (("num_tokens", num_tokens), ("prompt_len", prompt_len), ("bias_row", bias_row), ("mask_row", mask_row)):
            if t is not None and t.numel() != R:
                raise ValueError(f"{name} must hold {R} values")
        a = _lib.PaLogits()
        a.logits, a.out, a.stride_row, a.out_stride_row = x.data_ptr(), o.data_ptr(), x.stride(0), o.stride(0)
        a.dtype, a.out_dtype, a.rows, a.vocab = _TORCH2PA[x.dtype], _TORCH2PA[o.dtype], R, V
        if tokens is not None:
            a.tokens, a.tokens_stride, a.max_tokens = tokens.data_ptr(), tokens.stride(0), tokens.shape[1]
        a.num_tokens, a.prompt_len = _ptr(num_tokens), _ptr(prompt_len)
        a.repetition, a.presence, a.frequency = _ptr(rep), _ptr(pres), _ptr(freq)
        a.repetition_value, a.presence_value, a.frequency_value = rep_v, pres_v, freq_v
        if bias is not None:
            a.bias, a.bias_stride, a.bias_rows, a.bias_row = bias.data_ptr(), bias.stride(0), bias.shape[0], _ptr(bias_row)
        if mask is not None:
            a.mask, a.mask_stride, a.mask_rows, a.mask_row = mask.data_ptr(), mask.stride(0), mask.shape[0], _ptr(mask_row)
        with torch.cuda.device(dev):
            _lib.check("logits_adjust", _lib.load().logits_adjust(a, _ptr(status), _stream(dev)))
    if _CHECK and status is not None:
        _raise_status("adjust_logits", status)
    return out
