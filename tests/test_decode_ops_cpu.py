"""CPU: argument checks and struct layouts of the operators of a decode step (rotation, logit rules)."""
import ctypes
import os
import subprocess

import numpy as np
import pytest
import torch

from conftest import ROOT
from test_capi_cpu import _descs


def test_struct_layouts_match_header(tmp_path):
    from pie_b200 import _lib

    structs = {"pa_rotate_t": _lib.PaRotate, "pa_logits_t": _lib.PaLogits}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "paged_attn_b200.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(lines + ["return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    for ln in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split("\n"):
        if ln:
            cname, field, val = ln.split()
            py = structs[cname]
            assert int(val) == (ctypes.sizeof(py) if field == "sizeof" else getattr(py, field).offset), ln


def _rotate_descs():
    from pie_b200 import _lib

    _, kv, pg = _descs()
    nw = _lib.PaKvNew()
    nw.k_new = nw.v_new = nw.seq_index = nw.positions = 1 << 22
    nw.dtype, nw.num_tokens = _lib.PA_DTYPE_F16, 5
    nw.k_stride_token = nw.v_stride_token = 256
    nw.k_stride_head = nw.v_stride_head = 128
    r = _lib.PaRotate()
    r.q = r.q_out = r.cos_sin = 1 << 23
    r.q_stride_token, r.q_stride_head, r.qo_stride_token, r.qo_stride_head = 1024, 128, 1024, 128
    r.cs_stride, r.num_q_heads, r.rot_dim, r.num_positions = 128, 8, 128, 100
    return nw, r, kv, pg


@pytest.mark.parametrize("mutate,code,msg", [
    (lambda nw, r, kv: setattr(r, "rot_dim", 24), -2, b"rot_dim"),
    (lambda nw, r, kv: setattr(r, "rot_dim", 144), -2, b"rot_dim"),
    (lambda nw, r, kv: setattr(r, "rot_dim", 0), -2, b"rot_dim"),
    (lambda nw, r, kv: setattr(r, "cos_sin", None), -1, b"cos_sin"),
    (lambda nw, r, kv: setattr(r, "cs_stride", 130), -1, b"cos_sin"),
    (lambda nw, r, kv: setattr(r, "cos_sin", (1 << 23) + 4), -1, b"cos_sin"),
    (lambda nw, r, kv: setattr(r, "q_out", None), -1, b"q_out"),
    (lambda nw, r, kv: setattr(r, "q_stride_head", 129), -1, b"q rows"),
    (lambda nw, r, kv: setattr(r, "num_q_heads", -1), -1, b"negative"),
    (lambda nw, r, kv: setattr(r, "num_q_heads", 1 << 25), -2, b"2\\^26"),
    (lambda nw, r, kv: setattr(nw, "dtype", 2), -1, b"dtype"),
    (lambda nw, r, kv: setattr(nw, "positions", None), -1, b"NULL"),
    (lambda nw, r, kv: setattr(kv, "dtype", 2), -1, b"k_scale"),
])
def test_rotate_arguments(mutate, code, msg):
    from pie_b200 import _lib

    lib = _lib.load()
    nw, r, kv, pg = _rotate_descs()
    mutate(nw, r, kv)
    assert lib.kv_rotate_write(nw, r, kv, pg, None, None) == code
    assert msg.replace(b"\\", b"") in lib.paged_attn_error_string()
    assert lib.kv_rotate_write(nw, None, kv, pg, None, None) == -1


def test_rotate_needs_scales_per_token():
    from pie_b200 import _lib

    lib = _lib.load()
    nw, r, kv, pg = _rotate_descs()
    kv.dtype, kv.k_scale, kv.v_scale = _lib.PA_DTYPE_I8, 1 << 24, 1 << 24
    kv.ks_stride_block = kv.vs_stride_block = 2
    kv.ks_stride_head = kv.vs_stride_head = 1
    assert lib.kv_rotate_write(nw, r, kv, pg, None, None) == -1
    assert b"per-token" in lib.paged_attn_error_string()


def _logits_desc():
    from pie_b200 import _lib

    a = _lib.PaLogits()
    a.logits, a.out, a.stride_row, a.out_stride_row = 1 << 22, 1 << 23, 1000, 1000
    a.dtype = a.out_dtype = _lib.PA_DTYPE_BF16
    a.rows, a.vocab, a.repetition_value = 4, 1000, 1.0
    return a


@pytest.mark.parametrize("mutate,msg", [
    (lambda a: setattr(a, "dtype", 2), b"dtype"),
    (lambda a: setattr(a, "out_dtype", 0), b"out dtype"),
    (lambda a: setattr(a, "out_dtype", 9), b"out dtype"),
    (lambda a: setattr(a, "vocab", 0), b"sizes"),
    (lambda a: setattr(a, "rows", -1), b"sizes"),
    (lambda a: setattr(a, "max_tokens", 3), b"NULL"),
    (lambda a: setattr(a, "logits", None), b"NULL"),
    (lambda a: setattr(a, "logits", (1 << 22) + 1), b"misaligned"),
    (lambda a: setattr(a, "stride_row", -1000), b"negative"),
    (lambda a: setattr(a, "out_stride_row", 999), b"overlap"),
    (lambda a: setattr(a, "repetition_value", 0.0), b"positive"),
    (lambda a: setattr(a, "repetition_value", float("nan")), b"positive"),
    (lambda a: (setattr(a, "bias", 1 << 24), setattr(a, "bias_rows", 3)), b"bias has 3 rows"),
    (lambda a: (setattr(a, "mask", 1 << 24), setattr(a, "mask_rows", 0)), b"mask has 0 rows"),
    (lambda a: (setattr(a, "out", 1 << 22), setattr(a, "out_dtype", 3)), b"over the logits"),
    (lambda a: (setattr(a, "out", 1 << 22), setattr(a, "out_stride_row", 1008)), b"over the logits"),
])
def test_logits_arguments(mutate, msg):
    from pie_b200 import _lib

    lib = _lib.load()
    a = _logits_desc()
    mutate(a)
    assert lib.logits_adjust(a, None, None) == -1
    assert msg in lib.paged_attn_error_string()
    assert lib.logits_adjust(None, None, None) == -1


@pytest.mark.parametrize("kw,msg", [
    (dict(k_new=torch.zeros(2, 3, 64)), "match the pool"),
    (dict(v_new=torch.zeros(2, 2, 64, dtype=torch.float16)), "dtype"),
    (dict(cos_sin=torch.zeros(9, 24)), "rot_dim"),
    (dict(cos_sin=torch.zeros(9, 80)), "rot_dim"),
    (dict(cos_sin=torch.zeros(9, 32).half()), "float32"),
    (dict(q=torch.zeros(2, 4, 128)), "q must be"),
    (dict(q=torch.zeros(2, 4, 64).half()), "q must be"),
    (dict(q=None, q_out=torch.zeros(2, 4, 64)), "without q"),
    (dict(q_out=torch.zeros(2, 4, 32)), "q_out"),
    (dict(positions=torch.zeros(3, dtype=torch.int32)), "one entry per token"),
    (dict(k_cache=torch.zeros(4, 16, 2, 64, dtype=torch.int8)), "one scale per"),
])
def test_rotate_front_end(kw, msg):
    from pie_b200 import ops

    args = dict(q=torch.zeros(2, 4, 64), k_new=torch.zeros(2, 2, 64), v_new=torch.zeros(2, 2, 64), cos_sin=torch.zeros(9, 32),
                block_table=torch.zeros(1, 3, dtype=torch.int32), seq_index=torch.zeros(2, dtype=torch.int32),
                positions=torch.zeros(2, dtype=torch.int32), k_cache=torch.zeros(4, 16, 2, 64), v_cache=torch.zeros(4, 16, 2, 64))
    if "k_new" in kw:
        kw = {**kw, "v_new": kw["k_new"]}
    with pytest.raises(ValueError, match=msg):
        ops.rotate_write_kv(**{**args, **kw})


@pytest.mark.parametrize("kw,msg", [
    (dict(logits=torch.zeros(2, 8, dtype=torch.int32)), "float32, float16 or bfloat16"),
    (dict(logits=torch.zeros(2, 0)), "vocabulary"),
    (dict(repetition_penalty=0.0), "positive"),
    (dict(repetition_penalty=torch.ones(3)), "2 values"),
    (dict(num_tokens=torch.zeros(2)), "come with tokens"),
    (dict(tokens=torch.zeros(3, 4, dtype=torch.int32)), "tokens must be"),
    (dict(tokens=torch.zeros(4, dtype=torch.int32)), "tokens must be"),
    (dict(bias=torch.zeros(3, 8)), "bias_row"),
    (dict(bias=torch.zeros(2, 9)), "bias must be"),
    (dict(mask=torch.zeros(2, 2, dtype=torch.int32)), "mask must be"),
    (dict(mask=torch.zeros(2, 1)), "mask must be"),
    (dict(mask=torch.zeros(3, 1, dtype=torch.int32)), "mask_row"),
    (dict(mask_row=torch.zeros(2, dtype=torch.int32)), "without mask"),
    (dict(out=torch.zeros(2, 8).half()), "out must be"),
    (dict(out=torch.zeros(2, 9)), "out must be"),
    (dict(out=torch.zeros(8, 2).t()), "contiguous"),
])
def test_logits_front_end(kw, msg):
    from pie_b200 import ops

    with pytest.raises(ValueError, match=msg):
        ops.adjust_logits(**{**dict(logits=torch.zeros(2, 8)), **kw})


def test_rope_table_checks():
    from pie_b200 import ops

    for bad in ((4, 3), (4, 0), (-1, 4)):
        with pytest.raises(ValueError):
            ops.rope_table(*bad, device="cpu")
    t = ops.rope_table(5, 4, 100.0, device="cpu")
    angle = np.arange(5)[:, None] * np.array([1.0, 0.1])
    assert np.abs(t.numpy() - np.concatenate([np.cos(angle), np.sin(angle)], 1)).max() < 2.0**-24
