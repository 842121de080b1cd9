"""GPU: shared_prefix_attention's outputs by the 2-norm of a head's error, for keys and values as the kernels multiply them.

The elementwise tolerance of test_gpu_shared_prefix.py has to allow every rounding at its worst at once, which for INT8 pools is
about the size of the outputs.  Here INT8 keys and values of a shared part are those that the tensor-core kernel takes, code
times scale rounded to fp16 once, so that what is left are roundings of the probabilities; see oracle/shared_prefix.py for the bound.
"""
import math

import pytest
import torch

from oracle.shared_prefix import attend, lse_bound, norm_bound
from test_gpu_shared_prefix import Problem

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from pie_b200 import ops as o
    assert torch.cuda.is_available()
    return o


def check_norms(p, O, L, shared, wide, rows=None, scale=None, range_=1.0):
    """``shared`` [B]: keys of each sequence that the prefix kernel reads; ``wide``: it is the tensor-core kernel.  INT8 codes times
    scales round to fp16 as in fp16 with ``range_`` (a power of two) times its range, which holds for values of any size as long
    as none of them lies below fp16's normal range then."""
    int8 = p.K.dtype == torch.int8
    operand = torch.float16 if int8 else p.K.dtype
    unit = torch.finfo(operand).eps / 2
    sc = scale or 1 / math.sqrt(p.D)
    G = p.Hq // p.Hkv
    for b in range(p.B) if rows is None else rows:
        n_rows = min(int(p.q_len[b]), p.maxq)
        k, v = p.keys(b)
        n = k.shape[0]
        codes = None
        if int8:
            cut = shared[b] if wide else 0
            for t in (k, v):
                t[:cut] = (t[:cut] / range_).half().double() * range_
            ids = p.table[b, :-(-n // p.BS)].long()
            codes = p.V[ids].flatten(0, 1)[:n].double().norm(dim=2)  # [n, Hkv]
            if wide:  # the prefix's probabilities carry no scale
                codes[:cut] = v[:cut].norm(dim=2)
            codes = codes.repeat_interleave(G, 1)
        k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
        for m in range(n_rows):
            seen = min(n, int(p.kv_len[b]) - n_rows + m + 1)
            q = p.Q[b, :, m].double()
            step = 0.0
            if p.Q.dtype != operand and not (operand == torch.float16 and bool((q.half().double() == q).all())):
                step = q.abs() * unit
            if int8:  # the split-K kernel's fixed point
                step = torch.zeros_like(q) + step + q.abs().amax(1, keepdim=True) / 65024
            o, lse, w = attend(q, k[:seen], v[:seen], sc)
            bound = norm_bound(q, k[:seen], v[:seen], sc, o, w, unit, step, p_times=None if codes is None else codes[:seen])
            off = (O[b, :, m].double() - o).norm(dim=1)
            assert bool((off <= bound).all()), (b, m, (off / bound).max().item(), (off / o.norm(dim=1)).max().item())
            off = (L[b, :, m].double() - lse).abs()
            assert bool((off <= lse_bound(q, k[:seen], sc, lse, step)).all()), (b, m, off.max().item())


def parts(groups, BS, alone=0):
    return [s // BS * BS if n > 1 else 0 for n, s in groups for _ in range(n)] + [0] * alone


def both_forms(p, ops, monkeypatch, shared, rows=None, range_=1.0):
    for wide in (True, False):
        if not wide:
            monkeypatch.setenv("PIE_B200_NO_TCGEN05", "1")
        O, L = ops.shared_prefix_attention(*p.args())
        check_norms(p, O, L, shared, wide, rows, range_=range_)
    monkeypatch.delenv("PIE_B200_NO_TCGEN05")


@pytest.mark.parametrize("scale_dtype,big", [(torch.float32, 300.0), (torch.float32, 600.0), (torch.float32, 50000.0), (torch.float32, 3e5),
                                             (torch.float16, 600.0), (torch.float16, 60000.0)])
@pytest.mark.parametrize("D", [64, 128])
def test_keys_beyond_the_range_of_fp16(ops, monkeypatch, scale_dtype, big, D):
    """INT8 keys of which some pass 65504 with their scales: the logits are finite, and so are the outputs.  A whole tile of
    such keys, and a few among 32 or 128 others; queries so small that logits are a few units (all of them numbers of fp16)."""
    groups = [(20, 700), (9, 320)]
    p = Problem(groups, [[5] * 20, [40] * 9], pool=torch.int8, D=D, scale_dtype=scale_dtype, seed=int(big) % 1000 + D)
    for b, at in ((0, range(128, 256)), (0, (300, 301, 350)), (0, range(513, 640, 7)), (20, (5, 200, 319))):
        for i in at:
            p.ks[p.table[b, i // p.BS].long(), i % p.BS] = big
    p.Q = (p.Q.float() * 2.0 ** -math.ceil(math.log2(big * 127 / 4))).half()
    assert bool((p.Q != 0).any(-1).all())
    both_forms(p, ops, monkeypatch, parts(groups, 16), rows=[0, 7, 19, 20, 28], range_=1024.0)


@pytest.mark.parametrize("scale_dtype,big", [(torch.float32, 512.0), (torch.float32, 600.0), (torch.float32, 65000.0), (torch.float16, 600.0),
                                             (torch.float16, 65504.0)])
@pytest.mark.parametrize("D", [64, 128])
def test_values_beyond_the_range_of_fp16(ops, scale_dtype, big, D):
    """INT8 values beyond 65504 of keys that weigh little (zeros: a logit of 0), so that the outputs are within fp16."""
    groups = [(20, 700), (9, 320)]
    p = Problem(groups, [[5] * 20, [40] * 9], pool=torch.int8, D=D, scale_dtype=scale_dtype, seed=int(big) % 1000 + D)
    for b, at in ((0, (3, 300, 301, 640)), (20, (5, 200, 319))):
        for i in at:
            block, slot = p.table[b, i // p.BS].long(), i % p.BS
            p.vs[block, slot] = big
            p.K[block, slot] = 0
    O, L = ops.shared_prefix_attention(*p.args())
    assert big < 2000 or float(O.abs().max()) > 100  # they show
    check_norms(p, O, L, parts(groups, 16), True, rows=[0, 7, 19, 20, 28], range_=1024.0)
