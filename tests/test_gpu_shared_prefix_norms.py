"""GPU: shared_prefix_attention's outputs by the 2-norm of a head's error, for keys and values as the kernels multiply them.

The elementwise tolerance of test_gpu_shared_prefix.py has to allow every rounding at its worst at once, which for INT8 pools is
about the size of the outputs.  Here INT8 keys and values of a shared part are those that the tensor-core kernel takes, code
times scale rounded to fp16 once, so that what is left are roundings of the probabilities; see oracle/shared_prefix.py for the bound.
tests/test_shared_prefix_norms_cpu.py shows that it does not pass what a wrong tile would give.
"""
import math

import numpy as np
import pytest
import torch

from oracle.shared_prefix import attend, lse_bound, norm_bound
from test_gpu_shared_prefix import POOLS, Problem

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


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("BS", [8, 16, 64])
def test_groups_of_all_sizes(ops, monkeypatch, pool, D, BS):
    rng = np.random.default_rng(BS)
    groups = [(2, 64), (5, 320), (1, 200), (0, 500), (9, 129 + BS), (3, 1000)]
    own = [rng.integers(1, 90, n).tolist() for n, _ in groups]
    p = Problem(groups, own, alone=[1, 33, 300], D=D, BS=BS, pool=pool, seed=BS + D)
    both_forms(p, ops, monkeypatch, parts(groups, BS, 3))


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("n,shared,Hq", [(64, 2048, 8), (33, 4097, 8), (100, 640, 4), (3, 20000, 2), (130, 1280, 2)])
def test_many_members_and_long_prefixes(ops, monkeypatch, pool, n, shared, Hq):
    rng = np.random.default_rng(n)
    p = Problem([(n, shared)], [rng.integers(1, 60, n).tolist()], Hq=Hq, Hkv=2, pool=pool, seed=n)
    both_forms(p, ops, monkeypatch, parts([(n, shared)], 16), rows=rng.choice(n, min(n, 24), replace=False).tolist() if n > 3 else range(3))


@pytest.mark.parametrize("scale_dtype,per_block", [(torch.float32, False), (torch.float32, True), (torch.float16, True)])
@pytest.mark.parametrize("maxq", [1, 3])
def test_scales(ops, monkeypatch, scale_dtype, per_block, maxq):
    groups = [(20, 300), (6, 64)]
    p = Problem(groups, [[5] * 20, [40] * 6], pool=torch.int8, scale_dtype=scale_dtype, per_block=per_block, seed=5, maxq=maxq)
    both_forms(p, ops, monkeypatch, parts(groups, 16))


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


def test_a_captured_step_over_an_int8_cache():
    """DecodeStepGraph with a rotation table and shared prefixes: forks of one prompt over an INT8 cache."""
    from pie_b200 import ops as o
    from pie_b200.block_pool import DeviceBlockManager
    from pie_b200.decode_step import DecodeStepGraph
    from pie_b200.workloads import empty_head_major_scales
    from test_gpu_forked_decode import Step, turned

    BS, Hkv, D, Hq, NB, n = 16, 2, 128, 8, 160, 533
    gen = torch.Generator(device="cuda").manual_seed(8)
    k, v = (torch.zeros(NB, BS, Hkv, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (empty_head_major_scales(NB, BS, Hkv, device="cuda").zero_() for _ in range(2))
    pool = DeviceBlockManager(NB, BS, 12, 40)
    pool.attach_caches(k, v, ks, vs)
    table = o.rope_table(600, D, device="cuda")
    graph = DecodeStepGraph(pool, k, v, ks, vs, Hq, 11, rope=table, share_prefixes=True)
    pool.allocate(0, -(-n // BS))
    inp = pool.step_inputs([0], [n], [n])
    rows = [torch.randn(n, Hkv, D, device="cuda", generator=gen).half() for _ in range(2)]
    o.rotate_write_kv(None, *rows, table, inp["block_table"], inp["token_seq"], inp["positions"], k, v, ks, vs)
    ids = list(range(9))
    for child in ids[1:]:
        pool.fork(0, child, n)
    for step in range(1, 20):
        q, kn, vn = (torch.randn(len(ids), h, D, device="cuda", generator=gen).half() for h in (Hq, Hkv, Hkv))
        out = graph.step(ids, [n + step] * len(ids), q, kn, vn).clone().unsqueeze(2)
        held = pool.block_table
        at = torch.full((len(ids),), n + step - 1, device="cuda")
        p = Step(turned(q, table, at, False), k, v, ks, vs, [held[s] for s in ids], [n + step] * len(ids), BS)
        check_norms(p, out, graph.lse[:len(ids)], [n // BS * BS] * len(ids), True)
    graph.check()
