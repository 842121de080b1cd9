"""GPU: rotate_write_kv (queries and keys turned by their positions, K/V rows written into the paged pool).

The kernel rounds every product and sum of a rotation to fp32 by itself, so its
rows equal the same operations in numpy bit for bit, INT8 codes and scales among
them.  Against 64 bits a rotated value a c - b s may be off by the two products'
and the sum's roundings, 2^-24 (|a c| + |b s|) + 2^-24 |a c - b s| (1 + 2^-23) <= 2^-22 (|a c| + |b s|),
and by half a step of its type.
"""
import numpy as np
import pytest
import torch

from oracle import decode_step as orc
from oracle import paged_attention as pa

pytestmark = pytest.mark.gpu

DTYPES = [torch.float16, torch.bfloat16, torch.float32]


@pytest.fixture(scope="module")
def ops():
    from pie_b200 import ops as o
    assert torch.cuda.is_available()
    return o


def make(T, Hq, Hkv, D, R, BS, dtype, pool, seed=0, seqs=3, num_positions=500, scale_dtype=torch.float16):
    """Tokens at distinct places of ``seqs`` sequences; every page of the tables exists."""
    g = torch.Generator().manual_seed(seed)
    rng = np.random.default_rng(seed)
    cols = -(-num_positions // BS)
    NB = seqs * cols + 3
    table = rng.permutation(NB)[:seqs * cols].reshape(seqs, cols).astype(np.int32)
    place = rng.permutation(seqs * num_positions)[:T]
    row, pos = (place // num_positions).astype(np.int32), (place % num_positions).astype(np.int32)
    x = torch.randn(T, Hq + 2 * Hkv, D, generator=g) * torch.where(torch.rand(D, generator=g) < 0.05, 9.0, 1.0)
    x = x.to(dtype).cuda()
    q, k, v = x.split([Hq, Hkv, Hkv], 1)
    angle = torch.rand(num_positions, R // 2, generator=g, dtype=torch.float64) * 1000
    cs = torch.cat([angle.cos(), angle.sin()], 1).float().cuda()
    kc = torch.zeros(NB, BS, Hkv, D, dtype=pool, device="cuda")
    scales = [torch.full((NB, BS, Hkv), 7.0, dtype=scale_dtype, device="cuda") for _ in range(2)] if pool == torch.int8 else [None, None]
    return dict(q=q, k=k, v=v, cs=cs, table=torch.from_numpy(table).cuda(), row=torch.from_numpy(row).cuda(),
                pos=torch.from_numpy(pos).cuda(), kc=kc, vc=kc.clone(), ks=scales[0], vs=scales[1], np=(table, row, pos))


def call(ops, s, interleaved, **kw):
    return ops.rotate_write_kv(s["q"], s["k"], s["v"], s["cs"], s["table"], s["row"], s["pos"], s["kc"], s["vc"], s["ks"],
                               s["vs"], interleaved=interleaved, **kw)


def expect(s, interleaved, keep=None):
    """(rotated q, K pool, V pool, K scales, V scales) as numpy, from fp32 operations one at a time."""
    table, row, pos = s["np"]
    cs = s["cs"].cpu().numpy()
    half = cs.shape[1] // 2
    ok = np.ones(len(pos), bool) if keep is None else keep
    c, sn = cs[np.where(ok, pos, 0), :half], cs[np.where(ok, pos, 0), half:]
    f = lambda t: t.float().cpu().numpy()  # noqa: E731
    q = orc.rotate(f(s["q"]), c, sn, interleaved)
    k = orc.rotate(f(s["k"]), c, sn, interleaved)
    BS = s["kc"].shape[1]
    out = []
    for x, cache, scale in ((k, s["kc"], s["ks"]), (f(s["v"]), s["vc"], s["vs"])):
        pool = torch.zeros_like(cache).cpu()
        sc = None if scale is None else torch.full(scale.shape, 7.0, dtype=scale.dtype)
        for t in np.nonzero(ok)[0]:
            blk, slot = int(table[row[t], pos[t] // BS]), int(pos[t]) % BS
            if scale is None:
                pool[blk, slot] = torch.from_numpy(x[t]).to(cache.dtype)
            else:
                codes, step = pa.quantize_rows(x[t])
                pool[blk, slot] = torch.from_numpy(codes)
                sc[blk, slot] = torch.from_numpy(step).to(scale.dtype)
        out += [pool, sc]
    return torch.from_numpy(q).to(s["q"].dtype), out[0], out[2], out[1], out[3]


def check(s, got_q, want):
    q, k, v, ks, vs = want
    assert torch.equal(got_q.cpu(), q)
    assert torch.equal(s["kc"].cpu(), k) and torch.equal(s["vc"].cpu(), v)
    if ks is not None:
        assert torch.equal(s["ks"].cpu(), ks) and torch.equal(s["vs"].cpu(), vs)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("pool", [torch.int8, torch.float16, torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,Hq,Hkv,D,R,BS", [(1, 32, 8, 128, 128, 16), (37, 6, 3, 64, 64, 8), (90, 5, 5, 128, 32, 32),
                                             (3, 1, 1, 128, 96, 1), (41, 12, 2, 64, 16, 64), (64, 7, 1, 128, 112, 16)])
def test_equals_the_operations_one_by_one(ops, T, Hq, Hkv, D, R, BS, dtype, pool, interleaved):
    s = make(T, Hq, Hkv, D, R, BS, dtype, pool, seed=T + R)
    check(s, call(ops, s, interleaved), expect(s, interleaved))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("dtype", DTYPES)
def test_against_64_bits(ops, dtype, interleaved):
    s = make(200, 4, 2, 128, 64, 16, dtype, dtype, seed=8)
    q = call(ops, s, interleaved).double().cpu().numpy()
    cs = s["cs"].double().cpu().numpy()[s["np"][2]]
    x = s["q"].double().cpu().numpy()
    want = orc.rotate(x, cs[:, :32], cs[:, 32:], interleaved)
    size = orc.rotate(np.abs(x), np.abs(cs[:, :32]), -np.abs(cs[:, 32:]), interleaved)  # |a c| + |b s| for the first of a pair
    size2 = orc.rotate(np.abs(x), np.abs(cs[:, :32]), np.abs(cs[:, 32:]), interleaved)
    size = np.maximum(size, size2)
    half_step = torch.finfo(dtype).eps / 2
    tol = 2.0**-22 * size + half_step * (np.abs(want) + 2.0**-22 * size) + torch.finfo(dtype).tiny * half_step
    assert (np.abs(q - want)[..., :64] <= tol[..., :64]).all()
    assert np.array_equal(q[..., 64:], x[..., 64:])


def test_rope_table_and_write_kv_of_rotated_rows(ops):
    """The table helper's angles, and the same cache as write_kv on rows that were rotated before."""
    R, D = 64, 128
    cs = ops.rope_table(300, R, 5000.0, scaling=2.0)
    angle = np.arange(300)[:, None] / 2.0 * 5000.0**(-np.arange(0, R, 2) / R)
    want = np.concatenate([np.cos(angle), np.sin(angle)], 1)
    assert np.abs(cs.cpu().numpy() - want).max() <= 2.0**-24 + 1e-12 and cs.shape == (300, R)
    for pool in (torch.int8, torch.float16):
        s = make(120, 4, 3, D, R, 16, torch.float32, pool, seed=2, num_positions=300)
        s["cs"] = cs
        call(ops, s, False)
        c = cs[s["pos"].long()]
        rotated = torch.from_numpy(orc.rotate(s["k"].cpu().numpy(), c[:, :R // 2].cpu().numpy(), c[:, R // 2:].cpu().numpy(), False)).cuda()
        o = make(120, 4, 3, D, R, 16, torch.float32, pool, seed=2, num_positions=300)
        ops.write_kv(rotated, s["v"].contiguous(), s["table"], s["row"], s["pos"], o["kc"], o["vc"], o["ks"], o["vs"])
        assert torch.equal(s["kc"], o["kc"]) and torch.equal(s["vc"], o["vc"])
        if pool == torch.int8:
            assert torch.equal(s["ks"], o["ks"]) and torch.equal(s["vs"], o["vs"])


def test_far_positions_and_long_tables(ops):
    """A position near 2^20: table rows past 2^31 bytes are addressed in 64 bits."""
    P, R = 1 << 20, 128
    cs = torch.zeros(P, 5 * R, device="cuda")[:, :R]  # a wide row stride: row P - 1 starts 2.7 GB in
    cs[P - 1, :R // 2], cs[P - 1, R // 2:] = 0.0, 1.0  # a quarter turn
    s = make(2, 2, 1, 128, R, 16, torch.float16, torch.float16)
    pos = torch.tensor([P - 1, 0], dtype=torch.int32, device="cuda")
    table = torch.zeros(1, P // 16, dtype=torch.int32, device="cuda")
    table[0, -1] = 1
    q = ops.rotate_write_kv(s["q"], s["k"], s["v"], cs, table, torch.zeros(2, dtype=torch.int32, device="cuda"), pos, s["kc"], s["vc"])
    a, b = s["q"][0, :, :64], s["q"][0, :, 64:]
    assert torch.equal(q[0], torch.cat([-b, a], -1)) and not q[1].any()
    assert torch.equal(s["kc"][1, 15, 0], torch.cat([-s["k"][0, 0, 64:], s["k"][0, 0, :64]])) and torch.equal(s["vc"][0, 0, 0], s["v"][1, 0])


def test_strides_in_place_and_without_queries(ops):
    """Rows of one projection's output, tokens last but one in memory, q rotated in place, no q, no tokens, other index types."""
    for inter in (False, True):
        s = make(33, 4, 2, 128, 64, 16, torch.bfloat16, torch.int8, seed=5)
        want = expect(s, inter)
        s["q"] = s["q"].transpose(0, 1).contiguous().transpose(0, 1)
        s["k"] = s["k"].transpose(0, 1).contiguous().transpose(0, 1)
        s["kc"] = s["kc"].transpose(1, 2).contiguous().transpose(1, 2)  # [block, head, slot, d]
        s["ks"] = s["ks"].transpose(1, 2).contiguous().transpose(1, 2)
        s["row"], s["pos"] = s["row"].long(), s["pos"].long()
        got = call(ops, s, inter, q_out=s["q"])
        assert got is s["q"]
        check(s, got, want)
    s = make(33, 4, 2, 128, 64, 16, torch.bfloat16, torch.float16, seed=6)
    want = expect(s, False)
    q, s["q"] = s["q"], None
    assert call(ops, s, False) is None
    assert torch.equal(s["kc"].cpu(), want[1]) and torch.equal(s["vc"].cpu(), want[2])
    empty = s["k"][:0]
    none = s["row"][:0]
    before = s["kc"].clone()
    assert ops.rotate_write_kv(q[:0], empty, empty, s["cs"], s["table"], none, none, s["kc"], s["vc"]).shape == (0, 4, 128)
    assert torch.equal(before, s["kc"])


def test_rows_without_a_place_are_left_out(ops):
    """Positions outside the table of angles or of blocks, rows and blocks that do not exist."""
    s = make(12, 8, 2, 128, 128, 16, torch.float16, torch.int8, seed=9, num_positions=64)
    table, row, pos = (a.copy() for a in s["np"])
    pos[0], pos[1] = -1, 64                    # no row of cos_sin: nothing of the token is written
    row[2], row[3] = -1, 3                     # no row of the block table: the query is rotated
    s["cs"] = torch.cat([s["cs"], s["cs"][:16]])
    table_wide = s["table"].clone()
    pos[1] = 80
    pos[4] = 70                                # angles, but no block
    bad = int(np.argmax(pos == pos[5]))
    table_wide[row[5], pos[5] // 16] = 10000
    same = (row == row[5]) & (pos // 16 == pos[5] // 16)
    s["np"] = (table, row, pos)
    s["row"], s["pos"], s["table"] = torch.from_numpy(row).cuda(), torch.from_numpy(pos).cuda(), table_wide
    keep = ~same
    keep[[0, 1, 2, 3, 4]] = False
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    q_out = torch.full_like(s["q"], 3.0)
    got = call(ops, s, False, status=status, q_out=q_out)
    assert bad >= 0 and int(status.item()) == 1 | 2 | 8
    cs = s["cs"].cpu().numpy()
    turned = np.ones(12, bool)
    turned[[0, 1]] = False
    q = orc.rotate(s["q"].float().cpu().numpy(), cs[np.where(turned, pos, 0), :64], cs[np.where(turned, pos, 0), 64:], False)
    want_q = torch.where(torch.from_numpy(turned)[:, None, None], torch.from_numpy(q).half(), torch.tensor(3.0).half())
    assert torch.equal(got.cpu(), want_q)
    check(s, got, (want_q, *expect(s, False, keep)[1:]))


def test_zeros_small_scales_infinities_and_nan(ops):
    """A zero row has scale 1; rows whose scale is subnormal, infinite values and NaN stay in their own rows."""
    s = make(6, 2, 2, 64, 64, 16, torch.float32, torch.int8, seed=4, scale_dtype=torch.float32)
    k = s["k"].clone()
    k[0] = 0
    k[1] *= 1e-38
    k[2] *= 2e-37
    s["k"] = k
    q = s["q"].clone()
    q[3, 0, 5], q[4, 1, 40] = float("inf"), float("nan")
    s["q"] = q
    want = expect(s, False)
    got = call(ops, s, False)
    check(s, torch.nan_to_num(got, nan=123.0), (torch.nan_to_num(want[0], nan=123.0), *want[1:]))


def test_another_stream_and_a_captured_graph(ops):
    s = make(50, 8, 4, 128, 128, 16, torch.bfloat16, torch.int8, seed=11)
    want = expect(s, False)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call(ops, s, False)
    torch.cuda.current_stream().wait_stream(stream)
    check(s, got, want)
    out = torch.empty_like(s["q"])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        call(ops, s, False, q_out=out)
    for seed in (12, 13):
        n = make(50, 8, 4, 128, 128, 16, torch.bfloat16, torch.int8, seed=seed)
        for key in ("q", "k", "v", "cs", "table", "row", "pos"):
            s[key].copy_(n[key])
        for key in ("kc", "vc"):
            s[key].zero_()
        for key in ("ks", "vs"):
            s[key].fill_(7.0)
        s["np"] = n["np"]
        graph.replay()
        check(s, out, expect(s, False))


def test_both_backends_agree(ops):
    got = []
    saved = ops.BACKEND
    try:
        for backend in ("torch", "ctypes"):
            ops.BACKEND = backend
            for pool in (torch.int8, torch.bfloat16):
                s = make(70, 6, 2, 128, 64, 16, torch.bfloat16, pool, seed=3)
                got.append((call(ops, s, True), s["kc"], s["vc"], s["ks"], s["vs"]))
    finally:
        ops.BACKEND = saved
    for a, b in zip(got[:2], got[2:]):
        for x, y in zip(a, b):
            assert (x is None and y is None) or torch.equal(x, y)


def test_what_is_converted_and_refused(ops):
    """64-bit indexes, rows with other strides, and arguments that the op refuses."""
    T, Hq, Hkv, D, BS = 5, 4, 2, 64, 16
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(T, h, D, device="cuda", generator=g).half() for h in (Hq, Hkv, Hkv))
    table = ops.rope_table(40, D, device="cuda")
    bt = torch.tensor([[2, 0, 1]], dtype=torch.int32, device="cuda")
    row, pos = torch.zeros(T, dtype=torch.int32, device="cuda"), torch.arange(14, 14 + T, dtype=torch.int32, device="cuda")
    pools = [torch.zeros(4, BS, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(4)]
    want = ops.rotate_write_kv(q, k, v, table, bt, row, pos, *pools[:2])
    spread = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)  # noqa: E731
    got = ops.rotate_write_kv(spread(q), spread(k), spread(v), table.t().contiguous().t(), bt.long(), row.long().view(1, T), pos.long().view(1, T), *pools[2:])
    assert torch.equal(got, want) and torch.equal(pools[0], pools[2]) and torch.equal(pools[1], pools[3])
    args = dict(q=q, k_new=k, v_new=v, cos_sin=table, block_table=bt, seq_index=row, positions=pos, k_cache=pools[0], v_cache=pools[1])
    before = [t.clone() for t in pools[:2]]
    for kw in (dict(q=q[:4]), dict(q=q.float()), dict(q=q.cpu()), dict(q=q[:, :, :32]), dict(k_new=k[:, :1]), dict(v_new=v.float()), dict(cos_sin=table.half()),
               dict(cos_sin=table[:, :24]), dict(cos_sin=table.cpu()), dict(cos_sin=table[0]), dict(positions=pos[:3]), dict(seq_index=row.cpu()),
               dict(block_table=bt[0]), dict(k_cache=pools[0].to(torch.int8), v_cache=pools[1].to(torch.int8)), dict(v_cache=pools[1][:3])):
        with pytest.raises(ValueError):
            ops.rotate_write_kv(**{**args, **kw})
    assert all(torch.equal(a, b) for a, b in zip(before, pools))
