"""GPU: shared_prefix_attention against attention in 64 bits, one query row at a time.

Tolerance of a row with logits s, p = exp(s - max s), l = sum p, o = sum p v / l, A = sum p |v| / l (per dim):
* a logit is off by at most e = (u_q + u_k + D 2^-23) sum |q k| scale: u_q the rounding of Q to the operand type (0
  where it is the pool's; INT8: 15 bits of the row's largest, amax / 65024 a value), u_k that of a
  dequantised key (INT8: 2^-11), the last term the fp32 sums; that changes o by at most 2 e' max |v - o| <= 4 e' max|v|
  with e' = e^(e) - 1;
* every p v is rounded with p (and with the dequantised v, INT8: 2^-11): u_p A; a p below the type's normal range
  is off by half of the smallest step, n 2^-25 max|v| / l (fp16; INT8 times 127 steps);
* sums in fp32: n 2^-23 A; ex2 and the joins: 2^-18 A; the output: 2^-11 |o| + 2^-25.
The log-sum-exp is off by e' + 2^-18 + n 2^-23 and by 2^-11 of itself.
"""
import math

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def ops():
    from pie_b200 import ops as o
    assert torch.cuda.is_available()
    return o


class Problem:
    """Groups of sequences over common blocks.  ``groups``: (members, shared tokens); ``own``: keys of every sequence beyond
    its group's, alone: keys of sequences behind the last group.  Slots that hold no token are NaN (INT8: their scales)."""

    def __init__(self, groups, own, alone=(), Hq=8, Hkv=2, D=128, BS=16, pool=torch.float16, q_dtype=None, maxq=1, seed=0, layout="slots",
                 scale_dtype=torch.float16, per_block=False, q_len=None, spare=5):
        g = torch.Generator(device="cuda").manual_seed(seed)
        rng = np.random.default_rng(seed)
        dev = "cuda"
        lens, table_rows, nxt = [], [], 0
        for (n, shared), mine in zip(groups, own):
            full = shared // BS
            common = list(range(nxt, nxt + full))
            nxt += full
            for k in mine:
                total = full * BS + k
                more = -(-total // BS) - full
                table_rows.append(common + list(range(nxt, nxt + more)))
                nxt += more
                lens.append(total)
            assert len(mine) == n
        for k in alone:
            more = -(-k // BS)
            table_rows.append(list(range(nxt, nxt + more)))
            nxt += more
            lens.append(k)
        NB = nxt + spare
        names = rng.permutation(NB)
        B, cols = len(lens), max(1, max(map(len, table_rows)))
        table = np.full((B, cols), 10**6)  # what no sequence holds is out of the pool
        for b, r in enumerate(table_rows):
            table[b, :len(r)] = names[r]
        self.B, self.Hq, self.Hkv, self.D, self.BS, self.maxq = B, Hq, Hkv, D, BS, maxq
        held = torch.zeros(NB, BS, dtype=torch.bool, device=dev)
        for b, n in enumerate(lens):
            for i in range(-(-n // BS)):
                held[table[b, i], :min(BS, n - i * BS)] = True
        shape = (NB, BS, Hkv, D)
        self.ks = self.vs = None
        if pool == torch.int8:
            kv = [torch.randint(-127, 128, shape, dtype=torch.int8, device=dev, generator=g) for _ in range(2)]
            if per_block:
                sc = [(torch.rand(NB, Hkv, device=dev, generator=g) * 0.02 + 0.005).to(scale_dtype) for _ in range(2)]
            else:
                sc = [(torch.rand(NB, Hkv, BS, device=dev, generator=g) * 0.02 + 0.005).to(scale_dtype).transpose(1, 2) for _ in range(2)]
                for s in sc:
                    s[~held] = float("nan")
            self.ks, self.vs = sc
        else:
            kv = [torch.randn(shape, device=dev, generator=g).to(pool) for _ in range(2)]
            for t in kv:
                t[~held] = float("nan")
        if layout == "heads":
            kv = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in kv]
        self.K, self.V = kv
        self.q_dtype = q_dtype or (torch.bfloat16 if pool == torch.bfloat16 else torch.float16)
        self.Q = (torch.randn(B, Hq, maxq, D, device=dev, generator=g) * 1.5).to(self.q_dtype)
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device=dev)  # noqa: E731
        self.table, self.kv_len, self.blocks = i32(table), i32(lens), i32([len(r) for r in table_rows])
        self.q_len = i32([maxq] * B if q_len is None else q_len)
        starts = np.concatenate([[0], np.cumsum([n for n, _ in groups])])
        self.group_start, self.prefix_len = i32(starts), i32([s for _, s in groups])

    def args(self):
        return (self.Q, self.K, self.V, self.q_len, self.table, self.blocks, self.BS, self.kv_len, self.group_start, self.prefix_len, self.ks, self.vs)

    def keys(self, b):
        n = min(int(self.kv_len[b]), int(self.blocks[b]) * self.BS)
        ids = self.table[b, :-(-max(n, 0) // self.BS)].long()
        out = []
        for t, s in ((self.K, self.ks), (self.V, self.vs)):
            x = t[ids].double()
            if s is not None:
                x = x * (s[ids].double()[:, None, :, None] if s.dim() == 2 else s[ids].double()[..., None])
            out.append(x.flatten(0, 1)[:max(n, 0)])
        return out


def check(p, O, L, rows=None, scale=None):
    int8 = p.K.dtype == torch.int8
    operand = torch.float16 if int8 else p.K.dtype
    u_p = torch.finfo(operand).eps / 2 + (2.0**-11 if int8 else 0)
    u_q = torch.finfo(operand).eps / 2 if p.Q.dtype != operand else 0.0
    sc = scale or 1 / math.sqrt(p.D)
    G = p.Hq // p.Hkv
    for b in range(p.B) if rows is None else rows:
        n_rows = min(int(p.q_len[b]), p.maxq)
        if n_rows <= 0:
            continue
        k, v = (t.repeat_interleave(G, 1) for t in p.keys(b))  # [n, Hq, D]
        n = k.shape[0]
        for m in range(n_rows):
            seen = max(0, min(n, int(p.kv_len[b]) - n_rows + m + 1))
            o, lse = O[b, :, m].double(), L[b, :, m].double()
            if seen == 0:
                assert not o.any() and bool(torch.isneginf(lse).all()), (b, m)
                continue
            q = p.Q[b, :, m].double()
            s = torch.einsum("hd,nhd->hn", q, k[:seen]) * sc
            size = torch.einsum("hd,nhd->hn", q.abs(), k[:seen].abs()) * sc
            e = (size * (u_q + (2.0**-11 if int8 else 0) + p.D * 2.0**-23)).amax(1)
            if int8:
                e = e + (q.abs().amax(1)[:, None] / 65024 * k[:seen].abs().sum(2).T * sc).amax(1)
            e = torch.expm1(e)
            w = (s - s.amax(1, keepdim=True)).exp()
            l = w.sum(1)
            want = torch.einsum("hn,nhd->hd", w, v[:seen]) / l[:, None]
            A = torch.einsum("hn,nhd->hd", w, v[:seen].abs()) / l[:, None]
            vmax = v[:seen].abs().amax((0, 2))
            tiny = seen * 2.0**-25 * (127 if int8 else 1) * vmax.clamp(min=1) / l
            tol = 4 * (e * vmax)[:, None] + (u_p + seen * 2.0**-23 + 2.0**-18) * A + tiny[:, None] + 2.0**-11 * want.abs() + 2.0**-25
            assert bool(((o - want).abs() <= tol).all()), (b, m, ((o - want).abs() - tol).max().item(), (o - want).abs().max().item())
            ref = s.logsumexp(1)
            assert bool(((lse - ref).abs() <= e + 2.0**-18 + seen * 2.0**-23 + 2.0**-11 * ref.abs() + 2.0**-25).all()), (b, m)


def both(p, ops, monkeypatch, **kw):
    """The default kernels, and the split-K form for every group."""
    O, L = ops.shared_prefix_attention(*p.args(), **kw)
    check(p, O, L, scale=kw.get("softmax_scale"))
    monkeypatch.setenv("PIE_B200_NO_TCGEN05", "1")
    O2, L2 = ops.shared_prefix_attention(*p.args(), **kw)
    monkeypatch.delenv("PIE_B200_NO_TCGEN05")
    check(p, O2, L2, scale=kw.get("softmax_scale"))
    return O, L


POOLS = [torch.float16, torch.bfloat16, torch.int8]


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("BS", [1, 4, 8, 16, 64])
def test_groups_of_all_sizes(ops, monkeypatch, pool, D, BS):
    """Pairs, an odd group, a lone member, an empty group, sequences of no group; shared parts of one block to many tiles."""
    rng = np.random.default_rng(BS)
    groups = [(2, 64), (5, 320), (1, 200), (0, 500), (9, 129 + BS), (3, 1000)]
    own = [rng.integers(1, 90, n).tolist() for n, _ in groups]
    p = Problem(groups, own, alone=[1, 33, 300], D=D, BS=BS, pool=pool, seed=BS + D)
    both(p, ops, monkeypatch)


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("Hq,Hkv,maxq", [(1, 1, 1), (16, 1, 1), (6, 2, 1), (20, 4, 2), (8, 8, 1), (4, 4, 7), (10, 2, 3), (32, 8, 4), (24, 2, 1)])
def test_heads_and_rows(ops, monkeypatch, pool, Hq, Hkv, maxq):
    """One row to sixteen columns a KV head, rows that do not fill a tile, sequences with fewer rows than the longest."""
    rng = np.random.default_rng(Hq)
    groups = [(7, 176), (4, 400), (2, 32)]
    own = [rng.integers(maxq, 40, n).tolist() for n, _ in groups]
    q_len = rng.integers(1, maxq + 1, 13).tolist()
    q_len[3], q_len[12] = maxq, 0
    p = Problem(groups, own, Hq=Hq, Hkv=Hkv, maxq=maxq, pool=pool, seed=Hq + maxq, q_len=q_len)
    out = torch.full_like(p.Q, 7.0, dtype=torch.float16)
    lse = torch.full(p.Q.shape[:3], 7.0, dtype=torch.float16, device="cuda")
    ops.shared_prefix_attention(*p.args(), out=out, lse=lse)
    check(p, out, lse)
    for b, n in enumerate(q_len):  # rows behind a sequence's last stay as they were
        assert bool((out[b, :, n:] == 7).all()) and bool((lse[b, :, n:] == 7).all())
    both(p, ops, monkeypatch)


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("n,shared,Hq", [(64, 2048, 8), (33, 4097, 8), (100, 640, 4), (3, 20000, 2), (130, 1280, 2), (257, 144, 2)])
def test_many_members_and_long_prefixes(ops, monkeypatch, pool, n, shared, Hq):
    """Several tiles of rows and of keys, split over the GPU."""
    rng = np.random.default_rng(n)
    p = Problem([(n, shared)], [rng.integers(1, 60, n).tolist()], Hq=Hq, Hkv=2, pool=pool, seed=n)
    O, L = both(p, ops, monkeypatch)
    # the same attention, every sequence by itself: both within the tolerance above of 64 bits, so within twice of each other
    O2, L2 = ops.paged_attention(*p.args()[:8], p.ks, p.vs)
    check(p, O2, L2, rows=range(0, n, 17))


@pytest.mark.parametrize("pool", POOLS)
def test_what_is_shared_is_cut_to_what_every_row_sees(ops, monkeypatch, pool):
    """Members that end inside the prefix, without keys or rows, prefixes beyond every member, not of whole blocks, negative."""
    p = Problem([(4, 160), (3, 96), (4, 320), (2, 64)], [[1, 5, 9, 2], [7, 8, 9], [3, 50, 60, 1], [4, 4]], pool=pool, maxq=2, seed=3,
                q_len=[2, 1, 2, 1, 2, 2, 2, 1, 2, 0, 2, 1, 2])
    p.prefix_len[:] = torch.tensor([100000, 95, 320, -3], dtype=torch.int32)
    p.kv_len[1] = 40     # ends inside its group's prefix
    p.kv_len[4] = 0      # no keys: does not count
    p.blocks[4] = 0
    p.table[4] = 10**6
    p.kv_len[7], p.blocks[7] = 333, 3   # keys beyond its blocks: 48 are left
    p.kv_len[10] = 1     # one key for two rows: the first row sees none, so the group shares nothing
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    both(p, ops, monkeypatch, status=status)
    assert int(status.item()) == 0


@pytest.mark.parametrize("pool", POOLS)
def test_bad_groups_and_bad_blocks(ops, monkeypatch, pool):
    """Starts that fall or leave the batch: nothing is shared, the result is that of plain attention; blocks outside the pool are skipped."""
    p = Problem([(4, 160), (4, 160)], [[1, 5, 9, 2], [3, 4, 5, 6]], pool=pool, seed=4)
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    good = p.group_start.clone()
    for bad in ([0, 6, 4], [-1, 4, 8], [0, 4, 9], [2**31 - 1, 0, 1]):
        p.group_start = torch.tensor(bad, dtype=torch.int32, device="cuda")
        both(p, ops, monkeypatch, status=status)
        assert int(status.item()) == 8
        status.zero_()
    p.group_start = good
    p.table[4:, 3] = 999999
    O, L = ops.shared_prefix_attention(*p.args(), status=status)
    assert int(status.item()) == 1
    check(p, O, L, rows=range(4))
    assert bool(torch.isfinite(O).all())


@pytest.mark.parametrize("pool", [torch.int8])
@pytest.mark.parametrize("scale_dtype,per_block", [(torch.float32, False), (torch.float32, True), (torch.float16, True)])
def test_scales(ops, monkeypatch, pool, scale_dtype, per_block):
    p = Problem([(20, 300), (6, 64)], [[5] * 20, [40] * 6], pool=pool, scale_dtype=scale_dtype, per_block=per_block, seed=5)
    both(p, ops, monkeypatch)


@pytest.mark.parametrize("pool", POOLS)
def test_layouts_strides_types_and_scale(ops, monkeypatch, pool):
    """[block, head, slot, d] pools, Q and out with strides, the other 16-bit type and fp32 for Q, a softmax scale."""
    p = Problem([(24, 208), (3, 64)], [[9] * 24, [30] * 3], pool=pool, layout="heads", seed=6, maxq=2)
    both(p, ops, monkeypatch, softmax_scale=0.2)
    p.Q = p.Q.transpose(1, 2).contiguous().transpose(1, 2)
    out = torch.zeros(p.B, 2, p.Hq, 136, dtype=torch.float16, device="cuda")[..., :128].transpose(1, 2)
    lse = torch.zeros(p.B, 2, p.Hq, dtype=torch.float16, device="cuda").transpose(1, 2)
    both(p, ops, monkeypatch, out=out, lse=lse)
    for t in (torch.float16, torch.bfloat16):
        p.Q = p.Q.to(t)
        both(p, ops, monkeypatch)
    q32 = p.Q.float()
    O, L = ops.shared_prefix_attention(q32, *p.args()[1:])
    check(p, O, L)


def test_no_groups_no_sequences(ops, monkeypatch):
    p = Problem([], [], alone=[5, 100, 1], seed=7)
    both(p, ops, monkeypatch)
    e = Problem([(4, 64)], [[1, 2, 3, 4]], seed=8)
    O, L = ops.shared_prefix_attention(e.Q[:0], e.K, e.V, e.q_len[:0], e.table[:0], e.blocks[:0], 16, e.kv_len[:0],
                                       e.group_start[:1], e.prefix_len[:0])
    assert O.shape == (0, 8, 1, 128) and L.shape == (0, 8, 1)


@pytest.mark.parametrize("pool", POOLS)
def test_infinite_and_extreme_logits(ops, monkeypatch, pool):
    """Logits hundreds apart: the running maximum moves in most tiles; a row's NaN stays in its row."""
    p = Problem([(40, 700)], [[3] * 40], Hq=4, Hkv=2, pool=pool, seed=9)
    p.Q = p.Q * 30
    both(p, ops, monkeypatch)
    p.Q = p.Q / 30
    p.Q[7, 1] = float("nan")
    p.Q[9, 2] = 0
    for env in (None, "1"):
        if env:
            monkeypatch.setenv("PIE_B200_NO_TCGEN05", env)
        O, L = ops.shared_prefix_attention(*p.args())
        if pool != torch.int8:
            assert bool(torch.isnan(O[7, 1]).all())
        check(p, O, L, rows=[b for b in range(40) if b != 7])
        q = p.Q.clone()
        q[7, 1] = 0
        O2, L2 = ops.shared_prefix_attention(q, *p.args()[1:])
        other = torch.ones(40, 4, dtype=torch.bool, device="cuda")
        other[7, 1] = False
        assert torch.equal(O[other], O2[other]) and torch.equal(L[other], L2[other])


@pytest.mark.parametrize("pool", POOLS)
def test_replays_streams_and_repeats(ops, pool):
    """A captured call on new data, calls on two streams at once, and the same call twice: bit for bit the eager result."""
    mk = lambda seed: Problem([(40, 1600), (6, 320)], [[9] * 40, [30] * 6], pool=pool, seed=seed)  # noqa: E731
    p = mk(10)
    O, L = ops.shared_prefix_attention(*p.args())
    check(p, O, L, rows=range(0, 46, 9))
    again = ops.shared_prefix_attention(*p.args())
    assert torch.equal(O, again[0]) and torch.equal(L, again[1])
    others = [mk(s) for s in (11, 12, 13, 14)]
    eager = [ops.shared_prefix_attention(*o.args()) for o in others]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in others]
    got = []
    for _ in range(3):
        for o, s in zip(others, streams):
            with torch.cuda.stream(s):
                got.append(ops.shared_prefix_attention(*o.args()))
    torch.cuda.synchronize()
    for i, (a, l) in enumerate(got):
        assert torch.equal(a, eager[i % 4][0]) and torch.equal(l, eager[i % 4][1])
    graph, graph2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        cap = ops.shared_prefix_attention(*p.args())
    q = mk(12)
    with torch.cuda.graph(graph2):
        cap2 = ops.shared_prefix_attention(*q.args())
    for i, o in enumerate(others):
        for name in ("Q", "K", "V", "q_len", "table", "blocks", "kv_len", "group_start", "prefix_len") + (("ks", "vs") if pool == torch.int8 else ()):
            getattr(p, name).copy_(getattr(o, name))
        torch.cuda.synchronize()
        with torch.cuda.stream(streams[0]):
            graph.replay()
        with torch.cuda.stream(streams[1]):
            graph2.replay()
        torch.cuda.synchronize()
        assert torch.equal(cap[0], eager[i][0]) and torch.equal(cap[1], eager[i][1])
        assert torch.equal(cap2[0], eager[1][0]) and torch.equal(cap2[1], eager[1][1])


@pytest.mark.parametrize("pool", POOLS)
def test_both_backends_agree(ops, pool):
    p = Problem([(20, 500)], [[9] * 20], alone=[70], pool=pool, seed=15)
    saved, got = ops.BACKEND, []
    try:
        for ops.BACKEND in ("torch", "ctypes"):
            got.append(ops.shared_prefix_attention(*p.args()))
    finally:
        ops.BACKEND = saved
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])


def test_a_full_batch(ops, monkeypatch):
    """4096 sequences in 1000 groups."""
    rng = np.random.default_rng(0)
    sizes = np.full(1000, 4)
    groups = [(4, int(s)) for s in rng.integers(0, 80, 1000)]
    p = Problem(groups, [rng.integers(1, 20, 4).tolist() for _ in sizes], alone=[3] * 96, Hq=2, Hkv=1, D=64, BS=8, seed=16)
    for env in ("0", "1"):
        if env == "1":
            monkeypatch.setenv("PIE_B200_NO_TCGEN05", env)
        O, L = ops.shared_prefix_attention(*p.args())
        check(p, O, L, rows=rng.integers(0, 4096, 60).tolist())
    with pytest.raises(RuntimeError, match="4096"):
        ops.shared_prefix_attention(torch.cat([p.Q, p.Q[:1]]), p.K, p.V, torch.cat([p.q_len, p.q_len[:1]]), torch.cat([p.table, p.table[:1]]),
                                    torch.cat([p.blocks, p.blocks[:1]]), 8, torch.cat([p.kv_len, p.kv_len[:1]]), p.group_start, p.prefix_len)


def test_what_is_converted_and_refused(ops):
    """64-bit metadata, float32 queries, the pool with heads in front, and arguments that the op refuses."""
    p = Problem([(3, 64)], [[5, 20, 1]], seed=11)
    Q, K, V, ql, bt, nb, BS, kl, gs, pl, _, _ = p.args()
    want = ops.shared_prefix_attention(*p.args())
    heads = [t.transpose(1, 2).contiguous() for t in (K, V)]
    got = ops.shared_prefix_attention(Q.float(), *heads, ql.long(), bt.long(), nb.long(), BS, kl.long(), gs.long(), pl.long())
    spread = ops.shared_prefix_attention(Q.transpose(1, 3).contiguous().transpose(1, 3), K, V, ql, bt, nb, BS, kl, gs, pl)
    assert all(torch.equal(a, b) and torch.equal(a, c) for a, b, c in zip(want, got, spread))
    args = dict(Q=Q, K=K, V=V, q_len_per_seq=ql, block_table=bt, num_blocks_per_seq=nb, block_size=BS, kv_len_per_seq=kl, group_start=gs, prefix_len=pl)
    for kw in (dict(Q=Q[0]), dict(Q=Q[..., :64]), dict(K=K[:, :8], V=V[:, :8]), dict(K=K.cpu()), dict(V=V.bfloat16()), dict(block_table=bt[:2]),
               dict(q_len_per_seq=ql[:2]), dict(kv_len_per_seq=kl.cpu()), dict(group_start=gs[:0]), dict(group_start=gs[:1]), dict(prefix_len=pl.view(1, 1)),
               dict(prefix_len=pl.cpu()), dict(K=K.to(torch.int8), V=V.to(torch.int8))):
        with pytest.raises(ValueError):
            ops.shared_prefix_attention(**{**args, **kw})
    with pytest.raises(RuntimeError, match="<= 16"):
        ops.shared_prefix_attention(**{**args, "Q": Q.repeat(1, 1, 5, 1)})
    with pytest.raises(RuntimeError, match="fp16, bf16 or int8"):
        ops.shared_prefix_attention(**{**args, "K": K.float(), "V": V.float()})


def test_two_calls_at_once(ops):
    """Two streams, and two graphs replayed together: a call's workspace is its own."""
    ps = [Problem([(40, 640), (9, 128)], [[3 + i % 50 for i in range(40)], [7] * 9], seed=s) for s in (1, 2)]
    wants = [ops.shared_prefix_attention(*p.args()) for p in ps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in ps]
    gots = [[], []]
    for _ in range(6):
        for i, p in enumerate(ps):
            with torch.cuda.stream(streams[i]):
                gots[i].append(ops.shared_prefix_attention(*p.args()))
    graphs, outs = [], []
    torch.cuda.synchronize()
    for p in ps:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(ops.shared_prefix_attention(*p.args()))
        graphs.append(g)
    for _ in range(4):
        for s, g in zip(streams, graphs):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for want, got, out in zip(wants, gots, outs):
        for o, l in got + [out]:
            assert torch.equal(o, want[0]) and torch.equal(l, want[1])
