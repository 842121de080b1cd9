"""GPU: beam selection against its definition in 64 bits.

Score tolerance: a score is base + x - lse, formed in 64 bits and rounded once to fp32 (2^-24 of its size).  The
sum behind lse adds V terms in fp32 along at most 2^8 additions per partial sum (2^-24 each); a term's exponential is
good to 2^-22, and its argument (x - m) log2 e, |x - m| <= 30 where a term still counts (e^-30 * 2^18 < 2^-24), carries
two roundings of 2^-24 and the constant's 2^-25: 30 * 1.45 * 2.5 * 2^-24.  In all below 2^-24 * (256 + 4 + 109) = 2.2e-5
in the sum's relative error, that is in lse.
Where two candidates lie nearer than twice that, either order is right.
"""
import numpy as np
import pytest
import torch

from oracle import beam_search as obs

pytestmark = pytest.mark.gpu
LSE = 369 * 2.0**-24


@pytest.fixture(params=["torch", "ctypes"])
def ops(request, monkeypatch):
    from pie_b200 import ops as o

    monkeypatch.setattr(o, "BACKEND", request.param)
    return o


def _check(got, logits, scores, n, finished=None, eos=-1, exact_order=False):
    s, t, p = (a.cpu().numpy() for a in got)
    x, base = logits.float().cpu().numpy(), scores.cpu().numpy()
    fin = None if finished is None else finished.cpu().numpy().astype(bool)
    ws, wt, wp = obs.select(x, base, n, fin, eos)
    assert s.dtype == np.float32 and t.dtype == p.dtype == np.int32
    tol = LSE + 2.0**-24 * np.abs(np.where(np.isfinite(ws), ws, 0))
    assert np.array_equal(np.isfinite(s), np.isfinite(ws))
    both = np.isfinite(ws)
    assert (np.abs(np.where(both, s, 0) - np.where(both, ws, 0)) <= tol).all()
    assert np.array_equal(s[~both], ws[~both].astype(np.float32))
    differ = (t != wt) | (p != wp)
    if exact_order:
        assert not differ.any()
    else:  # another order only among candidates that the tolerance does not tell apart
        gap = np.full(ws.shape, np.inf)
        with np.errstate(invalid="ignore"):
            d = np.abs(np.diff(ws, axis=1))
        d = np.where(np.isnan(d), np.inf, d)
        gap[:, 1:], gap[:, :-1] = np.minimum(gap[:, 1:], d), np.minimum(gap[:, :-1], d)
        gap[:, -1] = 0
        assert (gap[differ] <= 2 * tol[differ]).all()
        flat = p.astype(np.int64) * x.shape[2] + t
        assert all(len(set(r)) == n for r in flat)


CASES = [  # seqs, beams, vocab, out
    (1, 1, 1, 1), (1, 2, 1, 2), (3, 1, 7, 7), (2, 4, 31, 8), (1, 32, 40, 32), (5, 3, 257, 6), (2, 5, 4096, 10),
    (1, 1, 8191, 32), (3, 2, 8193, 4), (2, 8, 50257, 16), (1, 4, 131072, 8), (40, 6, 1000, 12), (1, 7, 200003, 13),
    (300, 2, 3000, 3)]


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n", CASES)
def test_matches_the_definition(ops, B, K, V, n, dtype):
    g = torch.Generator(device="cuda").manual_seed(B * 1000 + V)
    x = (torch.randn(B, K, V, device="cuda", generator=g) * 3).to(dtype)
    s = -torch.rand(B, K, device="cuda", generator=g) * 30
    _check(ops.beam_select(x, s, n), x, s, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("offset", [0, 1, 3, 7])
def test_rows_at_any_address(ops, dtype, offset):
    """Views: rows that start off a 16-byte boundary, padded rows, beams and sequences swapped in memory."""
    g = torch.Generator(device="cuda").manual_seed(5)
    big = (torch.randn(4, 3, 9000, device="cuda", generator=g) * 2).to(dtype)
    s = -torch.rand(3, 4, device="cuda", generator=g)
    x = big.transpose(0, 1)[:, :, offset:offset + 8501]
    assert x.stride(2) == 1 and not x.is_contiguous()
    _check(ops.beam_select(x, s, 8), x, s, 8)
    y = big.transpose(1, 2).contiguous().transpose(1, 2)[:3]  # the vocabulary is not contiguous: copied
    _check(ops.beam_select(y, s.t().contiguous()[:3], 6), y, s.t().contiguous()[:3], 6)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("n", [1, 5, 32])
def test_ties_go_to_the_lowest(ops, dtype, n):
    """Equal logits, few distinct values, rising and falling rows: lower beam, then larger logit, then lower token."""
    V = 20001
    flat = torch.zeros(1, 3, V, device="cuda", dtype=dtype)
    s0 = torch.zeros(1, 3, device="cuda")
    _check(ops.beam_select(flat, s0, n), flat, s0, n, exact_order=True)
    _check(ops.beam_select(flat - 0.0, -s0, n), flat, s0, n, exact_order=True)
    zeros = torch.where(torch.arange(V, device="cuda") % 2 == 0, -0.0, 0.0).to(dtype).expand(1, 3, V)
    _check(ops.beam_select(zeros, s0, n), zeros, s0, n, exact_order=True)  # -0 is 0
    g = torch.Generator(device="cuda").manual_seed(n)
    few = torch.randint(0, 3, (1, 1, V), device="cuda", generator=g).to(dtype).expand(1, 3, V)
    _check(ops.beam_select(few, s0, n), few, s0, n, exact_order=True)
    rise = torch.arange(V, device="cuda").to(dtype).expand(1, 2, V) / 16
    _check(ops.beam_select(rise, s0[:, :2].contiguous(), n), rise, s0[:, :2], n, exact_order=True)
    _check(ops.beam_select(rise.flip(2), s0[:, :2].contiguous(), n), rise.flip(2), s0[:, :2], n, exact_order=True)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_masked_and_extreme_logits(ops, dtype):
    """-inf masks (whole rows too), the type's lowest value, NaN, +inf, scores of -inf and NaN."""
    V, n = 5003, 12
    g = torch.Generator(device="cuda").manual_seed(9)
    x = (torch.randn(9, 4, V, device="cuda", generator=g) * 2).to(dtype)
    s = -torch.rand(9, 4, device="cuda", generator=g) * 5
    lowest = torch.finfo(dtype).min
    inf = float("inf")
    x[0, 1] = -inf                      # a beam without any token
    x[1] = -inf                         # no beam has one
    x[2, :, 3:] = -inf                  # three tokens a beam: fewer than n in a beam, enough in all
    x[3, 0, :] = lowest                 # a row of the mask value is uniform
    x[3, 2, 10:] = lowest
    x[4, :, ::3] = float("nan")
    x[5, 0, [7, 5000]] = inf            # +inf counts as the largest float: two equal maxima
    x[5, 1] = float("nan")
    s[6, [0, 2]] = -inf                 # beams not started yet
    s[7, 1] = float("nan")
    x[8, :, 0] = lowest
    x[8, :, 1:] = -inf
    _check(ops.beam_select(x, s, n), x, s, n)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_runs_of_nan(ops, dtype):
    """Stretches of NaN that fill whole threads, warps and parts beside ordinary logits."""
    V = 40013
    g = torch.Generator(device="cuda").manual_seed(12)
    x = (torch.randn(4, 2, V, device="cuda", generator=g) * 2).to(dtype)
    s = -torch.rand(4, 2, device="cuda", generator=g)
    x[0, :, 100:9000] = float("nan")
    x[1, :, 8:] = float("nan")
    x[2, 0, :-3] = float("nan")
    x[2, 1, 20000:] = float("nan")
    x[3].view(2, -1)[:, 1024:2048] = float("nan")
    _check(ops.beam_select(x, s, 9), x, s, 9)


@pytest.mark.parametrize("shift", [-3e4, 8000.25, 12345.625, 1e6, -1e30])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_logits_far_from_zero(ops, dtype, shift):
    """Only differences of logits count: a common shift of any size leaves the sums as good."""
    if dtype == torch.float16 and abs(shift) > 6e4:
        pytest.skip("past fp16")
    g = torch.Generator(device="cuda").manual_seed(14)
    x = (torch.randn(2, 3, 9001, device="cuda", generator=g) * 2 + shift).to(dtype)
    s = -torch.rand(2, 3, device="cuda", generator=g)
    _check(ops.beam_select(x, s, 9), x, s, 9)


def test_beams_with_scores_of_very_different_size(ops):
    """A beam at 1e6 whose candidates come back to ordinary scores: its fp32 sums are coarse, the others' must not suffer."""
    V = 5000
    g = torch.Generator(device="cuda").manual_seed(13)
    x = torch.randn(3, 3, V, device="cuda", generator=g)
    x[:, 0, 77] = 1e6                       # log-sum-exp 1e6: token v scores 1e6 + (x - 1e6)
    x[:, 2, 11] = -1e6
    s = torch.tensor([1e6, 11.5, 11.0], device="cuda").expand(3, 3).contiguous()
    for n in (1, 7, 16, 32):
        _check(ops.beam_select(x, s, n), x, s, n)


@pytest.mark.parametrize("n", [2, 16, 32])
def test_coarse_sums_of_another_beam_do_not_hide_a_candidate(ops, n):
    """Beam 0's scores pass 1e6, where fp32 steps by 1/16: 0.04 is 0.0625 there, above beam 1's 0.05."""
    x = torch.full((1, 2, 4096), 0.04, device="cuda")
    x[0, 0, 77] = 1e6
    x[0, 1] = -100.0
    x[0, 1, 5] = 0.0
    s = torch.tensor([[1e6, 0.05]], device="cuda")
    got = ops.beam_select(x, s, n)
    _check(got, x, s, n, exact_order=True)
    assert got[2][0, :2].tolist() == [0, 1] and got[1][0, :2].tolist() == [77, 5]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_finished_beams(ops, dtype):
    B, K, V, n, eos = 6, 4, 10007, 8, 17
    g = torch.Generator(device="cuda").manual_seed(3)
    x = (torch.randn(B, K, V, device="cuda", generator=g) * 2).to(dtype)
    s = -torch.rand(B, K, device="cuda", generator=g) * 8
    fin = torch.rand(B, K, device="cuda", generator=g) < 0.5
    fin[0] = True       # all: more candidates asked for than there are finite ones
    fin[1] = False
    fin[2, 1:] = True
    s[3, 2] = -float("inf")
    fin[3, 2] = True
    x[fin] = float("nan")  # not read
    _check(ops.beam_select(x, s, n, finished=fin, eos_id=eos), x, s, n, fin, eos)
    _check(ops.beam_select(x, s, n, finished=fin.to(torch.uint8), eos_id=eos), x, s, n, fin, eos)
    for V2, e in ((3, 0), (3, 2), (5, 3)):
        y = x[:, :, :V2]
        _check(ops.beam_select(y, s, 6, finished=fin, eos_id=e), y, s, 6, fin, e)


def test_equal_rows_rank_equal_and_calls_repeat(ops):
    """Copies of one row give the same bits wherever they stand, and a call gives the same bits again."""
    g = torch.Generator(device="cuda").manual_seed(1)
    x = (torch.randn(1, 1, 60001, device="cuda", generator=g) * 3).bfloat16().expand(7, 5, 60001).contiguous()
    s = torch.zeros(7, 5, device="cuda")
    a, b = ops.beam_select(x, s, 15), ops.beam_select(x, s, 15)
    assert all(torch.equal(u, v) for u, v in zip(a, b))
    assert all((t == t[:1]).all() for t in a)
    _check([t[:1] for t in a], x[:1], s[:1], 15, exact_order=True)


def test_empty_batch_and_default_width(ops):
    x = torch.empty(0, 3, 100, device="cuda")
    got = ops.beam_select(x, torch.empty(0, 3, device="cuda"))
    assert [tuple(t.shape) for t in got] == [(0, 3)] * 3


def test_other_streams_and_two_captured_graphs(ops):
    """Two graphs of different shapes replayed at once on two streams, and an eager call between them."""
    g = torch.Generator(device="cuda").manual_seed(2)
    xs = [(torch.randn(B, K, 30011, device="cuda", generator=g) * 2).half() for B, K in ((4, 6), (9, 2))]
    ss = [-torch.rand(x.shape[:2], device="cuda", generator=g) for x in xs]
    want = [ops.beam_select(x, s, 6) for x, s in zip(xs, ss)]
    torch.cuda.synchronize()
    graphs, outs, streams = [], [], [torch.cuda.Stream(), torch.cuda.Stream()]
    for x, s in zip(xs, ss):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            outs.append(ops.beam_select(x, s, 6))
        graphs.append(gr)
    for _ in range(20):
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        ops.beam_select(xs[0], ss[0], 6)
    torch.cuda.synchronize()
    for w, o in zip(want, outs):
        assert all(torch.equal(a, b) for a, b in zip(w, o))
    xs[0].copy_(xs[0].flip(0))  # a replay reads the new inputs
    torch.cuda.synchronize()
    graphs[0].replay()
    torch.cuda.synchronize()
    _check(outs[0], xs[0], ss[0], 6)


def test_logits_past_two_to_the_31(ops):
    """The last sequence's logits lie more than 2^31 elements into the tensor."""
    V, B = 131072, 16385
    x = torch.empty(B, 1, V, dtype=torch.bfloat16, device="cuda")
    x[-1] = torch.randn(V, device="cuda").to(torch.bfloat16)
    x[0] = 0
    s = torch.zeros(2, 1, device="cuda")
    y = x.as_strided((2, 1, V), ((B - 1) * V, V, 1))  # sequence 1 starts at element 2^31
    _check(ops.beam_select(y, s, 4), y, s, 4)


def test_refusals_on_the_gpu(ops):
    x, s = torch.zeros(2, 3, 50, device="cuda"), torch.zeros(2, 3, device="cuda")
    for bad in (dict(s=s[:1]), dict(s=s.half()), dict(s=s.cpu()), dict(fin=torch.zeros(2, 2, dtype=torch.bool, device="cuda")),
                dict(fin=torch.zeros(2, 3, device="cuda"))):
        a = dict(s=s, fin=None) | bad
        with pytest.raises(ValueError):
            ops.beam_select(x, a["s"], 3, finished=a["fin"], eos_id=1)
    with pytest.raises(RuntimeError, match="num_out"):
        ops.beam_select(x, s, 33)
    with pytest.raises(RuntimeError, match="num_beams"):
        ops.beam_select(torch.zeros(1, 33, 50, device="cuda"), torch.zeros(1, 33, device="cuda"), 3)


@pytest.mark.parametrize("B,n", [(1, 3), (3, 7), (5, 32)])
def test_outputs_are_tensors_of_their_own(ops, tmp_path, B, n):
    """As the schema says: each starts a storage (compiled code takes that for 16-byte alignment), and all can be saved."""
    g = torch.Generator(device="cuda").manual_seed(B)
    x, s = torch.randn(B, 4, 1000, device="cuda", generator=g), torch.zeros(B, 4, device="cuda")
    got = ops.beam_select(x, s, n)
    assert [t.storage_offset() for t in got] == [0] * 3 and all(t.data_ptr() % 16 == 0 for t in got)
    assert len({t.untyped_storage().data_ptr() for t in got}) == 3
    assert all(t.untyped_storage().nbytes() == 4 * B * n for t in got)
    torch.save(got, tmp_path / "beams.pt")
    assert all(torch.equal(a, b) for a, b in zip(torch.load(tmp_path / "beams.pt"), got))


def test_compiled_call_with_odd_outputs():
    """Through torch.compile, whose generated code asserts the outputs' alignment; 1 x 3 outputs of 4 bytes."""
    from pie_b200 import _torch_ext

    op = _torch_ext.ops().beam_select
    x = torch.randn(1, 3, 500, device="cuda")
    s = torch.zeros(1, 3, device="cuda")
    want = op(x, s, 3, None, -1)
    got = torch.compile(lambda x, s: op(x, s, 3, None, -1), fullgraph=True)(x, s)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    torch.library.opcheck(op.default if hasattr(op, "default") else op, (x, s, 3, None, -1),
                          test_utils=("test_schema", "test_faketensor"))


# ---- parts of several units ------------------------------------------------------------
# With many rows a row has few parts, and a part several units (a unit: 4096 logits in fp32, 8192 in 16 bits).
LONG = [  # seqs, beams, vocab, out, units of a part in fp32 and in 16 bits at least
    (6, 16, 65536, 32, 2, 2), (760, 1, 33001, 4, 3, 2), (33, 16, 113435, 26, 7, 7), (32, 32, 152064, 16, 10, 10),
    (1, 32, 2**20, 32, 32, 16), (1, 32, 2**20 - 5, 32, 32, 16)]


def _part_units(dtype, B, K, V, n):
    import ctypes

    from pie_b200 import _lib

    lib, size = _lib.load(), ctypes.c_size_t(0)
    a = _lib.PaBeamSelect(dtype={torch.float32: 3, torch.float16: 0, torch.bfloat16: 1}[dtype], num_seqs=B, num_beams=K,
                          vocab=V, num_out=n, eos_id=-1)
    assert lib.beam_select_workspace_size(a, ctypes.byref(size)) == 0
    unit = 4096 if dtype == torch.float32 else 8192
    return -(-(-(-V // unit)) // (size.value // (B * K * (8 * n + 8))))


def _check_each(got, x, s, n, seqs=None, finished=None, eos=-1):
    """Every output scored again in 64 bits: its own score and the column's best must both be the returned one."""
    B, K, V = x.shape
    score, token, parent = got
    assert score.shape == token.shape == parent.shape == (B, n)
    assert (0 <= token).all() and (token < V).all() and (0 <= parent).all() and (parent < K).all()
    for b in range(B) if seqs is None else seqs:
        y = x[b].double().nan_to_num(nan=-np.inf, posinf=torch.finfo(torch.float32).max, neginf=-np.inf)
        top = y.amax(-1, keepdim=True)
        lp = y - torch.where(top.isinf(), 0.0, top)
        lp = torch.where(top.isinf(), -np.inf, lp - lp.exp().sum(-1, keepdim=True).log())
        if finished is not None:
            one = torch.full((V,), -np.inf, dtype=torch.float64, device=x.device)
            one[eos] = 0
            lp = torch.where(finished[b].bool()[:, None], one, lp)
        total = (s[b].double()[:, None] + lp).nan_to_num(nan=-np.inf, posinf=np.inf, neginf=-np.inf).flatten()
        want = total.topk(n).values
        at = parent[b].long() * V + token[b].long()
        assert at.unique().numel() == n
        mine, have = total[at], score[b].double()
        assert torch.equal(have.isinf(), want.isinf()) and torch.equal(mine.isinf(), want.isinf())
        some = ~want.isinf()
        tol = LSE + 2.0**-24 * want.abs()
        assert ((have - mine).abs()[some] <= tol[some]).all()
        assert ((have - want).abs()[some] <= tol[some]).all()
        assert ((want - mine)[some] <= 2 * tol[some]).all()  # no better candidate was left out
    return got


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n,u32,u16", LONG)
def test_parts_of_several_units(ops, B, K, V, n, u32, u16, dtype):
    """Independent logits, rows off 16-byte boundaries, then rising, flat and tied rows and runs of NaN."""
    assert _part_units(dtype, B, K, V, n) >= (u32 if dtype == torch.float32 else u16)
    g = torch.Generator(device="cuda").manual_seed(V)
    few = sorted({0, B // 2, B - 1})
    s = -torch.rand(B, K, device="cuda", generator=g) * 3
    R = min(B * K, 48)  # rows that differ; the others repeat them
    rows = (torch.randn(R, V + 3, device="cuda", generator=g) * 2.5).to(dtype)
    pick = torch.arange(B * K, device="cuda") % R
    x = rows[pick].view(B, K, V + 3)
    _check_each(ops.beam_select(x[..., :V], s, n), x[..., :V], s, n, few)
    _check_each(ops.beam_select(x[..., 3:], s, n), x[..., 3:], s, n, few)
    ramp = torch.arange(V, device="cuda", dtype=torch.float64) / V
    for y in (ramp * 0.5, ramp * 40 - 20, -ramp * 40, torch.zeros_like(ramp), (ramp * 7 * V).long() % 3 * 1.0):
        y = y.to(dtype).expand(B, K, V)
        got = _check_each(ops.beam_select(y, s, n), y, s, n, few)
        if not y[0, 0].any():  # flat: the best beam's lowest tokens
            best = s.argmax(1, keepdim=True).expand(B, n)
            assert torch.equal(got[2].long(), best) and torch.equal(got[1], torch.arange(n, device="cuda").int().expand(B, n))
    z = rows[:1, :V].clone()
    z[0, 9000:30000] = float("nan")
    z[0, V - 4000:] = float("nan")
    z[0, 2:4] = -float("inf")
    z = z.expand(B, K, V)
    _check_each(ops.beam_select(z, s, n), z, s, n, few)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_long_parts_with_finished_beams_and_masks(ops, dtype):
    """Rows of which a few tokens are allowed, spread over units and parts, beside finished beams."""
    B, K, V, n, eos = 40, 16, 100003, 20, 77
    assert _part_units(dtype, B, K, V, n) >= 5
    g = torch.Generator(device="cuda").manual_seed(8)
    x = (torch.randn(B, K, V, device="cuda", generator=g) * 2).to(dtype)
    s = -torch.rand(B, K, device="cuda", generator=g) * 3
    keep = torch.zeros(4, V, dtype=torch.bool, device="cuda")
    keep[0, torch.randperm(V, device="cuda", generator=g)[:50]] = True
    keep[1, [5, 60000, V - 1]] = True
    keep[2] = True
    keep[3, 70000:70100] = True
    x.masked_fill_(~keep[torch.arange(B, device="cuda") % 4][:, None], -float("inf"))
    fin = torch.rand(B, K, device="cuda", generator=g) < 0.3
    x[3].masked_fill_(x[3].isinf(), torch.finfo(dtype).min)
    _check_each(ops.beam_select(x, s, n, finished=fin, eos_id=eos), x, s, n, None, fin, eos)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("B,K,V,n", CASES)
def test_each_output_is_the_one_it_says(ops, B, K, V, n, dtype):
    """The identity of every output, the last one's too, by its score from the definition."""
    g = torch.Generator(device="cuda").manual_seed(B + 17 * V)
    x = (torch.randn(B, K, V, device="cuda", generator=g) * 3).to(dtype)
    s = -torch.rand(B, K, device="cuda", generator=g) * 30
    _check_each(ops.beam_select(x, s, n), x, s, n)
