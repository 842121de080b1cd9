"""GPU: adjust_logits (penalties for repeated tokens, biases, grammar masks).

Every operation is rounded to fp32 by itself, in a stated order, so the kernel
equals the same operations in numpy (fp32) bit for bit before the one rounding to
the output's type.  Against 64 bits: x / r or x * r is off by 2^-24 |x r^+-1|, freq n by 2^-24,
each of the three sums by 2^-24 of its result, so the whole by at most 5 * 2^-24 of the largest
magnitude on the way, and by half a step of the output's type.
"""
import numpy as np
import pytest
import torch

from oracle import decode_step as orc

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


@pytest.fixture(scope="module")
def ops():
    from pie_b200 import ops as o
    assert torch.cuda.is_available()
    return o


def pack(allowed: np.ndarray) -> torch.Tensor:
    """bool [M, V] -> int32 [M, ceil(V / 32)], bit v % 32 of word v // 32."""
    M, V = allowed.shape
    full = np.zeros((M, (V + 31) // 32 * 32), bool)
    full[:, :V] = allowed
    return torch.from_numpy(np.packbits(full, axis=1, bitorder="little").view(np.int32).copy()).cuda()


def make(R, V, L, dtype, seed=0, biases=2, masks=3):
    rng = np.random.default_rng(seed)
    x = torch.from_numpy(rng.normal(0, 3, (R, V)).astype(np.float32)).to(dtype)
    tokens = rng.integers(0, max(1, min(V, 3 * L // 2 + 1)), (R, L)).astype(np.int32) * 131 % V
    count = rng.integers(0, L + 1, R).astype(np.int32)
    return dict(x=x, tokens=tokens, count=count, prompt=(count * rng.random(R)).astype(np.int32),
                rep=rng.uniform(0.7, 1.6, R).astype(np.float32), pres=rng.uniform(-0.5, 1, R).astype(np.float32),
                freq=rng.uniform(-0.2, 0.5, R).astype(np.float32), bias=(rng.normal(0, 4, (biases, V)) * (rng.random((biases, V)) < 0.1)).astype(np.float32),
                bias_row=rng.integers(-1, biases, R).astype(np.int32), allowed=rng.random((masks, V)) < rng.random((masks, 1)),
                mask_row=rng.integers(-1, masks, R).astype(np.int32))


def cuda(a):
    return torch.from_numpy(np.ascontiguousarray(a)).cuda()


def call(ops, s, x=None, **kw):
    args = dict(tokens=cuda(s["tokens"]), num_tokens=cuda(s["count"]), prompt_len=cuda(s["prompt"]), repetition_penalty=cuda(s["rep"]),
                presence_penalty=cuda(s["pres"]), frequency_penalty=cuda(s["freq"]), bias=cuda(s["bias"]), bias_row=cuda(s["bias_row"]),
                mask=pack(s["allowed"]), mask_row=cuda(s["mask_row"]))
    args.update(kw)
    return ops.adjust_logits(s["x"].cuda() if x is None else x, **args)


def expect(s, dtype=np.float32):
    x = s["x"].double().numpy().astype(dtype)
    rows = []
    for r in range(x.shape[0]):
        n, p = max(0, min(int(s["count"][r]), s["tokens"].shape[1])), max(0, int(s["prompt"][r]))
        b, m = int(s["bias_row"][r]), int(s["mask_row"][r])
        rows.append(orc.adjust_row(x[r], s["tokens"][r, :n].tolist(), s["tokens"][r, p:n].tolist(), s["rep"][r], s["pres"][r], s["freq"][r],
                                   s["bias"][b] if 0 <= b < len(s["bias"]) else None, s["allowed"][m] if 0 <= m < len(s["allowed"]) else None))
    return np.stack(rows)


def same(got, want32, dtype):
    want = torch.from_numpy(want32).to(dtype)
    assert got.dtype == dtype and got.shape == want.shape
    got = got.cpu()
    nan = torch.isnan(want)
    assert torch.equal(torch.isnan(got), nan) and torch.equal(got.masked_fill(nan, 0), want.masked_fill(nan, 0))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,L", [(1, 1, 1), (3, 7, 5), (2, 31, 40), (4, 32, 33), (5, 8191, 300), (3, 8193, 2000), (2, 32000, 777), (9, 50257, 1500), (2, 131072, 9000)])
def test_equals_the_operations_one_by_one(ops, R, V, L, dtype):
    s = make(R, V, L, dtype, seed=V + L)
    want = expect(s)
    same(call(ops, s), want, dtype)
    out = torch.empty(R, V, device="cuda")
    assert call(ops, s, out=out) is out
    same(out, want, torch.float32)
    x = s["x"].cuda()
    assert call(ops, s, x=x, out=x) is x  # in place
    same(x, want, dtype)


@pytest.mark.parametrize("dtype", DTYPES)
def test_against_64_bits(ops, dtype):
    s = make(6, 5003, 900, dtype, seed=1)
    got, want = call(ops, s).double().cpu().numpy(), expect(s, np.float64)
    fine = np.isfinite(want)
    assert np.array_equal(fine, np.isfinite(got))
    # no step of a row passes this size: |x| max(r, 1 / r), |freq| n, |pres|, |bias| together
    size = 1.6 / 0.7 * s["x"].abs().double().max().item() + 0.5 * 900 + 1 + np.abs(s["bias"]).max()
    # the count of most tokens is small: a bound per value
    n = np.zeros_like(want)
    for r in range(6):
        for v in s["tokens"][r, s["prompt"][r]:s["count"][r]]:
            n[r, v] += 1
    size = np.minimum(size, 1.6 / 0.7 * np.abs(s["x"].double().numpy()) + 0.5 * n + 1 + np.abs(s["bias"]).max(0))
    tol = 5 * 2.0**-24 * size
    tol = tol + torch.finfo(dtype).eps / 2 * (np.abs(np.where(fine, want, 0)) + tol) + torch.finfo(dtype).tiny
    assert (np.abs(np.where(fine, got - np.where(fine, want, 0), 0)) <= tol).all()


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("off,off_out", [(0, 0), (1, 1), (3, 0), (0, 5), (7, 6)])
def test_rows_at_any_address(ops, dtype, off, off_out):
    """Rows, outputs, biases and tokens that start off a 16-byte boundary, padded rows; what lies around stays as it was."""
    R, V = 4, 9001
    s = make(R, V, 200, dtype, seed=off)
    big = torch.full((R, V + 19), 5.0, dtype=dtype, device="cuda")
    x = big[:, off:off + V]
    x.copy_(s["x"])
    bias = torch.zeros(2, V + 3, device="cuda")[:, 1:V + 1].copy_(cuda(s["bias"]))
    tokens = torch.zeros(R, 203, dtype=torch.int32, device="cuda")[:, 2:202].copy_(cuda(s["tokens"]))
    for t in {dtype, torch.float32}:
        wide = torch.full((R, V + 23), 9.0, dtype=t, device="cuda")
        out = wide[:, off_out:off_out + V]
        call(ops, s, x=x, out=out, bias=bias, tokens=tokens)
        same(out, expect(s), t)
        assert bool((wide[:, :off_out] == 9).all()) and bool((wide[:, off_out + V:] == 9).all())
    call(ops, s, x=x, out=x, bias=bias, tokens=tokens)
    same(x, expect(s), dtype)
    assert bool((big[:, :off] == 5).all()) and bool((big[:, off + V:] == 5).all())


@pytest.mark.parametrize("dtype", DTYPES)
def test_each_part_alone_and_default_rows(ops, dtype):
    s = make(4, 4099, 60, dtype, seed=3, biases=4, masks=4)
    x = s["x"].cuda()
    none = dict(rep=np.ones(4, np.float32), pres=np.zeros(4, np.float32), freq=np.zeros(4, np.float32), bias_row=np.full(4, -1), mask_row=np.full(4, -1))
    same(ops.adjust_logits(x), expect({**s, **none}), dtype)
    same(ops.adjust_logits(x, bias=cuda(s["bias"])), expect({**s, **none, "bias_row": np.arange(4)}), dtype)
    same(ops.adjust_logits(x, bias=cuda(s["bias"][2])), expect({**s, **none, "bias_row": np.full(4, 2)}), dtype)
    same(ops.adjust_logits(x, mask=pack(s["allowed"])), expect({**s, **none, "mask_row": np.arange(4)}), dtype)
    same(ops.adjust_logits(x, mask=pack(s["allowed"])[1]), expect({**s, **none, "mask_row": np.full(4, 1)}), dtype)
    # numbers for all rows; all tokens count, all as generated
    every = dict(count=np.full(4, 60), prompt=np.zeros(4, int), rep=np.full(4, 1.3, np.float32), pres=np.full(4, 0.25, np.float32), freq=np.full(4, 0.1, np.float32))
    got = ops.adjust_logits(x, tokens=cuda(s["tokens"]), repetition_penalty=1.3, presence_penalty=0.25, frequency_penalty=0.1)
    same(got, expect({**s, **none, **every}), dtype)
    # only the prompt: no generated token
    got = ops.adjust_logits(x, tokens=cuda(s["tokens"]), prompt_len=cuda(np.full(4, 60, np.int32)), repetition_penalty=1.3, presence_penalty=0.25, frequency_penalty=0.1)
    same(got, expect({**s, **none, **every, "prompt": np.full(4, 60)}), dtype)
    # [B, K, V] with its own leading dims, 64-bit indexes
    got = ops.adjust_logits(x.view(2, 2, -1), tokens=cuda(s["tokens"]).view(2, 2, -1).long(), num_tokens=cuda(s["count"]).view(2, 2).long(), repetition_penalty=cuda(s["rep"]).view(2, 2))
    same(got.view(4, -1), expect({**s, **none, "rep": s["rep"]}), dtype)
    # beams and sequences swapped in memory, a vocabulary that is not contiguous
    y = x.view(2, 2, -1).transpose(0, 1)
    same(ops.adjust_logits(y, bias=cuda(s["bias"])).reshape(4, -1), expect({**s, "x": s["x"][[0, 2, 1, 3]], **none, "bias_row": np.arange(4)}), dtype)
    same(ops.adjust_logits(x.t().contiguous().t(), mask=pack(s["allowed"])), expect({**s, **none, "mask_row": np.arange(4)}), dtype)
    assert ops.adjust_logits(x[:0]).shape == (0, 4099)
    one = torch.zeros(4099, device="cuda", dtype=dtype)
    assert torch.equal(ops.adjust_logits(one, tokens=torch.tensor([3, 3], device="cuda"), frequency_penalty=0.5)[2:5].cpu(), torch.tensor([0, -1.0, 0], dtype=dtype))


@pytest.mark.parametrize("dtype", DTYPES)
def test_infinities_nan_and_rows_without_a_token(ops, dtype):
    s = make(5, 1037, 80, dtype, seed=6)
    x = s["x"]
    x[0, ::3] = float("inf")
    x[1, ::2] = float("-inf")
    x[2, 5:900] = float("nan")
    x[3] = torch.finfo(dtype).min
    s["allowed"][0] = False           # nothing may follow
    s["mask_row"][:] = [0, -1, 0, -1, 1]
    s["bias_row"][:] = [-1, 0, 1, -1, -1]
    s["bias"][0, 100:200] = float("-inf")
    s["bias"][1, ::7] = float("nan")
    same(call(ops, s), expect(s), dtype)


def test_ids_lengths_and_rows_outside(ops):
    """Token ids outside the vocabulary, lengths outside the list, bias and mask rows that do not exist."""
    s = make(6, 3001, 50, torch.float32, seed=7)
    s["tokens"][:, ::4] = -1
    s["tokens"][:, 1::4] = 3001
    s["tokens"][2, 2] = 2**31 - 1
    s["count"][:] = [-5, 0, 50, 51, 1000, 10]
    s["prompt"][:] = [0, 3, -2, 60, 10, 11]
    s["bias_row"][:] = [-1, 0, 1, 2, -2, 0]
    s["mask_row"][:] = [0, 1, 2, -1, 3, 100]
    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    same(call(ops, s, status=status), expect(s), torch.float32)
    assert int(status.item()) == 8


def test_many_repeats_of_one_token(ops):
    """Counts beyond 16 bits."""
    L = 70001
    tokens = torch.full((1, L), 4, dtype=torch.int32, device="cuda")
    x = torch.zeros(1, 9, device="cuda")
    got = ops.adjust_logits(x, tokens=tokens, frequency_penalty=0.5, presence_penalty=0.25)
    assert got[0].tolist() == [0, 0, 0, 0, -0.5 * L - 0.25, 0, 0, 0, 0]


def test_another_stream_and_a_captured_graph(ops):
    s = make(5, 20011, 100, torch.bfloat16, seed=20)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        got = call(ops, s)
    torch.cuda.current_stream().wait_stream(stream)
    same(got, expect(s), torch.bfloat16)
    t = dict(tokens=cuda(s["tokens"]), num_tokens=cuda(s["count"]), prompt_len=cuda(s["prompt"]), repetition_penalty=cuda(s["rep"]), presence_penalty=cuda(s["pres"]),
             frequency_penalty=cuda(s["freq"]), bias=cuda(s["bias"]), bias_row=cuda(s["bias_row"]), mask=pack(s["allowed"]), mask_row=cuda(s["mask_row"]))
    x = s["x"].cuda()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.adjust_logits(x, **t)
    for seed in (21, 22):
        n = make(5, 20011, 100, torch.bfloat16, seed=seed)
        x.copy_(n["x"])
        for key, a in (("tokens", "tokens"), ("num_tokens", "count"), ("prompt_len", "prompt"), ("repetition_penalty", "rep"), ("presence_penalty", "pres"),
                       ("frequency_penalty", "freq"), ("bias", "bias"), ("bias_row", "bias_row"), ("mask_row", "mask_row")):
            t[key].copy_(torch.from_numpy(n[a]))
        t["mask"].copy_(pack(n["allowed"]))
        graph.replay()
        same(out, expect(n), torch.bfloat16)


def test_both_backends_agree(ops):
    s = make(7, 12345, 300, torch.bfloat16, seed=30)
    saved = ops.BACKEND
    try:
        got = []
        for backend in ("torch", "ctypes"):
            ops.BACKEND = backend
            got.append((call(ops, s), call(ops, s, out=torch.empty(7, 12345, device="cuda")), ops.adjust_logits(s["x"].cuda())))
    finally:
        ops.BACKEND = saved
    assert all(torch.equal(a, b) for a, b in zip(*got))


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("R,V,L", [(80, 32003, 300), (20, 131072, 2600), (1200, 2100, 50)])
def test_many_columns(ops, dtype, R, V, L):
    """Enough columns for the wide pieces and for spans of several chunks; also in place."""
    s = make(R, V, L, dtype, seed=R)
    want = expect(s)
    same(call(ops, s), want, dtype)
    x = s["x"].cuda()
    assert call(ops, s, x=x, out=x) is x
    same(x, want, dtype)


def test_spans_with_many_tokens(ops):
    """A long history over several spans, each column seen more than once, counts of 32 bits."""
    s = make(30, 90001, 66000, torch.bfloat16, seed=5)
    s["count"][:] = 66000
    s["prompt"][:15] = 0
    got = call(ops, s)
    rows = [0, 7, 16, 29]
    part = {k: (v if k in ("bias", "allowed") else v[rows]) for k, v in s.items()}
    same(got[rows], expect(part), torch.bfloat16)


def test_what_is_converted(ops):
    """Leading dimensions, 64-bit integers, penalties and biases of other types, one bias and one mask for all rows."""
    V, L = 4099, 33
    s = make(6, V, L, torch.float16, seed=8, biases=1, masks=1)
    s["bias_row"][:] = 0
    s["mask_row"][:] = 0
    want = expect(s)
    kw = dict(tokens=cuda(s["tokens"]).long().view(2, 3, L), num_tokens=cuda(s["count"]).long().view(2, 3), prompt_len=cuda(s["prompt"]).view(2, 3),
              repetition_penalty=cuda(s["rep"]).double().view(2, 3), presence_penalty=cuda(s["pres"]).view(2, 3), frequency_penalty=cuda(s["freq"]).view(6, 1),
              bias=cuda(s["bias"][0]).double(), mask=pack(s["allowed"])[0])
    x = s["x"].cuda().view(2, 3, V)
    got = ops.adjust_logits(x, **kw)
    assert got.shape == (2, 3, V)
    same(got.view(6, V), want, torch.float16)
    out = torch.empty(2, 3, V, device="cuda")
    same(ops.adjust_logits(x, out=out, **kw).view(6, V), want, torch.float32)
    turned = x.view(6, V).t().contiguous().t()  # vocabulary not contiguous
    flat = {k: v.reshape(6, -1) if k == "tokens" else v.reshape(6) if k not in ("bias", "mask") else v for k, v in kw.items()}
    same(ops.adjust_logits(turned, **flat), want, torch.float16)


def test_refusals_on_the_device(ops):
    x = torch.zeros(2, 8, device="cuda")
    i32 = dict(dtype=torch.int32, device="cuda")
    for kw in (dict(repetition_penalty=0.0), dict(repetition_penalty=torch.ones(3, device="cuda")), dict(num_tokens=torch.zeros(2, **i32)),
               dict(tokens=torch.zeros(3, 4, **i32)), dict(tokens=torch.zeros(4, **i32)), dict(tokens=torch.zeros(2, 4, dtype=torch.int32)),
               dict(bias=torch.zeros(3, 8, device="cuda")), dict(bias=torch.zeros(2, 9, device="cuda")), dict(bias=torch.zeros(2, 8)),
               dict(mask=torch.zeros(2, 2, **i32)), dict(mask=torch.zeros(2, 1, device="cuda")), dict(mask=torch.zeros(3, 1, **i32)),
               dict(mask_row=torch.zeros(2, **i32)), dict(bias=torch.zeros(1, 8, device="cuda"), bias_row=torch.zeros(3, **i32))):
        with pytest.raises(ValueError):
            ops.adjust_logits(x, **kw)
    for bad in (torch.zeros(2, 0, device="cuda"), torch.zeros(2, 8, device="cuda", dtype=torch.int32), torch.zeros(2, 8, device="cuda", dtype=torch.float64)):
        with pytest.raises(ValueError):
            ops.adjust_logits(bad)
    assert ops.adjust_logits(torch.zeros(0, 8, device="cuda")).shape == (0, 8)
