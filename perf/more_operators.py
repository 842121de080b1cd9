"""The operators of a decode step over sequences that share a prefix, as cases to be timed and compared.

Three operators: ``append`` (new keys rotated by their positions and written, with the values, into the paged cache;
the queries rotated on the way), ``prefix`` (attention of a batch whose groups share the pages of a long prefix, which
is read once for a whole group) and ``logits`` (penalties for repeated tokens, biases and grammar masks, before a
token is chosen).  With ``own`` false ``run`` computes them with elementary torch operations; with ``own`` true it
calls the package.
"""
import math
import os
import sys

import numpy as np
import torch

own = False

sys.path.append(os.path.join(os.getcwd(), "paged-inference-engine_b200"))  # the package's folder

_DTYPES = {"fp32": torch.float32, "fp16": torch.float16, "bf16": torch.bfloat16, "int8": torch.int8}
_BYTES = {"fp32": 4, "fp16": 2, "bf16": 2, "int8": 1}


def listed():
    return [
        # the first token of one request's decode step: latency decides
        dict(name="append 1 fp16", op="append", tokens=1, seqs=1, context=700, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, dtype="fp16", pool="fp16", block=16),
        # a decode batch over an INT8 cache
        dict(name="append 64 int8", op="append", tokens=64, seqs=64, context=4096, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, dtype="bf16", pool="int8", block=16),
        # chunks of a few prompts; an odd number of tokens, half of each head rotated, in neighbouring pairs
        dict(name="append 3001 bf16 pairs", op="append", tokens=3001, seqs=5, context=9000, heads=20, kv_heads=5, dim=128, rot=64, interleaved=True, dtype="bf16", pool="bf16", block=32),
        # whole prompts into an INT8 cache: bandwidth decides
        dict(name="append 16384 int8", op="append", tokens=16384, seqs=8, context=32768, heads=32, kv_heads=8, dim=128, rot=128, interleaved=False, dtype="bf16", pool="int8", block=16),
        # four beams of one chat request
        dict(name="prefix 1x4 of 592 fp16", op="prefix", groups=1, members=4, prefix=592, suffix=30, rows=1, heads=32, kv_heads=8, dim=128, pool="fp16", block=16),
        # a few system prompts, heads of 64, groups of five heads, two rows a sequence as when a draft is checked
        dict(name="prefix 5x7 of 1504 bf16 d64", op="prefix", groups=5, members=7, prefix=1504, suffix=200, rows=2, heads=20, kv_heads=4, dim=64, pool="bf16", block=32),
        # a chat batch behind one long system prompt
        dict(name="prefix 1x64 of 8192 fp16", op="prefix", groups=1, members=64, prefix=8192, suffix=300, rows=1, heads=32, kv_heads=8, dim=128, pool="fp16", block=16),
        # several documents, each asked many questions, in an INT8 cache
        dict(name="prefix 4x32 of 16384 int8", op="prefix", groups=4, members=32, prefix=16384, suffix=200, rows=1, heads=32, kv_heads=8, dim=128, pool="int8", block=16),
        # many samples of one very long prompt
        dict(name="prefix 1x128 of 65536 bf16", op="prefix", groups=1, members=128, prefix=65536, suffix=500, rows=1, heads=32, kv_heads=8, dim=128, pool="bf16", block=16),
        # one chat request with penalties
        dict(name="logits 1 of 32000 fp32", op="logits", rows=1, vocab=32000, history=500, dtype="fp32", biases=0, masks=0),
        # a batch over a vocabulary of odd size: rows start at odd addresses; two users' biases, some grammars
        dict(name="logits 48 of 50257 bf16", op="logits", rows=48, vocab=50257, history=2000, dtype="bf16", biases=2, masks=30),
        # a full batch of beams over a large vocabulary
        dict(name="logits 512 of 131072 bf16", op="logits", rows=512, vocab=131072, history=1500, dtype="bf16", biases=1, masks=64),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "prefix", "prefix", "logits"])
    if op == "logits":
        rows, vocab = _log_int(rng, 1, 512), _log_int(rng, 300, 131072)
        return dict(op=op, rows=rows, vocab=vocab, history=_log_int(rng, 1, 3000), dtype=rng.choice(["fp32", "fp16", "bf16", "bf16"]) if rows * vocab < 1 << 25 else "bf16",
                    biases=rng.choice([0, 1, rng.randint(2, 5)]), masks=rng.choice([0, rng.randint(1, rows)]))
    dim = rng.choice([64, 128, 128])
    heads = dict(kv_heads=rng.randint(1, 8), dim=dim, block=rng.choice([8, 16, 32]))
    group = rng.choice([1, 2, 3, 4, 4, 5, 8])
    if op == "append":
        tokens = _log_int(rng, 1, 16384)
        pool = rng.choice(["int8", "fp16", "bf16"])
        rot = rng.choice([dim, dim, dim // 2, 16 * rng.randint(1, dim // 16)])
        return dict(op=op, tokens=tokens, seqs=rng.randint(1, min(tokens, 64)), context=tokens + _log_int(rng, 10, 32768), heads=heads["kv_heads"] * min(group, 4), rot=rot,
                    interleaved=rng.random() < 0.4, dtype=rng.choice(["fp16", "bf16"]) if pool == "int8" else pool, pool=pool, **heads)
    groups, members = _log_int(rng, 1, 12), _log_int(rng, 2, 128)
    prefix = heads["block"] * max(1, _log_int(rng, 16, 65536) // heads["block"])
    rows = 2 if group <= 4 and rng.random() < 0.2 else 1
    while groups > 1 and groups * members * rows * prefix * group > 128 * 65536 * 4 // 4:
        groups //= 2
    while members * rows * prefix * group > 128 * 65536 * 4 // 4 and members > 2:
        members //= 2
    return dict(op=op, groups=groups, members=members, prefix=prefix, suffix=max(2, _log_int(rng, 2, 500)), rows=rows, heads=heads["kv_heads"] * group,
                pool=rng.choice(["int8", "fp16", "bf16"]), **heads)


# ---- inputs ------------------------------------------------------------------------------------------------------
def _pool(case, blocks, gen, fill):
    """K and V pools (one tensor) and an INT8 pool's scales, kept head-major as the package keeps them."""
    H, BS, dev = case["kv_heads"], case["block"], torch.device("cuda")
    shape = (2, blocks, BS, H, case["dim"])
    if case["pool"] == "int8":
        kv = torch.randint(-127, 128, shape, dtype=torch.int8, device=dev, generator=gen) if fill else torch.zeros(shape, dtype=torch.int8, device=dev)
        scale = (torch.rand(2, blocks, H, BS, device=dev, generator=gen) * 0.02 + 0.008).half() if fill else torch.ones(2, blocks, H, BS, device=dev).half()
        scale = scale.transpose(2, 3)
        return dict(kv=kv, scale=scale, k=kv[0], v=kv[1], ks=scale[0], vs=scale[1])
    dtype = _DTYPES[case["pool"]]
    kv = torch.randn(shape, dtype=dtype, device=dev, generator=gen) if fill else torch.zeros(shape, dtype=dtype, device=dev)
    return dict(kv=kv, scale=None, k=kv[0], v=kv[1], ks=None, vs=None)


def _i32(a):
    return torch.from_numpy(np.ascontiguousarray(a).astype(np.int32)).cuda()


def _lengths(case, seed):
    """Of a prefix case: shared tokens of every group (whole pages) and all tokens of every sequence."""
    g = np.random.default_rng(seed)
    shared = np.array([max(case["block"], case["prefix"] - 3 * i * case["block"]) for i in range(case["groups"])])
    own_tokens = g.integers(case["rows"], max(case["rows"], case["suffix"]) + 1, case["groups"] * case["members"])
    return shared, np.repeat(shared, case["members"]) + own_tokens


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    g = np.random.default_rng(seed + 1)
    dev = torch.device("cuda")
    randn = lambda *shape: torch.randn(shape, device=dev, generator=gen)  # noqa: E731
    if case["op"] == "append":
        T, S, BS, R = case["tokens"], case["seqs"], case["block"], case["rot"]
        # S sequences take shares of the tokens, each behind what it holds already
        cuts = np.sort(g.permutation(T - 1)[:S - 1]) + 1 if S > 1 else np.array([], np.int64)
        share = np.diff(np.concatenate([[0], cuts, [T]]))
        held = g.integers(0, case["context"] - share + 1)
        row = np.repeat(np.arange(S), share)
        pos = held[row] + np.arange(T) - np.repeat(np.cumsum(share) - share, share)
        # pages: only those that are written to exist
        first, last = held // BS, (held + share - 1) // BS
        table = np.zeros((S, int(last.max()) + 1), np.int64)
        pages = min(T, T // BS + 2 * S) + 3  # the most that any seed writes to, and some more
        ids = g.permutation(pages)
        at = np.cumsum(last - first + 1) - (last - first + 1)
        for s in range(S):
            table[s, first[s]:last[s] + 1] = ids[at[s]:at[s] + last[s] - first[s] + 1]
        angle = torch.arange(case["context"], dtype=torch.float64, device=dev)[:, None] * 10000.0**(-torch.arange(0, R, 2, dtype=torch.float64, device=dev) / R)
        dtype = _DTYPES[case["dtype"]]
        qkv = randn(T, case["heads"] + 2 * case["kv_heads"], case["dim"])
        qkv *= 1 + 6 * (torch.rand(case["dim"], device=dev, generator=gen) > 0.97)  # a few channels stand out, as in a model's keys
        q, k, v = qkv.to(dtype).split([case["heads"], case["kv_heads"], case["kv_heads"]], 1)  # rows of one projection's output
        return dict(op="append", q=q, k_new=k, v_new=v, angles=torch.cat([angle.cos(), angle.sin()], 1).float(), pairs=case["interleaved"], table=_i32(table), row=_i32(row), pos=_i32(pos),
                    **_pool(case, pages, gen, False))
    if case["op"] == "prefix":
        n, G, BS, B = case["members"], case["groups"], case["block"], case["groups"] * case["members"]
        shared, lens = _lengths(case, seed)
        full, have = shared // BS, -(-lens // BS)
        mine = have - np.repeat(full, n)
        pages = int(full.sum() + mine.sum())
        ids = g.permutation(pages)
        table = np.zeros((B, int(have.max())), np.int64)
        at = np.concatenate([[0], np.cumsum(full), full.sum() + np.cumsum(mine)])
        for b in range(B):
            f = int(full[b // n])
            table[b, :f] = ids[at[b // n]:at[b // n] + f]
            table[b, f:have[b]] = ids[at[G + b]:at[G + b] + mine[b]]
        q = randn(B, case["heads"], case["rows"], case["dim"]).to(torch.float16 if case["pool"] == "int8" else _DTYPES[case["pool"]])
        return dict(op="prefix", q=q, q_len=_i32(np.full(B, case["rows"])), table=_i32(table), pages=_i32(have), block=BS, kv_len=_i32(lens), group_start=_i32(np.arange(G + 1) * n),
                    shared=_i32(shared), members=n, most_shared=int(full.max()), most_own=int(mine.max()), **_pool(case, pages, gen, True))
    R, V, L = case["rows"], case["vocab"], case["history"]
    x = randn(R, V) * 2.2
    peaks = torch.randint(0, V, (R, 12), device=dev, generator=gen)
    x.scatter_add_(1, peaks, torch.rand(R, 12, device=dev, generator=gen) * 9)
    # tokens repeat as words do, a few of them very often
    tokens = np.minimum(V - 1, (V**g.random((R, L)) - 1).astype(np.int64)) * 7919 % V
    count = g.integers(max(1, L // 2), L + 1, R)
    prompt = (count * g.random(R)).astype(np.int64)
    bias = randn(case["biases"], V) * (torch.rand(case["biases"], V, device=dev, generator=gen) < 0.002) * 8 if case["biases"] else None
    bits = None
    if case["masks"]:
        words = torch.randint(-2**31, 2**31, (2, case["masks"], (V + 31) // 32), device=dev, generator=gen)
        # every other grammar allows few tokens, the others most
        bits = torch.where(torch.arange(case["masks"], device=dev)[:, None] % 2 == 0, words[0] & words[1] & words[1].roll(1, 1) & words[0].roll(1, 1), words[0] | words[1]).int()
    uniform = lambda lo, hi: torch.rand(R, device=dev, generator=gen) * (hi - lo) + lo  # noqa: E731
    return dict(op="logits", logits=x.to(_DTYPES[case["dtype"]]), tokens=_i32(tokens), count=_i32(count), prompt=_i32(prompt), repetition=uniform(1.0, 1.4), presence=uniform(0.0, 0.6),
                frequency=uniform(0.0, 0.3), bias=bias, bias_row=_i32(g.integers(-1, case["biases"], R)) if case["biases"] else None, mask=bits,
                mask_row=_i32(np.where(g.random(R) < 0.3, -1, g.integers(0, max(1, case["masks"]), R))) if case["masks"] else None)


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _rotate(x, cos, sin, pairs):
    """The first dims of every head turned by their angles, in 32 bits: pairs of neighbours, or of the two halves."""
    half = cos.shape[-1]
    x = x.float()
    turn, rest = x[..., :2 * half], x[..., 2 * half:]
    a, b = (turn[..., 0::2], turn[..., 1::2]) if pairs else (turn[..., :half], turn[..., half:])
    a, b = a * cos - b * sin, b * cos + a * sin
    turned = torch.stack([a, b], -1).flatten(-2) if pairs else torch.cat([a, b], -1)
    return torch.cat([turned, rest], -1)


def _append(s):
    angles = s["angles"][s["pos"].long()][:, None]
    cos, sin = angles.chunk(2, -1)
    block = s["kv"].shape[2]
    page = s["table"][s["row"].long(), s["pos"].long() // block].long()
    slot = s["pos"].long() % block
    new = torch.stack([_rotate(s["k_new"], cos, sin, s["pairs"]), s["v_new"].float()])
    if s["scale"] is not None:
        most = new.abs().amax(-1)
        scale = torch.where(most == 0, 1.0, most / 127)
        s["scale"][:, page, slot] = scale.half()
        new = (new / scale[..., None]).round().clamp(-127, 127)
    s["kv"][:, page, slot] = new.to(s["kv"].dtype)
    return _rotate(s["q"], cos, sin, s["pairs"]).to(s["q"].dtype)


def _pages(s, ids):
    """Keys and values of these pages [.., n], in 32 bits, as [2, .., n * block, heads, dim]."""
    kv = s["kv"][:, ids].float()
    if s["scale"] is not None:
        kv = kv * s["scale"][:, ids].float()[..., None]
    return kv.flatten(-4, -3)


def _prefix(s):
    q, n, BS = s["q"].float(), s["members"], s["block"]
    B, Hq, M, D = q.shape
    dev, H = q.device, s["kv"].shape[3]
    g, G = Hq // H, B // n
    rows = q.view(G, n, H, g * M, D).transpose(1, 2).flatten(2, 3) * D**-0.5  # [G, H, n * g * M, D]
    # the shared pages, through the first member's table
    k, v = _pages(s, s["table"][::n, :s["most_shared"]].long())
    seen = torch.arange(k.shape[1], device=dev) < s["shared"][:, None]
    a = (rows @ k.permute(0, 2, 3, 1)).masked_fill(~seen[:, None, None], -math.inf)
    # every sequence's own pages
    first = (s["shared"] // BS).repeat_interleave(n)
    col = first[:, None] + torch.arange(s["most_own"], device=dev)
    own_k, own_v = _pages(s, s["table"].gather(1, col.clamp(max=s["table"].shape[1] - 1).long()).long())
    place = first[:, None] * BS + torch.arange(own_k.shape[1], device=dev)
    seen = place[:, None] <= (s["kv_len"][:, None] - M + torch.arange(M, device=dev))[..., None]  # [B, M, keys]
    b = (q.view(B, H, g, M, D) * D**-0.5) @ own_k.permute(0, 2, 3, 1)[:, :, None]
    b = b.masked_fill(~seen[:, None, None], -math.inf)
    part = lambda t: t.unflatten(2, (n, g * M)).transpose(1, 2).reshape(B, H, g, M, *t.shape[3:])  # noqa: E731
    top = torch.maximum(part(a.amax(-1)), b.amax(-1))
    whole = top.reshape(G, n, H, g * M).transpose(1, 2).flatten(2)
    a = (a - whole[..., None]).exp()
    b = (b - top[..., None]).exp()
    total = part(a.sum(-1)) + b.sum(-1)
    o = part(a @ v.transpose(1, 2)) + b @ own_v.transpose(1, 2)[:, :, None]
    return (o / total[..., None]).reshape(B, Hq, M, D).half(), (top + total.log()).reshape(B, Hq, M).half()


def _logits(s):
    x = s["logits"].float()
    R, V = x.shape
    place = torch.arange(s["tokens"].shape[1], device=x.device)
    held = place < s["count"][:, None]
    made = held & (place >= s["prompt"][:, None])
    tokens = s["tokens"].long()
    zero = torch.zeros(R, V, device=x.device)
    seen = zero.scatter_add(1, tokens, held.float()) > 0
    times = zero.scatter_add(1, tokens, made.float())
    again = s["repetition"][:, None]
    x = torch.where(seen, torch.where(x > 0, x / again, x * again), x)
    x = x - s["frequency"][:, None] * times
    x = x - s["presence"][:, None] * (times > 0)
    if s["bias"] is not None:
        row = s["bias_row"].long()
        x = torch.where((row >= 0)[:, None], x + s["bias"][row.clamp(min=0)], x)
    if s["mask"] is not None:
        row, token = s["mask_row"].long(), torch.arange(V, device=x.device)
        allowed = s["mask"][row.clamp(min=0)][:, token // 32] >> (token % 32) & 1
        x = x.masked_fill((row >= 0)[:, None] & (allowed == 0), -math.inf)
    return x.to(s["logits"].dtype)


# ---- one pass ----------------------------------------------------------------------------------------------------
def _held(s):
    """The cache; an INT8 cache as the values that its codes stand for."""
    return s["kv"] if s["scale"] is None else s["kv"] * s["scale"][..., None]


def run(state):
    s, op = state, state["op"]
    if op == "append":
        if own:
            from pie_b200 import ops

            q = ops.rotate_write_kv(s["q"], s["k_new"], s["v_new"], s["angles"], s["table"], s["row"], s["pos"], s["k"], s["v"], s["ks"], s["vs"], interleaved=s["pairs"])
        else:
            q = _append(s)
        return q, _held(s)
    if op == "prefix":
        if own:
            from pie_b200 import ops

            return ops.shared_prefix_attention(s["q"], s["k"], s["v"], s["q_len"], s["table"], s["pages"], s["block"], s["kv_len"], s["group_start"], s["shared"], s["ks"], s["vs"])
        return _prefix(s)
    if own:
        from pie_b200 import ops

        return ops.adjust_logits(s["logits"], tokens=s["tokens"], num_tokens=s["count"], prompt_len=s["prompt"], repetition_penalty=s["repetition"], presence_penalty=s["presence"],
                                 frequency_penalty=s["frequency"], bias=s["bias"], bias_row=s["bias_row"], mask=s["mask"], mask_row=s["mask_row"])
    return _logits(s)


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def work(case):
    if case["op"] == "append":
        T, dim, H = case["tokens"], case["dim"], case["kv_heads"]
        rows = case["heads"] + 2 * H
        scale = 4 * H if case["pool"] == "int8" else 0  # two fp16 scales a head
        moved = T * (rows * dim * _BYTES[case["dtype"]] + case["heads"] * dim * _BYTES[case["dtype"]] + 2 * H * dim * _BYTES[case["pool"]] + scale + 12)
        return dict(bytes=moved + 4 * case["rot"] * min(T, case["context"]), flops=3 * T * (case["heads"] + H) * case["rot"])
    if case["op"] == "prefix":
        shared, lens = _lengths(case, 0)
        alone = int((lens - np.repeat(shared, case["members"])).sum())
        slot = 2 * case["kv_heads"] * (case["dim"] * _BYTES[case["pool"]] + (2 if case["pool"] == "int8" else 0))
        rows = len(lens) * case["heads"] * case["rows"]
        return dict(bytes=(int(shared.sum()) + alone) * slot + rows * (4 * case["dim"] + 2) + 4 * int((lens // case["block"]).sum()),
                    flops=4 * case["heads"] * case["rows"] * case["dim"] * int(lens.sum()))
    R, V, e = case["rows"], case["vocab"], _BYTES[case["dtype"]]
    return dict(bytes=2 * R * V * e + 4 * case["biases"] * V + case["masks"] * 4 * ((V + 31) // 32) + R * 3 * case["history"], flops=R * V * (1 if case["biases"] else 0) + R * 4 * case["history"])


# ---- the definitions in 64 bits ----------------------------------------------------------------------------------
def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "append":
        half, block = case["rot"] // 2, case["block"]
        # a turn by an angle is a product of complex numbers
        turn = torch.complex(s["angles"][:, :half].double(), s["angles"][:, half:].double())[s["pos"].long()][:, None]

        def turned(x):
            x = x.double().clone()
            part = x[..., :2 * half]
            z = torch.view_as_complex(part.unflatten(-1, (half, 2)).contiguous()) if case["interleaved"] else torch.complex(part[..., :half], part[..., half:])
            z = z * turn
            x[..., :2 * half] = torch.view_as_real(z).flatten(-2) if case["interleaved"] else torch.cat([z.real, z.imag], -1)
            return x

        kv = s["kv"].double()
        at = s["table"][s["row"].long(), (s["pos"] // block).long()].long() * block + s["pos"].long() % block
        for i, x in enumerate((turned(s["k_new"]), s["v_new"].double())):
            if case["pool"] == "int8":
                step = x.abs().amax(-1, keepdim=True) / 127
                step = torch.where(step == 0, torch.ones_like(step), step)
                x = torch.round(x / step) * step
            kv[i].view(-1, *kv.shape[3:])[at] = x
        return turned(s["q"]), kv
    if case["op"] == "prefix":
        got, D, g, M, BS = [], case["dim"], case["heads"] // case["kv_heads"], case["rows"], case["block"]
        lens = s["kv_len"].tolist()
        if sum(lens) * case["heads"] > 1 << 31:
            return None
        for b, n in enumerate(lens):
            ids = s["table"][b, :-(-n // BS)].long()
            k, v = (s["kv"][i][ids].double() for i in range(2))
            if s["scale"] is not None:
                k, v = k * s["ks"][ids].double()[..., None], v * s["vs"][ids].double()[..., None]
            k, v = (t.flatten(0, 1)[:n].repeat_interleave(g, 1) for t in (k, v))
            a = torch.einsum("hmd,nhd->hmn", s["q"][b].double(), k) / math.sqrt(D)
            a = torch.where(torch.arange(n, device=a.device) < n - M + 1 + torch.arange(M, device=a.device)[:, None], a, -math.inf)
            got.append((torch.einsum("hmn,nhd->hmd", a.softmax(-1), v), a.logsumexp(-1)))
        return tuple(torch.stack(t) for t in zip(*got))
    out = s["logits"].double()
    for r in range(case["rows"]):
        n, p = int(s["count"][r]), int(s["prompt"][r])
        rep, pres, freq = (float(s[t][r]) for t in ("repetition", "presence", "frequency"))
        ids = s["tokens"][r, :n].long().unique()
        x = out[r, ids]
        out[r, ids] = torch.where(x > 0, x / rep, x * rep)
        ids, times = s["tokens"][r, p:n].long().unique(return_counts=True)
        out[r, ids] -= freq * times + pres
        if s["bias"] is not None and s["bias_row"][r] >= 0:
            out[r] += s["bias"][s["bias_row"][r]].double()
        if s["mask"] is not None and s["mask_row"][r] >= 0:
            bits = s["mask"][s["mask_row"][r]].cpu().numpy().view(np.uint8)
            out[r, torch.from_numpy(np.unpackbits(bits, bitorder="little")[:case["vocab"]] == 0).cuda()] = -math.inf
    return out
