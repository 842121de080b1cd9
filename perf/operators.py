"""The beam-search and page operators of the paged cache, as cases to be timed and compared.

Four operators: ``select`` (the best continuations of every sequence's beams over the vocabulary), ``copy`` (pages
copied inside the paged K/V pools of several layers), ``reorder`` (beams take over their parents' pages: shared
full pages, copied partial pages, freed pages) and ``compact`` (live pages moved to the lowest ids).  With
``own`` false ``run`` computes them with elementary torch operations; with ``own`` true it calls the package.
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
        # one chat request decoded with four beams: latency decides
        dict(name="select 1x4 of 32000 fp32", op="select", seqs=1, beams=4, vocab=32000, out=8, dtype="fp32", finished=0),
        # a small batch over a vocabulary of odd size: rows start at odd addresses
        dict(name="select 16x4 of 50257 bf16", op="select", seqs=16, beams=4, vocab=50257, out=8, dtype="bf16", finished=0),
        # wide beams of which a quarter has ended: their rows need not be read
        dict(name="select 6x16 of 65536 fp16", op="select", seqs=6, beams=16, vocab=65536, out=32, dtype="fp16", finished=4),
        # a full decode batch over a large vocabulary: bandwidth decides
        dict(name="select 64x8 of 131072 bf16", op="select", seqs=64, beams=8, vocab=131072, out=16, dtype="bf16", finished=0),
        # the partial pages of a few forks in an INT8 pool of one layer
        dict(name="copy 6 pages int8", op="copy", layers=1, pairs=6, block=16, heads=8, dim=128, dtype="int8", layout="slots", ragged=True),
        # pages in the [block, head, slot, d] layout, an odd number of heads, partly filled
        dict(name="copy 100 pages x 4 fp16", op="copy", layers=4, pairs=100, block=32, heads=5, dim=64, dtype="fp16", layout="heads", ragged=True),
        # whole pages of every layer of a model, as a cache fork or swap-in copies them
        dict(name="copy 256 pages x 16 bf16", op="copy", layers=16, pairs=256, block=16, heads=8, dim=128, dtype="bf16", layout="slots", ragged=False),
        # one request's beams after a step
        dict(name="reorder 1x4 int8", op="reorder", groups=1, beams=4, forks=2, tokens=700, prompt=500, layers=1, block=16, heads=8, dim=128, dtype="int8"),
        # a batch of beams over a model's layers
        dict(name="reorder 16x6 fp16", op="reorder", groups=16, beams=6, forks=3, tokens=3001, prompt=2000, layers=8, block=16, heads=4, dim=128, dtype="fp16"),
        # a full batch with long contexts
        dict(name="reorder 64x8 bf16", op="reorder", groups=64, beams=8, forks=4, tokens=4095, prompt=3500, layers=4, block=32, heads=8, dim=128, dtype="bf16"),
        # a small pool with holes
        dict(name="compact 500 int8", op="compact", blocks=500, live=200, moves=60, rows=30, layers=2, block=16, heads=8, dim=64, dtype="int8"),
        # a large pool after many requests have come and gone
        dict(name="compact 8192 bf16", op="compact", blocks=8192, live=4000, moves=1900, rows=256, layers=4, block=16, heads=8, dim=128, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["select", "copy", "reorder", "compact"])
    if op == "select":
        beams = rng.randint(1, 16)
        dtype = rng.choice(["fp32", "bf16", "fp16"])
        seqs = _log_int(rng, 1, 64)
        vocab = _log_int(rng, 300, 131072)
        while seqs * beams * vocab * _BYTES[dtype] > 64 * 8 * 131072 * 2:
            seqs = max(1, seqs // 2)
        return dict(op=op, seqs=seqs, beams=beams, vocab=vocab, out=rng.randint(beams, 2 * beams), dtype=dtype,
                    finished=rng.randint(0, beams - 1) if rng.random() < 0.4 else 0)
    pages = dict(layers=_log_int(rng, 1, 16), block=rng.choice([8, 16, 32]), heads=rng.randint(1, 8),
                 dim=rng.choice([64, 128]), dtype=rng.choice(["int8", "fp16", "bf16", "fp32"]))
    page = pages["layers"] * 2 * pages["block"] * pages["heads"] * pages["dim"] * _BYTES[pages["dtype"]]
    if op == "copy":
        pairs = _log_int(rng, 1, 256)
        return dict(op=op, pairs=max(1, min(pairs, (256 << 20) // page)), layout=rng.choice(["slots", "heads"]),
                    ragged=rng.random() < 0.5, **pages)
    if op == "reorder":
        beams = rng.randint(2, 16)
        groups = _log_int(rng, 1, 64)
        tokens = _log_int(rng, 40, 4096)
        prompt = rng.randint(1, tokens)
        while groups > 1 and groups * (prompt + beams * (tokens - prompt + 2 * pages["block"])) / pages["block"] * page > (1 << 30):
            groups = max(1, groups // 2)
        while pages["layers"] > 1 and groups * (prompt + beams * (tokens - prompt + 2 * pages["block"])) / pages["block"] * page > (1 << 30):
            page, pages["layers"] = page * (pages["layers"] // 2) // pages["layers"], pages["layers"] // 2
        return dict(op=op, groups=groups, beams=beams, forks=rng.randint(0, beams - 1), tokens=tokens, prompt=prompt, **pages)
    blocks = max(8, min(_log_int(rng, 50, 8192), (1 << 30) // page))
    live = rng.randint(1, blocks)
    return dict(op=op, blocks=blocks, live=live, moves=rng.randint(0, min(live, blocks - live)), rows=_log_int(rng, 1, 256), **pages)


# ---- inputs ------------------------------------------------------------------------------------------------------
def _pages(case, blocks, gen, layout="slots"):
    """K and V pools of every layer (one tensor), and an INT8 pool's scales, kept head-major as the package keeps them."""
    L, BS, H, D = case["layers"], case["block"], case["heads"], case["dim"]
    shape = (L, 2, blocks, BS, H, D) if layout == "slots" else (L, 2, blocks, H, BS, D)
    dev = torch.device("cuda")
    scale = None
    if case["dtype"] == "int8":
        kv = torch.randint(-127, 128, shape, dtype=torch.int8, device=dev, generator=gen)
        scale = (torch.rand(L, 2, blocks, H, BS, device=dev, generator=gen) * 0.05 + 0.01).half().transpose(3, 4)
    else:
        kv = torch.randn(shape, dtype=_DTYPES[case["dtype"]], device=dev, generator=gen)
    if layout == "heads":
        kv = kv.transpose(3, 4)
    state = dict(kv=kv, scale=scale, k=[kv[l, 0] for l in range(L)], v=[kv[l, 1] for l in range(L)])
    state["ks"] = None if scale is None else [scale[l, 0] for l in range(L)]
    state["vs"] = None if scale is None else [scale[l, 1] for l in range(L)]
    return state


def _pool(table, count, blocks, g):
    """A pool's tables on the GPU as views of one buffer, with a saved copy: every pass starts from the saved tables."""
    used = table[np.arange(table.shape[1])[None, :] < count[:, None]]
    ref = np.bincount(used, minlength=blocks)
    free = g.permutation(np.nonzero(ref == 0)[0])
    stack = np.zeros(blocks, np.int64)
    stack[:len(free)] = free
    parts = [stack, np.array([len(free)]), table.reshape(-1), count, ref]
    sizes = [len(p) for p in parts]
    saved = torch.from_numpy(np.concatenate(parts).astype(np.int32)).cuda()
    now = saved.clone()
    stack, top, tab, cnt, ref = now.split(sizes)
    return dict(saved=saved, now=now, free_stack=stack, free_top=top, table=tab.view(table.shape), count=cnt, ref_count=ref,
                scratch=torch.zeros(16 + 4 * blocks + (blocks + 31) // 32, dtype=torch.int32, device="cuda"))


def prepare(case, seed):
    gen = torch.Generator(device="cuda")
    gen.manual_seed(seed)
    g = np.random.default_rng(seed)
    dev = torch.device("cuda")
    if case["op"] == "select":
        B, K, V = case["seqs"], case["beams"], case["vocab"]
        x = torch.randn(B, K, V, device=dev, generator=gen) * 2.2
        # a language model's rows are peaked: a few tokens stand far above the rest
        peaks = torch.randint(0, V, (B, K, 12), device=dev, generator=gen)
        x.scatter_add_(2, peaks, torch.rand(B, K, 12, device=dev, generator=gen) * 9)
        scores = -torch.rand(B, K, device=dev, generator=gen).cumsum(1) * 1.5 - 20
        ended = torch.zeros(B, K, dtype=torch.bool)
        for b in range(B):
            ended[b, torch.from_numpy(g.permutation(K)[:case["finished"]])] = True
        return dict(op="select", logits=x.to(_DTYPES[case["dtype"]]), scores=scores, finished=ended.cuda() if case["finished"] else None,
                    eos=2, out=case["out"])
    if case["op"] == "copy":
        n, BS = case["pairs"], case["block"]
        blocks = 2 * n + 7
        ids = torch.from_numpy(g.permutation(blocks)[:2 * n].astype(np.int32)).cuda()
        slots = torch.from_numpy(g.integers(1, BS, n).astype(np.int32)).cuda() if case["ragged"] else None
        return dict(op="copy", src=ids[:n].contiguous(), dst=ids[n:].contiguous(), slots=slots, **_pages(case, blocks, gen, case["layout"]))
    if case["op"] == "reorder":
        G, K, BS = case["groups"], case["beams"], case["block"]
        # groups differ a little in length, so that their partial pages hold between 1 and BS - 1 tokens
        lens = np.array([max(1, case["tokens"] - 3 * i % BS) for i in range(G)])
        cols = int(-(-lens.max() // BS)) + 1
        table = np.zeros((G * K + 3, cols), np.int64)
        rows = g.permutation(G * K + 3)[:G * K].reshape(G, K)
        count = np.full(G * K + 3, -1)
        nxt, parents = 0, np.zeros((G, K), np.int64)
        for i in range(G):
            full, have = lens[i] // BS, -(-lens[i] // BS)
            shared = min(full, case["prompt"] // BS)
            mine = np.zeros((K, have), np.int64)
            mine[:, :shared] = nxt + np.arange(shared)[None, :]
            nxt += shared
            fresh = nxt + np.arange(K * (have - shared)).reshape(K, have - shared)
            nxt += fresh.size
            mine[:, shared:] = fresh
            # what earlier steps left: the older a page, the fewer ancestors the beams have in common for it
            line = np.arange(K)
            for c in range(full - 1, shared - 1, -1):
                if g.random() < 0.3:
                    line = g.integers(0, K, K)[line]
                mine[:, c] = fresh[line, c - shared]
            table[rows[i], :have] = mine
            count[rows[i]] = have
            alive = g.permutation(K)[:K - case["forks"]]
            parents[i] = g.permutation(np.concatenate([alive, g.choice(alive, case["forks"])]))
        blocks = nxt + 5
        names = g.permutation(blocks)
        table = np.where(np.arange(cols)[None, :] < count[:, None], names[table], 0)
        put = lambda a: torch.from_numpy(a.astype(np.int32)).cuda()  # noqa: E731
        return dict(op="reorder", slots=put(rows), parents=put(parents), lens=put(lens), block=BS, pool=_pool(table, count, blocks, g),
                    **_pages(case, blocks, gen))
    blocks, live, moves = case["blocks"], case["live"], case["moves"]
    ids = np.concatenate([g.permutation(live)[:live - moves], live + g.permutation(blocks - live)[:moves]])
    ids = g.permutation(ids)
    have = np.diff((live * (np.arange(case["rows"] + 1) / case["rows"])**2).astype(np.int64))  # short and long sequences
    table = np.zeros((case["rows"] + 2, max(1, have.max()) + 1), np.int64)
    count = np.full(case["rows"] + 2, -1)
    at = 0
    for r in range(case["rows"]):
        table[r, :have[r]] = ids[at:at + have[r]]
        count[r] = have[r]
        at += have[r]
    # a second holder of a few sequences' pages, as a fork leaves them
    table[case["rows"], :have[0]], count[case["rows"]] = table[0, :have[0]], have[0]
    return dict(op="compact", pool=_pool(table, count, blocks, g), **_pages(case, blocks, gen))


# ---- the plain forms ---------------------------------------------------------------------------------------------
def _select(logits, scores, finished, eos, out):
    """Scores in 64 bits, because candidates of different beams are compared next to each other's values."""
    x = logits.float().nan_to_num(nan=-math.inf, posinf=torch.finfo(torch.float32).max, neginf=-math.inf) + 0.0
    B, K, V = x.shape
    token = torch.arange(V, device=x.device)
    if finished is not None:
        x = torch.where(finished[..., None], torch.where(token == eos, 0.0, -math.inf), x)
    top = x.amax(-1, keepdim=True)
    total = (x.double() - top.clamp(min=torch.finfo(torch.float32).min)).exp_().sum(-1, keepdim=True)
    # every row's best, the larger logit first and then the lower token, by one whole number for both
    bits = x.view(torch.int32).long()
    key = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) * 2**32 + (2**32 - 1 - token)
    key = key.topk(min(out, V), -1).values
    best = 2**32 - 1 - (key & 0xFFFFFFFF)
    part = x.gather(-1, best).double() - top
    part = torch.where(part.isnan(), -math.inf, part) - total.clamp(min=1e-300).log()
    score = (scores.double()[..., None] + part).nan_to_num(nan=-math.inf, posinf=math.inf, neginf=-math.inf).flatten(1)
    score, at = score.sort(dim=-1, descending=True, stable=True)
    at = at[:, :out]
    return score[:, :out].float(), best.flatten(1).gather(1, at).int(), (at // best.shape[-1]).int()


def _move(kv, scale, src, dst, slots):
    """Pages src to dst in every layer, the first `slots` slots of each."""
    keep = torch.arange(kv.shape[3], device=kv.device)[None, :, None, None] < slots[:, None, None, None]
    kv[:, :, dst] = torch.where(keep, kv[:, :, src], kv[:, :, dst])
    if scale is not None:
        scale[:, :, dst] = torch.where(keep[..., 0], scale[:, :, src], scale[:, :, dst])


def _reorder(s, pool):
    slots, parents = s["slots"].long(), s["parents"].long()
    K, device = slots.shape[1], slots.device
    beam = torch.arange(K, device=device)
    # the first child of a parent keeps the parent's row; the others take the rows of the beams without children
    again = ((parents[:, :, None] == parents[:, None, :]) & (beam[None, :, None] > beam[None, None, :])).any(-1)
    childless = ~(parents[:, :, None] == beam).any(1)
    spare = slots.gather(1, torch.where(childless, beam, beam + K).sort(1).indices)
    donor = slots.gather(1, parents)
    child = torch.where(again, spare.gather(1, (again.cumsum(1) - 1).clamp(min=0)), donor)
    # full pages are shared
    table, ref = pool["table"], pool["ref_count"]
    full = (s["lens"] // s["block"]).long()[:, None, None]
    whole = torch.arange(table.shape[1], device=device) < full
    old, new = table[child].long(), table[donor].long()
    row = torch.where(whole, new, old)
    one = whole.expand_as(row).int().flatten()
    after = ref.index_add(0, row.flatten(), one).index_add(0, old.flatten(), -one)
    freed = (ref > 0) & (after == 0)
    at = torch.where(freed, pool["free_top"] + freed.cumsum(0) - 1, ref.shape[0])
    stack = torch.cat([pool["free_stack"], pool["free_top"]]).scatter(0, at.long(), torch.arange(ref.shape[0], device=device, dtype=torch.int32))
    # partly filled pages are copied
    at = ((s["lens"] - 1) // s["block"]).long()[:, None, None].expand(-1, K, 1)
    part = (s["lens"] % s["block"])[:, None].expand(-1, K) * again
    _move(s["kv"], s["scale"], new.gather(2, at).flatten(), old.gather(2, at).flatten(), part.flatten())
    pool["free_stack"].copy_(stack[:-1])
    pool["free_top"].add_(freed.sum())
    table[child] = row.int()
    ref.copy_(after)
    return child.int()


def _compact(s, pool):
    ref, table = pool["ref_count"], pool["table"]
    blocks = ref.shape[0]
    page = torch.arange(blocks, device=ref.device)
    used = ref > 0
    live = used.sum()
    src, dst = (used & (page >= live)).nonzero()[:, 0], (~used & (page < live)).nonzero()[:, 0]
    s["kv"][:, :, dst] = s["kv"][:, :, src]
    if s["scale"] is not None:
        s["scale"][:, :, dst] = s["scale"][:, :, src]
    to = page.int().index_copy(0, src, dst.int())
    held = torch.arange(table.shape[1], device=ref.device) < pool["count"][:, None]
    table.copy_(torch.where(held, to[table.long()], table))
    ref[dst] = ref[src]
    ref[src] = 0
    pool["free_stack"].copy_(torch.where(page < blocks - live, blocks - 1 - page, pool["free_stack"]))
    pool["free_top"].copy_(blocks - live)
    return live.int().view(1)


# ---- the package's operators -------------------------------------------------------------------------------------
def _state(ops, pool):
    return ops.PoolState(pool["free_stack"], pool["free_top"], pool["table"], pool["count"], pool["ref_count"], pool["scratch"])


def run(state):
    s, op = state, state["op"]
    if op == "select":
        if own:
            from pie_b200 import ops

            return ops.beam_select(s["logits"], s["scores"], s["out"], finished=s["finished"], eos_id=s["eos"])
        return _select(s["logits"], s["scores"], s["finished"], s["eos"], s["out"])
    if op == "copy":
        if own:
            from pie_b200 import ops

            ops.copy_blocks(s["k"], s["v"], s["src"], s["dst"], s["ks"], s["vs"], num_slots=s["slots"])
        else:
            slots = s["slots"] if s["slots"] is not None else torch.full_like(s["src"], s["kv"].shape[3])
            _move(s["kv"], s["scale"], s["src"].long(), s["dst"].long(), slots)
        return [s["kv"], s["scale"]]
    # the tables change under the operator: each pass starts from the saved ones
    pool = s["pool"]
    pool["now"].copy_(pool["saved"])
    if op == "reorder":
        if own:
            from pie_b200 import ops

            got = ops.reorder_beams(_state(ops, pool), s["slots"], s["parents"], s["lens"], s["k"], s["v"], s["ks"], s["vs"])
        else:
            got = _reorder(s, pool)
    elif own:
        from pie_b200 import ops

        got = ops.compact_blocks(_state(ops, pool), s["k"], s["v"], s["ks"], s["vs"])
    else:
        got = _compact(s, pool)
    return [got, pool["now"], s["kv"], s["scale"]]


# ---- what a pass cannot do without -------------------------------------------------------------------------------
def _slot_bytes(case):
    """K and V of one token in every layer, with an INT8 pool's two fp16 scales a head."""
    return case["layers"] * 2 * case["heads"] * (case["dim"] * _BYTES[case["dtype"]] + (2 if case["dtype"] == "int8" else 0))


def work(case):
    if case["op"] == "select":
        rows = case["seqs"] * (case["beams"] - case["finished"])
        return dict(bytes=rows * case["vocab"] * _BYTES[case["dtype"]] + case["seqs"] * (5 * case["beams"] + 12 * case["out"]),
                    flops=3 * rows * case["vocab"])
    if case["op"] == "copy":
        slots = case["block"] / 2 if case["ragged"] else case["block"]
        return dict(bytes=2 * case["pairs"] * slots * _slot_bytes(case), flops=0)
    if case["op"] == "reorder":
        BS = case["block"]
        lens = [max(1, case["tokens"] - 3 * i % BS) for i in range(case["groups"])]
        # both rows of every fork are read, and the partial page is read and written
        return dict(bytes=sum(case["forks"] * (8 * (n // BS) + 2 * (n % BS) * _slot_bytes(case)) + 12 * case["beams"] for n in lens), flops=0)
    return dict(bytes=2 * case["moves"] * case["block"] * _slot_bytes(case) + 8 * case["blocks"] + 8 * case["live"], flops=0)


# ---- the definition in 64 bits -----------------------------------------------------------------------------------
def exact(case, seed):
    if case["op"] != "select":
        return None  # pages and tables are moved, not computed
    s = prepare(case, seed)
    V, got = case["vocab"], []
    for b in range(case["seqs"]):
        logp = torch.log_softmax(s["logits"][b].double(), -1)
        if s["finished"] is not None:
            ended = s["finished"][b].nonzero()[:, 0]
            logp[ended] = -math.inf
            logp[ended, s["eos"]] = 0
        total = (s["scores"][b].double()[:, None] + logp).flatten()
        score, at = torch.sort(total, descending=True, stable=True)
        at = at[:case["out"]]
        got.append((score[:case["out"]], (at % V).int(), (at // V).int()))
    return tuple(torch.stack(x) for x in zip(*got))
