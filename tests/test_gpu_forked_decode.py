"""GPU: a decode step's operators together, as a user has them: rotated appends, attention over shared prefixes, logit rules.

* the captured decode step over forks of one prompt, with a rotation table and shared prefixes;
* beam search with penalties, a bias and masks, its steps through rotate_write_kv and shared_prefix_attention.
"""
import math

import numpy as np
import pytest
import torch

from oracle import decode_step as ods
from test_gpu_block_sharing import Model
from test_gpu_shared_prefix import Problem, check

pytestmark = pytest.mark.gpu


def turned(x, table, positions, interleaved):
    """Rows rotated in fp32, a product or a sum at a time, and rounded once to their type, as the operator's."""
    cs = table[positions.long()].float().cpu().numpy()
    h = cs.shape[1] // 2
    y = ods.rotate(x.float().cpu().numpy(), cs[:, :h], cs[:, h:], interleaved)
    return torch.from_numpy(y).to(x.dtype).to(x.device)


class Step(Problem):
    """What a step attended to, read back from the pool and the caches, for test_gpu_shared_prefix.check."""

    def __init__(self, q, k, v, ks, vs, rows, lens, BS):
        self.K, self.V, self.ks, self.vs, self.BS = k, v, ks, vs, BS
        self.Q = q.unsqueeze(2)
        self.B, self.Hq, self.D, self.Hkv, self.maxq = q.shape[0], q.shape[1], q.shape[2], k.shape[2], 1
        i32 = lambda a: torch.tensor(a, dtype=torch.int32, device="cuda")  # noqa: E731
        width = max(map(len, rows))
        self.table = i32([r + [0] * (width - len(r)) for r in rows])
        self.kv_len, self.blocks, self.q_len = i32(lens), i32([len(r) for r in rows]), i32([1] * len(lens))


@pytest.mark.parametrize("dtype,interleaved", [(torch.float16, False), (torch.float16, True), (torch.int8, False)])
def test_decode_graph_rotates_and_reads_shared_prefixes_once(dtype, interleaved):
    from pie_b200 import ops as o
    from pie_b200.block_pool import DeviceBlockManager
    from pie_b200.decode_step import DecodeStepGraph
    from pie_b200.workloads import empty_head_major_scales

    BS, Hkv, D, Hq, NB, n = 16, 2, 128, 8, 160, 333
    gen = torch.Generator(device="cuda").manual_seed(6)
    k, v = (torch.zeros(NB, BS, Hkv, D, dtype=dtype, device="cuda") for _ in range(2))
    ks = vs = None
    if dtype == torch.int8:
        ks, vs = (empty_head_major_scales(NB, BS, Hkv, device="cuda").zero_() for _ in range(2))
    pool = DeviceBlockManager(NB, BS, 12, 24)
    pool.attach_caches(k, v, ks, vs)
    table = o.rope_table(400, D, device="cuda")
    graph = DecodeStepGraph(pool, k, v, ks, vs, Hq, 11, rope=table, interleaved=interleaved, share_prefixes=True)
    pool.allocate(0, -(-n // BS))
    inp = pool.step_inputs([0], [n], [n])
    rows = [torch.randn(n, Hkv, D, device="cuda", generator=gen).half() for _ in range(2)]
    assert o.rotate_write_kv(None, *rows, table, inp["block_table"], inp["token_seq"], inp["positions"], k, v, ks, vs,
                             interleaved=interleaved) is None
    lens = {0: n}
    for child in range(1, 7):
        pool.fork(0, child, n)
        lens[child] = n
    for child in (7, 8):
        pool.fork(0, child, 40)  # an earlier point: another group
        lens[child] = 40
    pool.allocate(9, 1)          # alone
    lens[9] = 0
    assert pool.shared_runs(sorted(lens)) == ([0, 7, 9, 10], [n // BS, 40 // BS, 0])
    for step in range(20):
        if step == 8:
            pool.release_blocks(3)
            del lens[3]
        ids = sorted(lens)
        if step == 12:
            ids = ids[::-1]
        for s in ids:
            lens[s] += 1
        B = len(ids)
        q, kn, vn = (torch.randn(B, h, D, device="cuda", generator=gen).half() for h in (Hq, Hkv, Hkv))
        out = graph.step(ids, [lens[s] for s in ids], q, kn, vn).clone().unsqueeze(2)
        held = pool.block_table
        at = torch.tensor([lens[s] - 1 for s in ids], device="cuda")
        if dtype == torch.float16:  # the appended rows
            where = torch.tensor([held[s][(lens[s] - 1) // BS] for s in ids], device="cuda")
            assert torch.equal(k[where, at % BS], turned(kn, table, at, interleaved))
            assert torch.equal(v[where, at % BS], vn)
        p = Step(turned(q, table, at, interleaved), k, v, ks, vs, [held[s] for s in ids], [lens[s] for s in ids], BS)
        check(p, out, graph.lse[:B])
    graph.check()
    assert pool.status.item() == 0


class RotatedModel(Model):
    """The small model with rotated queries and keys (fp16 rows, turned in fp32)."""

    def __init__(self, table, *a, **kw):
        super().__init__(*a, **kw)
        self.table = table.cpu()

    def qkv(self, tokens, positions):
        q, k, v = super().qkv(tokens, positions)
        return turned(q, self.table, positions, False), turned(k, self.table, positions, False), v


def search64(model, prompt, K, eos, steps, rule, allowed):
    """Beam search in 64 bits that recomputes everything; ``rule(logits, prompt, line, allowed)`` adjusts a row."""
    beams = [(0.0, [], False)]
    for t in range(steps):
        cand = []
        for j, (s, line, fin) in enumerate(beams):
            if fin:
                cand.append((s, j, eos))
                continue
            lp = torch.log_softmax(rule(model.logits64(prompt + line), prompt, line, allowed(t)), -1)
            cand += [(s + lp[w].item(), j, w) for w in range(model.V)]
        cand.sort(key=lambda c: (-c[0], c[1]))
        beams = [(s, beams[j][1] + [w], beams[j][2] or w == eos) for s, j, w in cand[:K]]
    return beams


@pytest.mark.parametrize("K,prompts,steps,BS", [(3, [21, 37], 12, 16), (6, [16], 9, 4), (1, [5, 3, 9], 6, 2)])
def test_beam_search_with_rules_over_shared_prompts(K, prompts, steps, BS):
    """Append (rotated), attend (prompts read once), adjust, select, reorder, step by step, against the 64-bit search.

    As in the search without rules the fp16 attention outputs make a logit uncertain by 0.02; dividing or multiplying by
    a repetition penalty of 1.3 makes that 0.026 for logits below zero, and a log-softmax takes the difference of
    two: scores are compared within 0.03 a step, the rounding of a logit to fp32 being far below the rest.
    """
    from pie_b200 import ops as o
    from pie_b200.beam import BeamSearch
    from pie_b200.block_pool import DeviceBlockManager

    V, H, Hkv, D, eos, NB = 40, 4, 2, 64, 7, 200
    table = o.rope_table(64, D)
    model = RotatedModel(table, V, H, Hkv, D, seed=K)
    r = np.random.default_rng(K)
    rep, pres, freq = 1.3, 0.4, 0.25
    bias = torch.from_numpy(r.standard_normal(V)).float()
    keep = [r.random(V) < 0.7 for _ in range(steps)]
    for t, m in enumerate(keep):
        m[eos] = t > 2
        m[:K + 1] = True
    words = [torch.from_numpy(np.packbits(np.pad(m, (0, -V % 32)), bitorder="little").view(np.int32).copy()).cuda() for m in keep]

    def rule(x, prompt, line, allowed):
        return torch.from_numpy(ods.adjust_row(x.numpy(), prompt + line, line, rep, pres, freq, bias.numpy(), allowed))

    pool = DeviceBlockManager(NB, BS, 40, 40)
    k, v = (torch.full((NB, BS, Hkv, D), float("nan"), dtype=torch.float16, device="cuda") for _ in range(2))
    pool.attach_caches(k, v)
    lines = [[int(t) for t in r.integers(0, V, n)] for n in prompts]
    out_w, table = model.out.float().cuda(), table.cuda()
    for i, n in enumerate(prompts):
        pool.allocate(i, -(-n // BS))

    def rows(tokens, inp):
        q, kn, vn = (t.cuda() for t in Model.qkv(model, tokens.cpu().long(), inp["positions"].cpu().long()))
        return o.rotate_write_kv(q, kn, vn, table, inp["block_table"], inp["token_seq"], inp["positions"], k, v)

    inp = pool.step_inputs(range(len(prompts)), prompts, prompts)
    q = rows(torch.tensor(sum(lines, [])), inp)
    out, _ = o.paged_attention_varlen(q, inp["cu_seqlens"], k, v, inp["block_table"], inp["num_blocks_per_seq"], BS, inp["kv_len"],
                                      max_q_len=max(prompts))
    logits = (out.float().flatten(1) @ out_w)[inp["cu_seqlens"][1:].long() - 1]
    search = BeamSearch(pool, list(range(len(prompts))), prompts, logits, K, eos, steps, prompt_tokens=lines,
                        repetition_penalty=rep, presence_penalty=pres, frequency_penalty=freq, bias=bias, mask=words[0])
    for t in range(1, steps):
        inp = search.step_inputs()
        assert inp["group_start"].tolist() == [K * i for i in range(len(prompts) + 1)]
        assert inp["prefix_len"].tolist() == [n // BS * BS for n in prompts]
        q = rows(search.tokens.reshape(-1), inp)
        out, _ = o.shared_prefix_attention(q.unsqueeze(2), k, v, inp["q_len"], inp["block_table"], inp["num_blocks_per_seq"], BS,
                                           inp["kv_len"], inp["group_start"], inp["prefix_len"])
        logits = (out[:, :, 0].float().flatten(1) @ out_w).view(len(prompts), K, V)
        mask = words[t]
        if t % 3 == 1:
            mask = mask.expand(len(prompts), -1).contiguous()
        elif t % 3 == 2:
            mask = mask.expand(len(prompts), K, -1).contiguous()
        search.advance(logits, mask)
    found = search.finish()
    assert pool.status.item() == 0 and pool.num_free_blocks() == NB == pool.free_top.item()
    for line, beams in zip(lines, found):
        best = search64(model, line, K, eos, steps, rule, lambda t: keep[t])[0][0]
        assert len(beams) == K
        for score, got in beams:
            exact, ctx = 0.0, []
            for t, w in enumerate(got):
                assert keep[t][w]
                exact += torch.log_softmax(rule(model.logits64(line + ctx), line, ctx, keep[t]), -1)[w].item()
                ctx.append(w)
            assert math.isfinite(score) and abs(score - exact) <= 0.03 * len(got)
        assert beams[0][0] >= best - 0.03 * steps


def test_beam_search_rules_refuse():
    from pie_b200.beam import BeamSearch
    from pie_b200.block_pool import DeviceBlockManager

    NB, BS = 20, 4
    k, v = (torch.zeros(NB, BS, 1, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    pool = DeviceBlockManager(NB, BS, 12, 4)
    pool.attach_caches(k, v)
    for s in (0, 1):
        pool.allocate(s, 2)
    x = torch.zeros(2, 30, device="cuda")
    for bad in (dict(repetition_penalty=1.2), dict(presence_penalty=0.5), dict(prompt_tokens=[[1] * 7]),
                dict(prompt_tokens=[[1] * 7, [2] * 6]), dict(bias=torch.zeros(31, device="cuda")),
                dict(bias=torch.zeros(3, 30, device="cuda")), dict(mask=torch.zeros(2, dtype=torch.int32, device="cuda")),
                dict(mask=torch.zeros(3, 1, dtype=torch.int32, device="cuda")),
                dict(prompt_tokens=[[1] * 7] * 2, repetition_penalty=0.0)):
        with pytest.raises(ValueError):
            BeamSearch(pool, [0, 1], [7, 7], x, 2, 0, 5, **bad)
    pool.flush()
    assert pool.num_free_blocks() == NB - 4 == pool.free_top.item()
    search = BeamSearch(pool, [0, 1], [7, 7], x, 2, 0, 5, bias=torch.ones(2, 30, device="cuda"))
    search.step_inputs()
    with pytest.raises(ValueError):
        search.advance(torch.zeros(2, 2, 30, device="cuda"), torch.zeros(4, 2, dtype=torch.int32, device="cuda"))
    search.advance(torch.zeros(2, 2, 30, device="cuda"))
    search.finish()


@pytest.mark.parametrize("maxq", [1, 3])
def test_an_eager_step_over_forks(maxq):
    """The reference-named wrappers and DeviceBlockManager.shared_prefixes: several new tokens a sequence, forks of forks, one released."""
    from kernels.flash_attention import flash_attention_shared_prefix, rotate_write_kv_cache
    from pie_b200 import ops as o
    from pie_b200.block_pool import DeviceBlockManager

    BS, Hkv, D, Hq, NB, n = 16, 2, 64, 4, 120, 150
    gen = torch.Generator(device="cuda").manual_seed(maxq)
    k, v = (torch.full((NB, BS, Hkv, D), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    pool = DeviceBlockManager(NB, BS, 12, 16)
    pool.attach_caches(k, v)
    table = o.rope_table(300, D, device="cuda")

    def rows(count, heads):
        return torch.randn(count, heads, D, device="cuda", generator=gen).bfloat16()

    pool.allocate(0, -(-n // BS))
    inp = pool.step_inputs([0], [n], [n])
    rotate_write_kv_cache(None, rows(n, Hkv), rows(n, Hkv), table, inp["block_table"], inp["token_seq"], inp["positions"], k, v)
    lens = {0: n, "a": n, "b": 70, "c": 70, 4: n}
    pool.fork(0, "a", n)
    pool.fork("a", "b", 70)
    pool.fork("b", "c", 70)
    pool.fork(0, 4, n)
    pool.release_blocks(0)
    del lens[0]
    ids = ["a", 4, "b", "c"]
    for _ in range(3):
        for s in ids:
            lens[s] += maxq
            need = -(-lens[s] // BS) - pool.blocks_of(s)
            if need:
                pool.allocate(s, need)
        inp = pool.step_inputs(ids, [maxq] * 4, [lens[s] for s in ids])
        q = rotate_write_kv_cache(rows(4 * maxq, Hq), rows(4 * maxq, Hkv), rows(4 * maxq, Hkv), table, inp["block_table"], inp["token_seq"],
                                  inp["positions"], k, v)
        groups = pool.shared_prefixes(ids)
        assert groups["group_start"].tolist() == [0, 2, 4] and groups["prefix_len"].tolist() == [n // BS * BS, 70 // BS * BS]
        Q = q.view(4, maxq, Hq, D).transpose(1, 2)
        out, lse = flash_attention_shared_prefix(Q, k, v, inp["q_len"], inp["block_table"], inp["num_blocks_per_seq"], BS, inp["kv_len"], **groups)
        held = pool.block_table
        p = Step(q.view(4, maxq, Hq, D)[:, 0], k, v, None, None, [held[s] for s in ids], [lens[s] for s in ids], BS)
        p.Q, p.maxq, p.q_len = Q, maxq, inp["q_len"]
        check(p, out, lse)
    with pytest.raises(KeyError):
        pool.shared_prefixes([0])
    assert pool.status.item() == 0
