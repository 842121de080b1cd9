"""GPU: forks, beams and their reordering in the device pool, bit for bit against the list model; beam search end to end."""
import ctypes
import random

import numpy as np
import pytest
import torch

from oracle.block_sharing import SUCCESS, SharedPool
from test_gpu_pages import _i32, host, make_caches, moved, ops, pool_arrays, pool_equals, random_model, same  # noqa: F401

pytestmark = pytest.mark.gpu


def manager(NB=60, BS=4, seqs=12, cols=9, **kw):
    from pie_b200.block_pool import DeviceBlockManager

    dm = DeviceBlockManager(NB, BS, seqs, cols)
    dm.attach_caches(*make_caches(NB, BS, 2, 64, **({"dtype": torch.float16} | kw)))
    return dm


@pytest.mark.parametrize("seed", range(6))
@pytest.mark.parametrize("dtype", [torch.float16, torch.int8])
def test_manager_follows_the_model(seed, dtype):
    """Random allocations, forks, releases and compactions: tables, counts, stack and pages."""
    from pie_b200.block_pool import AllocStatus

    r = random.Random(seed)
    NB, BS, seqs, cols = 60, 4, 12, 9
    dm, model = manager(dtype=dtype, layers=2), SharedPool(NB, seqs, cols, BS)
    want = host(dm.caches)
    nxt = 0
    for step in range(120):
        live = list(dm.ledger.blocks)
        what, copies = r.random(), []
        if what < 0.35 and len(live) < seqs:
            n = r.randint(0, 4)
            if dm.allocate(nxt, n).status is AllocStatus.SUCCESS:
                model.allocate(dm.slot_of(nxt), n)
            nxt += 1
        elif what < 0.75 and live and len(live) < seqs:
            p = r.choice(live)
            n = r.randint(0, dm.blocks_of(p) * BS)
            res = dm.fork(p, nxt, n)
            if res.status is AllocStatus.SUCCESS:
                st, copy = model.fork(dm.slot_of(nxt), n, dm.slot_of(p))
                assert st == SUCCESS
                copies = [copy] if copy else []
            nxt += 1
        elif what < 0.95 and live:
            s = r.choice(live)
            slot = dm.slot_of(s)
            assert dm.release_blocks(s) is AllocStatus.SUCCESS
            model.release(slot)
        elif what >= 0.95:
            dm.compact()
            copies = [(s, d, BS) for s, d in model.compact()[1]]
        moved(want, copies)
        if r.random() < 0.3:
            dm.flush(keep_results=True)
            if dm.last_results is not None:
                assert not dm.last_results.any()
            pool_equals(dm.state, model)
            same(dm.caches, want)
        assert dm.num_free_blocks() == len(model.stack)
    dm.flush()
    model.check()
    pool_equals(dm.state, model)
    same(dm.caches, want)
    assert dm.status.item() == 0


def test_apply_statuses():
    """FORK, ALLOCATE and RELEASE report what they cannot do and change nothing."""
    from pie_b200 import _lib

    dm, lib = manager(NB=5, seqs=4, cols=4), _lib.load()
    rows = [(0, 0, 3, 0), (2, 1, 9, 0), (2, 1, 9, 0), (2, 2, 13, 0), (2, 2, 3, 3), (2, 9, 0, 0), (2, 2, 1, -1), (2, 2, 1, 99),
            (2, 3, 10, 0), (2, 2, 4, 0), (2, 3, 11, 0), (0, 2, 1, 0), (1, 0, 0, 0), (1, 0, 0, 0), (1, 1, 0, 0), (1, 2, 0, 0),
            (7, 0, 0, 0), (0, 0, -1, 0), (2, 0, -3, 1), (0, 0, 5, 0), (0, 0, 2, 0)]
    want = [0, 0, 2, 3, 2, 4, 2, 2, 0, 0, 2, 1, 0, 2, 0, 0, 4, 4, 4, 1, 0]
    # after row 8 all five blocks are held (three, and two copies of last blocks)
    t = _i32(rows)
    res, copies = torch.full((len(rows),), -9, dtype=torch.int32, device="cuda"), torch.empty(3, len(rows), dtype=torch.int32, device="cuda")
    _lib.check("apply", lib.block_pool_apply_shared(ctypes.byref(dm._desc), ctypes.byref(dm._share), t.data_ptr(), len(rows), 4,
                                                    res.data_ptr(), copies[0].data_ptr(), copies[1].data_ptr(),
                                                    copies[2].data_ptr(), None))
    torch.cuda.synchronize()
    assert res.tolist() == want
    # the third block of row 0 is 2 (ids come off the end: 4, 3, 2): copied to 1, then to 0
    assert copies.t().tolist() == [[2, 1, 1] if i == 1 else [2, 0, 2] if i == 8 else [0, 0, 0] for i in range(len(rows))]
    # row 3 of the table still holds 4, 3 and 0; 2 and 1 came back, and row 0 took them again
    model = SharedPool(5, 4, 4, 4)
    for kind, slot, n, parent in rows:
        if slot < 4 and kind in (0, 1, 2) and n >= 0 and 0 <= parent < 4:
            model.allocate(slot, n) if kind == 0 else model.release(slot) if kind == 1 else model.fork(slot, n, parent)
    pool_equals(dm.state, model)


def beam_state(seed, G, K, BS, cols, forks=None, wide=0):
    """Groups of beams as forks and reorderings leave them, with other holders of their prompts."""
    r = np.random.default_rng(seed)
    m = SharedPool(G * (cols + K * cols) + 7, G * K + 4, cols + wide, BS)
    m.stack = r.permutation(m.NB).tolist()
    rows = r.permutation(G * K + 4)
    slots = rows[:G * K].reshape(G, K).tolist()
    lens = []
    for g in range(G):
        n = int(r.integers(1, (cols - 1) * BS))
        m.allocate(slots[g][0], -(-n // BS))
        for s in slots[g][1:]:
            m.fork(s, n, slots[g][0])
        if g < 2:
            m.fork(int(rows[G * K + g]), n // BS * BS, slots[g][0])
        while n < cols * BS - BS and r.random() < 0.95:
            if n % BS == 0:
                for s in slots[g]:
                    m.allocate(s, 1)
            n += 1
            slots[g], _, freed = m.reorder(slots[g], r.integers(0, K, K).tolist(), n)
            m.push(freed)
        lens.append(n)
    m.check()
    return m, slots, lens


@pytest.mark.parametrize("G,K,BS,cols", [(1, 1, 4, 5), (1, 2, 1, 6), (3, 4, 4, 7), (2, 32, 2, 5), (9, 5, 16, 3), (40, 7, 2, 12), (2, 3, 1, 2600)])
@pytest.mark.parametrize("dtype,layers,layout", [(torch.int8, 1, "slots"), (torch.float16, 3, "heads"), (torch.bfloat16, 65, "wide")])
def test_reorder(ops, G, K, BS, cols, dtype, layers, layout):  # noqa: F811
    if cols > 1000 and layers > 3:
        pytest.skip("the long tables are covered by the smaller layer counts")
    m, slots, lens = beam_state(G * K + BS, G, K, BS, cols)
    r = np.random.default_rng(1)
    pool = pool_arrays(ops, m, m.max_blocks)
    caches = make_caches(m.NB, BS, 1, 64, dtype, layers, layout)
    want = host(caches)
    st = _i32([0])
    dev_slots = _i32(slots)
    for _ in range(3):  # again and again over the same tokens
        parents = r.integers(0, K, (G, K))
        new, freed, copies = [], [], []
        for g in range(G):
            o, c, f = m.reorder(slots[g], parents[g].tolist(), lens[g])
            new.append(o)
            copies += c
            freed += f
        m.push(freed)
        m.check()
        slots = new
        dev_slots = ops.reorder_beams(pool, dev_slots, _i32(parents), _i32(lens), *caches, status=st)
        assert dev_slots.tolist() == slots
        pool_equals(pool, m)
        same(caches, moved(want, copies))
    assert st.item() == 0
    assert not pool.scratch[:16].any() and not pool.scratch[16:16 + (m.NB + 31) // 32].any()


def test_reorder_leaves_bad_groups_alone(ops):  # noqa: F811
    m, slots, lens = beam_state(5, 6, 3, 4, 6, wide=2)
    pool = pool_arrays(ops, m, m.max_blocks)
    caches = make_caches(m.NB, 4, 1, 64, torch.float16)
    want = host(caches)
    parents = np.array([[0, 0, 2], [0, 3, 1], [0, -1, 1], [1, 1, 0], [2, 2, 2], [1, 1, 1]])
    bad = [list(s) for s in slots]
    bad[0][1] = bad[0][0]               # a row twice
    bad[3][2] = len(m.rows)             # no such row
    wrong = list(lens)
    wrong[4] = 4 * (len(m.rows[slots[4][0]]) + 1)  # more tokens than blocks
    st = _i32([0])
    got = ops.reorder_beams(pool, _i32(bad), _i32(parents), _i32(wrong), *caches, status=st)
    new, copies, freed = m.reorder(slots[5], [1, 1, 1], lens[5])
    m.push(freed)
    assert got.tolist() == bad[:5] + [new]
    assert st.item() == 2 | 8
    pool_equals(pool, m)
    same(caches, moved(want, copies))
    # rows of one group with different numbers of blocks, and a row without an entry
    st.zero_()
    s = slots[0]
    m.allocate(s[2], 1)
    pool = pool_arrays(ops, m, m.max_blocks)
    assert ops.reorder_beams(pool, _i32([s]), _i32([[0, 0, 0]]), _i32(lens[:1]), *caches, status=st).tolist() == [s]
    free_row = next(i for i, x in enumerate(m.rows) if x is None)
    ops.reorder_beams(pool, _i32([[s[0], s[1], free_row]]), _i32([[0, 0, 0]]), _i32(lens[:1]), *caches, status=st)
    ops.reorder_beams(pool, _i32([s[:2]]), _i32([[0, 0]]), _i32([-1]), *caches, status=st)
    assert st.item() == 2
    pool_equals(pool, m)


def test_reorder_refusals(ops):  # noqa: F811
    m, slots, lens = beam_state(5, 2, 3, 4, 6)
    pool = pool_arrays(ops, m, m.max_blocks)
    caches = make_caches(m.NB, 4, 1, 64, torch.float16)
    s, n = _i32(slots), _i32(lens)
    with pytest.raises(ValueError):
        ops.reorder_beams(pool, s, s[:1], n, *caches)
    with pytest.raises(ValueError):
        ops.reorder_beams(pool, s, s, n[:1], *caches)
    with pytest.raises(ValueError):
        ops.reorder_beams(pool, s.cpu(), s, n, *caches)
    with pytest.raises(RuntimeError, match="scratch"):
        ops.reorder_beams(pool._replace(scratch=pool.scratch[:-1].contiguous()), s, s, n, *caches)
    with pytest.raises((RuntimeError, ValueError), match="hold"):
        ops.reorder_beams(pool, s, s, n, caches[0][0][:-1], caches[1][0][:-1])
    wide = torch.zeros(1, 33, dtype=torch.int32, device="cuda")
    with pytest.raises(RuntimeError, match="num_beams"):
        ops.reorder_beams(pool, wide, wide, n[:1], *caches)
    empty = ops.reorder_beams(pool, s[:0], s[:0], n[:0], *caches)
    assert tuple(empty.shape) == (0, 3)
    pool_equals(pool, m)


def test_captured_reorder_and_compaction():
    """A step captured once, replayed over changing parents and tokens, with a compaction between."""
    from pie_b200 import ops as o

    m, slots, lens = beam_state(3, 4, 4, 4, 8)
    pool, caches = pool_arrays(o, m, m.max_blocks), make_caches(m.NB, 4, 2, 64, torch.int8)
    want = host(caches)
    s, p, n = _i32(slots), _i32(np.zeros((4, 4))), _i32(lens)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    g1, g2 = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g1, stream=side):
        s.copy_(o.reorder_beams(pool, s, p, n, *caches))
    with torch.cuda.graph(g2, stream=side):
        o.compact_blocks(pool, *caches)
    r = np.random.default_rng(0)
    for _ in range(4):
        parents = r.integers(0, 4, (4, 4))
        p.copy_(_i32(parents))
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            g1.replay()
            g2.replay()
        torch.cuda.synchronize()
        freed, copies = [], []
        for i in range(4):
            slots[i], c, f = m.reorder(slots[i], parents[i].tolist(), lens[i])
            freed += f
            copies += c
        m.push(freed)
        moved(want, copies)
        moved(want, [(a, b, 4) for a, b in m.compact()[1]])
        assert s.tolist() == slots
        pool_equals(pool, m)
        same(caches, want)


def test_shrunk_pool_goes_on(ops):  # noqa: F811
    """After a compaction to fewer blocks the manager forks, reorders and frees within them."""
    dm = manager(NB=200, seqs=12, cols=9)
    model = SharedPool(200, 12, 9, 4)
    for s in range(6):
        dm.allocate(s, 3)
        model.allocate(dm.slot_of(s), 3)
    for s in (0, 2, 4):
        slot = dm.slot_of(s)
        dm.release_blocks(s)
        model.release(slot)
    with pytest.raises(ValueError):
        dm.compact(8)
    live = dm.compact(20)
    model.compact(20)
    assert live.item() == 9 and dm.num_blocks == 20 and dm.num_free_blocks() == 11
    model.NB, model.ref = 20, model.ref[:20]
    dm.attach_caches(*[None if c is None else [t[:20].clone() for t in c] for c in (dm.caches[0], dm.caches[1], None, None)])
    dm.fork_beams(1, ["a", "b"], 10)
    for b in ("a", "b"):
        model.fork(dm.slot_of(b), 10, dm.slot_of(1))
    slots = dm.beam_slots([1])
    got = dm.reorder_beams(slots, _i32([[1, 1, 0]]), _i32([10]))
    new, _, freed = model.reorder(slots.tolist()[0], [1, 1, 0], 10)
    model.push(freed)
    assert got.tolist() == [new]
    pool_equals(dm.state, model)
    dm.release_beams(1)
    dm.flush()
    assert dm.free_top.item() == dm.num_free_blocks() == 14
    assert sorted(dm.free_list()) == sorted(set(range(20)) - set(b for r in dm.block_table.values() for b in r))


def test_manager_refusals():
    from pie_b200.block_pool import AllocStatus, DeviceBlockManager

    dm = DeviceBlockManager(20, 4, 6, 8)
    dm.allocate(0, 2)
    for call in (lambda: dm.fork(0, 1, 5), lambda: dm.fork_beams(0, [1], 5), lambda: dm.compact(),
                 lambda: dm.reorder_beams(_i32([[0]]), _i32([[0]]), _i32([0]))):
        with pytest.raises(ValueError, match="attach_caches"):
            call()
    assert dm.fork(0, 1, 8).status is AllocStatus.SUCCESS  # full blocks move no page
    for bad in (make_caches(19, 4, 1, 64, torch.float16), make_caches(20, 8, 1, 64, torch.float16)):
        with pytest.raises(ValueError):
            dm.attach_caches(*bad)
    with pytest.raises(ValueError):
        dm.attach_caches(torch.zeros(20, 4, 1, 64), torch.zeros(20, 4, 1, 64))
    dm.flush()
    assert dm.ref_count.tolist()[-2:] == [2, 2]


# ---- beam search over a small attention model ------------------------------------------
class Model:
    """One paged attention layer between an embedding and a vocabulary."""

    def __init__(self, V, H, Hkv, D, seed=0):
        g = torch.Generator().manual_seed(seed)
        self.V, self.H, self.Hkv, self.D = V, H, Hkv, D
        self.emb = torch.randn(V + 64, 3, H * D, generator=g, dtype=torch.float64) * 0.7
        self.out = torch.randn(H * D, V, generator=g, dtype=torch.float64) * 0.6

    def qkv(self, tokens, positions):
        e = self.emb[tokens] + self.emb[self.V + positions]
        q, k, v = e.unbind(-2)
        D = self.D
        return (q.half().view(-1, self.H, D), k.half().view(-1, self.H, D)[:, :self.Hkv], v.half().view(-1, self.H, D)[:, :self.Hkv])

    def logits64(self, tokens):
        """Of the last token, in 64 bits from the fp16 rows."""
        q, k, v = (t.double() for t in self.qkv(torch.tensor(tokens), torch.arange(len(tokens))))
        rep = self.H // self.Hkv
        k, v = k.repeat_interleave(rep, 1), v.repeat_interleave(rep, 1)
        a = torch.softmax(torch.einsum("hd,thd->ht", q[-1], k) / self.D**0.5, -1)
        return torch.einsum("ht,thd->hd", a, v).reshape(-1) @ self.out


def search64(model, prompt, K, eos, steps):
    beams = [(0.0, [], False)]
    for _ in range(steps):
        cand = []
        for j, (s, line, fin) in enumerate(beams):
            if fin:
                cand.append((s, j, eos))
                continue
            lp = torch.log_softmax(model.logits64(prompt + line), -1)
            cand += [(s + lp[t].item(), j, t) for t in range(model.V)]
        cand.sort(key=lambda c: (-c[0], c[1]))
        beams = [(s, beams[j][1] + [t], beams[j][2] or t == eos) for s, j, t in cand[:K]]
    return [(s, line[:line.index(eos) + 1] if eos in line else line) for s, line, _ in beams]


@pytest.mark.parametrize("BS,K,prompts,steps", [(4, 3, [5, 8, 1], 11), (16, 4, [16, 30], 20), (2, 1, [3], 5), (1, 5, [4, 2], 6)])
def test_beam_search_matches_a_search_without_a_cache(BS, K, prompts, steps):
    """Prefill, then select -> reorder -> write -> attend per step, against a 64-bit search that recomputes everything.

    The attention outputs are fp16 (2^-11 of values up to 3, through 128 random weights of 0.6: about 0.02 in a logit),
    so the searches are compared by score: each found line is rescored in 64 bits, and the best score reached may fall
    short of the 64-bit search's by what the scores are uncertain by, 0.02 a step.
    """
    from pie_b200 import ops as o
    from pie_b200.beam import BeamSearch
    from pie_b200.block_pool import DeviceBlockManager

    V, H, Hkv, D, eos = 40, 2, 1, 64, 7
    model = Model(V, H, Hkv, D, seed=BS)
    NB = 160
    pool = DeviceBlockManager(NB, BS, 40, 64)
    k, v = (torch.zeros(NB, BS, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(2))
    pool.attach_caches(k, v)
    r = random.Random(K)
    lines = [[r.randrange(V) for _ in range(n)] for n in prompts]
    out_w = model.out.float().cuda()
    for i, n in enumerate(prompts):
        pool.allocate(i, -(-n // BS))
    inp = pool.step_inputs(range(len(prompts)), prompts, prompts)

    def attend(tokens, inp, max_q):
        q, kn, vn = (t.cuda() for t in model.qkv(tokens.cpu().long(), inp["positions"].cpu().long()))
        o.write_kv(kn, vn, inp["block_table"], inp["token_seq"], inp["positions"], k, v)
        out, _ = o.paged_attention_varlen(q, inp["cu_seqlens"], k, v, inp["block_table"], inp["num_blocks_per_seq"], BS,
                                          inp["kv_len"], max_q_len=max_q)
        return out.float().reshape(out.shape[0], -1) @ out_w

    last = inp["cu_seqlens"][1:].long() - 1
    logits = attend(torch.tensor(sum(lines, [])), inp, max(prompts))[last]
    free0 = pool.num_free_blocks()
    search = BeamSearch(pool, list(range(len(prompts))), prompts, logits, K, eos, steps)
    for _ in range(steps - 1):
        inp = search.step_inputs()
        logits = attend(search.tokens.reshape(-1), inp, 1).view(len(prompts), K, V)
        search.advance(logits)
    with pytest.raises(RuntimeError):
        search.step_inputs()
    slots = search.slots
    assert sorted(slots.view(-1).tolist()) == sorted(pool.ledger.slot.values())
    found = search.finish()
    assert pool.status.item() == 0
    assert pool.num_free_blocks() == NB == pool.free_top.item() and free0 <= NB
    assert not pool.ref_count.any()
    for line, beams in zip(lines, found):
        want = search64(model, line, K, eos, steps)
        assert len(beams) == K and [s for s, _ in beams] == sorted((s for s, _ in beams), reverse=True)
        assert len({tuple(t) for _, t in beams}) == K
        for score, got in beams:
            exact, ctx = 0.0, list(line)
            for t in got:
                exact += torch.log_softmax(model.logits64(ctx), -1)[t].item()
                ctx.append(t)
            assert abs(score - exact) <= 0.02 * len(got)
        assert beams[0][0] >= want[0][0] - 0.02 * steps


def test_beam_search_that_cannot_start_leaves_the_prompts():
    from pie_b200.beam import BeamSearch
    from pie_b200.block_pool import AllocStatus

    dm = manager(NB=8, seqs=12, cols=4)
    for s in (0, 1):
        dm.allocate(s, 2)
    x = torch.zeros(2, 30, device="cuda")
    with pytest.raises(RuntimeError, match="INSUFFICIENT"):
        BeamSearch(dm, [0, 1], [7, 7], x, 4, 0, 5)  # three forks each, four free blocks
    for bad in (dict(logits=x[:1]), dict(num_beams=0), dict(num_beams=31), dict(max_new_tokens=0), dict(eos_id=30),
                dict(eos_id=-1), dict(logits=x.double()), dict(num_tokens=[7, 3]), dict(seq_ids=[1, 1])):
        with pytest.raises(ValueError):
            BeamSearch(**(dict(pool=dm, seq_ids=[0, 1], num_tokens=[7, 7], logits=x, num_beams=2, eos_id=0, max_new_tokens=5) | bad))
    dm.flush()
    assert dm.num_free_blocks() == 4 == dm.free_top.item()
    assert dm.release_blocks(0) is AllocStatus.SUCCESS
    search = BeamSearch(dm, [1], [7], x[:1], 3, 0, 5)
    with pytest.raises(RuntimeError, match="step_inputs"):
        search.advance(x[:1].expand(1, 3, 30))
    search.step_inputs()
    with pytest.raises(ValueError):
        search.advance(x[:1])
    search.advance(x[:1].expand(1, 3, 30))
    search.step_inputs()
    search.step_inputs()  # again: nothing more is taken
    assert dm.num_free_blocks() == 1  # one shared block, and two for each beam
    search.finish()
    search.finish()
    with pytest.raises(RuntimeError, match="ended"):
        search.step_inputs()
    assert dm.num_free_blocks() == 8 == dm.free_top.item()


def test_beam_search_that_has_ended_moves_no_blocks():
    """advance() after finish(): its rows may belong to others by now."""
    from pie_b200.beam import BeamSearch

    x = torch.randn(1, 30, device="cuda")
    dm = manager(NB=12, seqs=4, cols=4)
    dm.allocate(0, 2)
    search = BeamSearch(dm, [0], [7], x, 2, 0, 9)
    search.step_inputs()
    search.finish()
    for s in (5, 6, 7, 8):  # all rows, with as many blocks each as a beam had
        dm.allocate(s, 2)
    dm.flush()
    before = [t.cpu() for t in dm.state[:5]]
    with pytest.raises(RuntimeError, match="ended"):
        search.advance(x.expand(1, 2, 30))
    assert all(torch.equal(a, b.cpu()) for a, b in zip(before, dm.state))


def test_beam_search_needs_the_caches_from_the_start():
    from pie_b200.beam import BeamSearch
    from pie_b200.block_pool import DeviceBlockManager

    dm = DeviceBlockManager(8, 4, max_seqs=4, max_blocks_per_seq=4)
    dm.allocate(0, 2)
    with pytest.raises(ValueError, match="attach_caches"):
        BeamSearch(dm, [0], [8], torch.zeros(1, 30, device="cuda"), 2, 0, 5)  # full blocks: no fork copies
    assert dm.num_free_blocks() == 6


def test_beam_search_at_the_ends_of_the_pool():
    """A row without room, and a pool without blocks: step_inputs refuses, takes nothing, and goes on when there is room."""
    from pie_b200.beam import BeamSearch

    x = torch.randn(1, 30, device="cuda")
    dm = manager(NB=8, seqs=12, cols=2)
    dm.allocate(0, 2)
    search = BeamSearch(dm, [0], [8], x, 2, 0, 9)
    with pytest.raises(RuntimeError, match="max_blocks_per_seq"):
        search.step_inputs()
    assert dm.num_free_blocks() == 6
    dm = manager(NB=6, seqs=12, cols=5)
    dm.allocate("other", 3)
    dm.allocate(0, 2)
    search = BeamSearch(dm, [0], [8], x, 2, 0, 9)
    with pytest.raises(RuntimeError, match="free"):
        search.step_inputs()
    dm.release_blocks("other")
    inp = search.step_inputs()
    assert inp["num_blocks_per_seq"].tolist() == [3, 3] and dm.num_free_blocks() == 2
    search.finish()
    assert dm.num_free_blocks() == 6 == dm.free_top.item()


def test_decode_graph_over_forked_sequences():
    """The captured decode step over a sequence and its forks: each attends to its own continuation of the shared prompt."""
    from pie_b200 import ops as o
    from pie_b200.block_pool import DeviceBlockManager
    from pie_b200.decode_step import DecodeStepGraph

    BS, Hkv, D, Hq, NB, n = 16, 2, 64, 4, 40, 21
    g = torch.Generator(device="cuda").manual_seed(4)
    k, v = (torch.zeros(NB, BS, Hkv, D, dtype=torch.float16, device="cuda") for _ in range(2))
    pool = DeviceBlockManager(NB, BS, 8, 6)
    pool.attach_caches(k, v)
    graph = DecodeStepGraph(pool, k, v, None, None, Hq, 4)
    pool.allocate(0, 2)
    inp = pool.step_inputs([0], [n], [n])
    rows = [torch.randn(n, Hkv, D, device="cuda", generator=g).half() for _ in range(2)]
    o.write_kv(*rows, inp["block_table"], inp["token_seq"], inp["positions"], k, v)
    pool.fork(0, 1, n)
    pool.fork(0, 2, 18)  # an earlier point
    pool.fork(1, 3, n)   # a fork of a fresh fork
    lens, have = [n, n, 18, n], [[r[:m] for r in rows] for m in (n, n, 18, n)]
    for _ in range(15):
        lens = [m + 1 for m in lens]
        q, kn, vn = (torch.randn(4, h, D, device="cuda", generator=g).half() for h in (Hq, Hkv, Hkv))
        out = graph.step([0, 1, 2, 3], lens, q, kn, vn).clone()
        for i in range(4):
            have[i] = [torch.cat([have[i][0], kn[i:i + 1]]), torch.cat([have[i][1], vn[i:i + 1]])]
            rep = Hq // Hkv
            kk, vv = (t.double().repeat_interleave(rep, 1) for t in have[i])
            a = torch.softmax(torch.einsum("hd,thd->ht", q[i].double(), kk) / D**0.5, -1)
            want = torch.einsum("ht,thd->hd", a, vv)
            # fp16 probabilities and output: 2^-11 each of values up to 4, and the exponentials' 2^-11 of the logits
            assert (out[i].double() - want).abs().max() < 8e-3
    graph.check()
    assert pool.status.item() == 0


def test_checked_mode_raises_what_the_status_says(monkeypatch):
    """PIE_B200_CHECK: the skipped pairs and groups become IndexErrors."""
    from pie_b200 import ops as o

    monkeypatch.setattr(o, "_CHECK", True)
    caches = make_caches(8, 16, 1, 64, torch.float16)
    o.copy_blocks(caches[0], caches[1], _i32([1]), _i32([2]))
    with pytest.raises(IndexError, match="another copy"):
        o.copy_blocks(caches[0], caches[1], _i32([1, 3]), _i32([2, 2]))
    with pytest.raises(IndexError, match="block id"):
        o.copy_blocks(caches[0], caches[1], _i32([1]), _i32([8]))
    m, slots, lens = beam_state(5, 2, 3, 4, 6)
    pool, caches = pool_arrays(o, m, m.max_blocks), make_caches(m.NB, 4, 1, 64, torch.float16)
    o.reorder_beams(pool, _i32(slots), _i32([[0, 1, 2]] * 2), _i32(lens), *caches)
    with pytest.raises(IndexError, match="sequence index"):
        o.reorder_beams(pool, _i32(slots), _i32([[0, 1, 3]] * 2), _i32(lens), *caches)
    with pytest.raises(IndexError, match="contradict"):
        o.compact_blocks(pool, *caches, num_blocks=1)
    o.compact_blocks(pool, *caches)


def test_a_beam_id_never_names_another_beams_row():
    """After a reordering the manager's older methods refuse the beams, and take the ids again once they are released."""
    from pie_b200 import ops as o
    from pie_b200.beam import BeamSearch
    from pie_b200.block_pool import DeviceBlockManager
    from pie_b200.decode_step import DecodeStepGraph

    NB, BS = 40, 16
    k, v = (torch.zeros(NB, BS, 2, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    pool = DeviceBlockManager(NB, BS, 8, 6)
    pool.attach_caches(k, v)
    graph = DecodeStepGraph(pool, k, v, None, None, 2, 3)
    pool.allocate(0, 2)
    pool.allocate(5, 1)
    search = BeamSearch(pool, [0], [20], torch.randn(1, 30, device="cuda"), 3, 0, 5)
    assert set(pool.block_table) == {DecodeStepGraph.PAD_SEQ, 0, 5, (0, 1), (0, 2)}
    inp = pool.step_inputs([0, 5, (0, 2)], [1, 1, 1], [20, 9, 20])
    assert inp["block_table"][0, 0] == inp["block_table"][2, 0] != inp["block_table"][1, 0]
    search.step_inputs()
    search.advance(torch.randn(1, 3, 30, device="cuda"))
    rows = torch.ones(1, 2, 64, dtype=torch.float16, device="cuda")
    before = [t.cpu() for t in pool.state[:5]]
    for s in (0, (0, 1), (0, 2)):
        for call in (lambda: pool.slot_of(s), lambda: pool.step_inputs([s], [1], [21]), lambda: pool.beam_slots([0]),
                     lambda: pool.block_table, lambda: graph.step([s], [22], rows, rows, rows)):
            with pytest.raises(ValueError, match="beam of"):
                call()
    assert graph.step([5], [10], rows, rows, rows).shape == (1, 2, 64)
    assert all(torch.equal(a, b.cpu()) for a, b in zip(before, pool.state))
    mine = {pool.table[pool.slot_of(s), 0].item() for s in (5, DecodeStepGraph.PAD_SEQ)}
    assert set(k.flatten(1).any(1).nonzero().flatten().tolist()) <= mine  # no beam's page was written
    search.finish()
    pool.allocate(0, 1)
    assert len(pool.block_table[0]) == 1 and pool.step_inputs([0], [1], [3])["num_blocks_per_seq"].tolist() == [1]


def test_reorder_refuses_tokens_inside_a_shared_block(ops):  # noqa: F811
    """Tokens rolled back below a shared block's end, in a group or to another sequence: left as they are, others go on."""
    BS = 4
    m = SharedPool(60, 12, 5, BS)
    caches = make_caches(m.NB, BS, 2, 64, torch.float16, 2)
    want = host(caches)
    groups = [[0, 1, 2], [5, 4, 3], [6, 7, 8]]
    for g in groups:
        m.allocate(g[0], 1)
        for s in g[1:]:
            m.fork(s, BS, g[0])
        for s in g:
            m.allocate(s, 1)
    m.push(m.reorder(groups[0], [1, 1, 2], 8)[2])   # beams 0 and 1 hold one second block
    m.fork(9, 8, groups[1][2])                      # another sequence holds beam 2's second block
    assert [m.may_reorder(g, 6) for g in groups] == [False, False, True]
    pool, st = pool_arrays(ops, m, m.max_blocks), _i32([0])
    parents = [[2, 2, 0], [1, 1, 0], [2, 0, 2]]
    got = ops.reorder_beams(pool, _i32(groups), _i32(parents), _i32([6, 7, 5]), *caches, status=st)
    new, copies, freed = m.reorder(groups[2], parents[2], 5)
    m.push(freed)
    m.check()
    assert got.tolist() == groups[:2] + [new] and st.item() == 128
    pool_equals(pool, m)
    same(caches, moved(want, copies))
    st.zero_()
    got = ops.reorder_beams(pool, _i32(groups[:2]), _i32(parents[:2]), _i32([4, 8]), *caches, status=st)  # whole blocks
    after = []
    for g, p, n in zip(groups, parents, (4, 8)):
        new, copies, freed = m.reorder(g, p, n)
        after.append(new)
        m.push(freed)
        assert not copies
    assert got.tolist() == after and st.item() == 0
    pool_equals(pool, m)


@pytest.mark.parametrize("wrong,refused", [(1000, True), (-5, True), (-3, False), (0, False)])
def test_a_search_that_left_the_pool_behind_returns_no_lines(wrong, refused):
    """A reordering that leaves a group as it is (the token count does not fit the rows): finish says so, and frees.

    The second sequence is at 8 tokens then, in blocks of 4: 3 tokens end inside the first block, which its beams share,
    5 inside the second, of which each has its own.
    """
    from pie_b200.beam import BeamSearch

    dm = manager(NB=40, seqs=12, cols=6)
    dm.allocate(0, 2)
    dm.allocate(1, 2)
    x = torch.randn(2, 30, device="cuda")
    dm.status.fill_(2)  # of something else: not the search's
    search = BeamSearch(dm, [0, 1], [7, 6], x, 3, 0, 9)
    for step in range(3):
        search.step_inputs()
        if step == 1:
            search.num_tokens[1] += wrong
        search.advance(torch.randn(2, 3, 30, device="cuda"))
    if refused:
        for _ in range(2):
            with pytest.raises(IndexError, match="beam search"):
                search.finish()
    else:
        assert [len(b) for b in search.finish()] == [3, 3]
    dm.flush()
    assert dm.num_free_blocks() == 40 == dm.free_top.item() and dm.status.item() == 2


@pytest.mark.parametrize("NB", [60, 20])
def test_sole_batches_keep_the_counts(NB):
    """More operations than a launch stages at once, refused ones among them: statuses, rows and counts as the general call's."""
    from pie_b200 import _lib

    r, lib = np.random.default_rng(3), _lib.load()
    rows = [(int(k), int(s), int(n)) for k, s, n in zip(r.choice([0, 0, 1, 5], 700), r.integers(-1, 13, 700), r.integers(-1, 5, 700))]
    a, b = manager(NB, seqs=12, cols=9), manager(NB, seqs=12, cols=9)
    res = torch.full((2, len(rows)), -9, dtype=torch.int32, device="cuda")
    t3, t4 = _i32(rows), _i32([(*x, 0) for x in rows])
    _lib.check("sole", lib.block_pool_apply_sole(ctypes.byref(a._desc), ctypes.byref(a._share), t3.data_ptr(), len(rows),
                                                 res[0].data_ptr(), None))
    _lib.check("shared", lib.block_pool_apply_shared(ctypes.byref(b._desc), ctypes.byref(b._share), t4.data_ptr(), len(rows), 4,
                                                     res[1].data_ptr(), None, None, None, None))
    torch.cuda.synchronize()
    model, want = SharedPool(NB, 12, 9, 4), []
    for kind, slot, n in rows:
        ok = kind in (0, 1) and 0 <= slot < 12 and n >= 0
        want.append(4 if not ok else model.allocate(slot, n) if kind == 0 else model.release(slot))
    assert res[0].tolist() == res[1].tolist() == want and (1 in want) == (NB == 20)
    pool_equals(a.state, model)
    pool_equals(b.state, model)


def test_blocks_that_reorderings_freed_can_be_had():
    """Beams that follow one line hold few blocks: the next step, other sequences and a smaller pool get the others."""
    from pie_b200.beam import BeamSearch
    from pie_b200.block_pool import AllocStatus

    dm = manager(NB=24, seqs=12, cols=9)
    dm.allocate(0, 2)
    dm.allocate(1, 1)
    x = torch.full((1, 30), -9.0, device="cuda")
    x[0, 1:5] = torch.tensor([5.0, 1.0, 0.5, 0.0], device="cuda")
    pull = x.expand(1, 4, 30).clone()
    search = BeamSearch(dm, [0], [6], x, 4, 0, 40)
    other = BeamSearch(dm, [1], [4], x, 2, 0, 40)
    for step in range(24):  # 6 columns of 4 blocks, were they private: more than there are
        search.step_inputs()
        search.scores[:, 1:] -= 1000.0  # the best beam has all children
        search.advance(pull)
    other.step_inputs()
    other.advance(pull[:, :2])
    assert dm.status.item() == 0 == search.status.item()
    before = dm.num_free_blocks()
    assert dm.recount() == dm.free_top.item() == dm.num_free_blocks() >= before
    assert dm.recount() == dm.free_top.item()  # again: the same
    spare = dm.num_free_blocks()
    assert spare >= 8 and dm.allocate("late", spare - 6).status is AllocStatus.SUCCESS
    for _ in range(2):
        search.step_inputs()
        search.scores[:, 1:] -= 1000.0
        search.advance(pull)
    with pytest.raises(ValueError, match="in use"):
        dm.compact(3)
    used = 24 - dm.recount()
    assert dm.compact(used + 1).item() == used and dm.num_free_blocks() == dm.free_top.item() == 1
    search.finish()
    assert dm.num_free_blocks() <= dm.free_top.item()
    other.finish()
    dm.release_blocks("late")
    assert dm.num_free_blocks() == used + 1 == len(dm.free_list()) and not dm.ref_count.any() and not dm.block_table


@pytest.mark.parametrize("seed", range(6))
def test_manager_with_searches_follows_the_model(seed):
    """Plain sequences, forks, searches, recounts and compactions in any order: tables, counts, stack, pages and free blocks."""
    from pie_b200.block_pool import AllocStatus

    r = random.Random(40 + seed)
    NB, BS, seqs, cols = 110, 4, 18, 9
    dm, model = manager(NB, BS, seqs, cols, layers=2), SharedPool(NB, seqs, cols, BS)
    want = host(dm.caches)
    plain, groups, nxt, queue = {}, {}, 0, []

    def applied():  # the list model follows the queued calls, in order
        for op in queue:
            op()
        queue.clear()

    def forked(slot, n, parent):
        st, copy = model.fork(slot, n, parent)
        assert st == SUCCESS
        moved(want, [copy] if copy else [])

    for _ in range(220):
        what = r.random()
        if what < 0.2 and len(dm.ledger.blocks) < seqs:
            n = r.randint(0, 14)
            if dm.allocate(nxt, -(-n // BS)).status is AllocStatus.SUCCESS:
                plain[nxt] = n
                queue.append(lambda s=dm.slot_of(nxt), k=-(-n // BS): model.allocate(s, k))
            nxt += 1
        elif what < 0.35 and plain and len(dm.ledger.blocks) < seqs:
            p = r.choice(list(plain))
            n = r.randint(0, plain[p])
            if dm.fork(p, nxt, n).status is AllocStatus.SUCCESS:
                plain[nxt] = n
                queue.append(lambda s=dm.slot_of(nxt), n=n, p=dm.slot_of(p): forked(s, n, p))
            nxt += 1
        elif what < 0.45 and plain:
            p, k = r.choice(list(plain)), r.randint(1, 4)
            if len(dm.ledger.blocks) + k - 1 <= seqs and (plain[p] % BS == 0 or dm.ledger.shared_columns(p) <= plain[p] // BS):
                if dm.fork_beams(p, [(p, j) for j in range(1, k)], plain[p]) is AllocStatus.SUCCESS:
                    slots = [dm.slot_of(b) for b in dm.ledger.beams[p]]
                    groups[p] = [slots, plain.pop(p)]
                    for s in slots[1:]:
                        queue.append(lambda s=s, n=groups[p][1], q=slots[0]: forked(s, n, q))
        elif what < 0.75 and groups:  # a step of one search
            g = r.choice(list(groups))
            slots, n = groups[g]
            if n % BS == 0:
                if n // BS >= cols or dm.allocate_beams(g, 1) is not AllocStatus.SUCCESS:
                    continue
                queue += [lambda s=dm.ledger.slot[b]: model.allocate(s, 1) for b in dm.ledger.beams[g]]
            applied()
            parents = [r.randrange(len(slots)) for _ in slots]
            out = dm.reorder_beams(_i32([slots]), _i32([parents]), _i32([n + 1]))
            new, copies, freed = model.reorder(slots, parents, n + 1)
            model.push(freed)
            moved(want, copies)
            assert out.tolist() == [new]
            groups[g] = [new, n + 1]
        elif what < 0.82 and groups:
            g = r.choice(list(groups))
            rows = [dm.ledger.slot[b] for b in dm.ledger.beams[g]]
            del groups[g]
            assert dm.release_beams(g) is AllocStatus.SUCCESS
            queue += [lambda s=s: model.release(s) for s in rows]
        elif what < 0.9 and plain:
            p = r.choice(list(plain))
            del plain[p]
            queue.append(lambda s=dm.slot_of(p): model.release(s))
            assert dm.release_blocks(p) is AllocStatus.SUCCESS
        elif what < 0.95:
            dm.recount()
            dm.flush()
            applied()
            assert dm.num_free_blocks() == len(model.stack) == dm.free_top.item()
        else:
            dm.compact()
            applied()
            moved(want, [(s, d, BS) for s, d in model.compact()[1]])
        if r.random() < 0.2:
            dm.flush()
            applied()
            model.check()
            pool_equals(dm.state, model)
            same(dm.caches, want)
            assert dm.num_free_blocks() <= len(model.stack)
    for g in list(groups):
        dm.release_beams(g)
    for p in plain:
        dm.release_blocks(p)
    dm.flush()
    assert dm.num_free_blocks() == NB == dm.free_top.item() and not dm.ref_count.any() and dm.status.item() == 0
