"""GPU: page copies and pool compaction, bit for bit against list models."""
import numpy as np
import pytest
import torch

from oracle.block_sharing import SharedPool, copy_pages

pytestmark = pytest.mark.gpu


@pytest.fixture(params=["torch", "ctypes"])
def ops(request, monkeypatch):
    from pie_b200 import ops as o

    monkeypatch.setattr(o, "BACKEND", request.param)
    return o


def _i32(a):
    return torch.tensor(np.asarray(a), dtype=torch.int32, device="cuda")


def make_caches(NB, BS, H, D, dtype, layers=1, layout="slots", scales="token16", seed=0, heads=None):
    """Lists of K, V and scale pools as [block, slot, head, d] views with random bytes."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for _ in range(2):
        pools = []
        for _ in range(layers):
            shape = dict(slots=(NB, BS, H, D), heads=(NB, H, BS, D), wide=(NB, BS, H + 3, D), layers=(NB, 2, BS, H, D))[layout]
            t = torch.randint(-127, 128, shape, device="cuda", generator=g)
            t = t.to(dtype) if dtype == torch.int8 else (t / 16).to(dtype)
            pools.append(dict(slots=lambda: t, heads=lambda: t.transpose(1, 2), wide=lambda: t[:, :, 2:2 + H],
                              layers=lambda: t[:, 1])[layout]())
        out.append(pools)
    for _ in range(2):
        if dtype != torch.int8:
            out.append(None)
            continue
        if scales == "block":
            out.append([torch.rand(NB, H, device="cuda", generator=g) for _ in range(layers)])
        elif scales == "token32":
            out.append([torch.rand(NB, BS, H, device="cuda", generator=g) for _ in range(layers)])
        else:
            out.append([torch.rand(NB, H, BS, device="cuda", generator=g).half().transpose(1, 2) for _ in range(layers)])
    return out


def host(caches):
    return [None if c is None else [t.float().cpu().numpy().copy() for t in c] for c in caches]


def moved(before, copies):
    """The list model's pools after the copies; per-block scales go whole."""
    for c in before:
        for a in c or []:
            copy_pages(a if a.ndim != 2 else a[:, None], [(s, d, n if a.ndim != 2 else 1) for s, d, n in copies])
    return before


def same(caches, want):
    for c, w in zip(host(caches), want):
        for a, b in zip(c or [], w or []):
            assert np.array_equal(a, b)


SHAPES = [  # blocks, slots, heads, d, type, layers, layout, scales
    (9, 16, 8, 128, torch.float16, 1, "slots", None), (9, 16, 3, 64, torch.bfloat16, 2, "heads", None),
    (40, 1, 1, 64, torch.int8, 3, "slots", "token16"), (12, 32, 5, 64, torch.int8, 2, "heads", "token32"),
    (12, 8, 4, 128, torch.int8, 1, "wide", "block"), (10, 64, 2, 128, torch.float32, 2, "wide", None),
    (11, 16, 2, 64, torch.float16, 70, "slots", None), (7, 256, 8, 128, torch.bfloat16, 1, "layers", None),
    (30, 2, 7, 64, torch.float32, 1, "heads", None)]


@pytest.mark.parametrize("NB,BS,H,D,dtype,layers,layout,scales", SHAPES)
@pytest.mark.parametrize("ragged", [False, True])
def test_copies(ops, NB, BS, H, D, dtype, layers, layout, scales, ragged):
    r = np.random.default_rng(NB + BS)
    caches = make_caches(NB, BS, H, D, dtype, layers, layout, scales or "token16")
    want = host(caches)
    n = NB // 2
    ids = r.permutation(NB)[:2 * n]
    slots = r.integers(0, BS + 1, n) if ragged else np.full(n, BS)
    st = _i32([0])
    ops.copy_blocks(caches[0], caches[1], _i32(ids[:n]), _i32(ids[n:]), caches[2], caches[3],
                    num_slots=_i32(slots) if ragged else None, status=st)
    same(caches, moved(want, [(s, d, k) for s, d, k in zip(ids[:n], ids[n:], slots) if k]))
    assert st.item() == 0


def test_one_source_to_many_and_no_pairs(ops):
    caches = make_caches(20, 16, 2, 64, torch.float16)
    want = host(caches)
    ops.copy_blocks(caches[0][0], caches[1][0], _i32([3] * 6 + [4]), _i32([5, 6, 7, 8, 9, 10, 4]))  # 4 -> 4: nothing
    same(caches, moved(want, [(3, d, 16) for d in range(5, 11)]))
    ops.copy_blocks(caches[0][0], caches[1][0], _i32([]), _i32([]))
    same(caches, want)


@pytest.mark.parametrize("extra", [0, 700])
def test_bad_ids_and_overlaps_are_skipped(ops, extra):
    """With few pairs (a pair a CTA) and many (a CTA checks many): the same rules."""
    NB = 1500
    caches = make_caches(NB, 2, 1, 64, torch.float16)
    want = host(caches)
    src = [0, 1, -1, 2, NB, 3, 4, 5, 6, 10, 12, 14]
    dst = [20, NB, 21, -5, 22, 23, 23, 6, 24, 11, 10, 14]
    slot = [2, 2, 2, 2, 2, 2, 2, 2, 2, 3, 2, 2]
    # 3 -> 23 is first, 4 -> 23 skipped; 5 -> 6 skipped since 6 is read; 10 -> 11 has bad slots and takes no part
    done = [(0, 20, 2), (3, 23, 2), (6, 24, 2), (12, 10, 2)]
    src += list(range(50, 50 + extra))
    dst += list(range(50 + extra, 50 + 2 * extra))
    slot += [1] * extra
    done += [(50 + i, 50 + extra + i, 1) for i in range(extra)]
    st = _i32([0])
    ops.copy_blocks(caches[0], caches[1], _i32(src), _i32(dst), num_slots=_i32(slot), status=st)
    same(caches, moved(want, done))
    assert st.item() == 1 | 2 | 64
    # the same targets over and over: the first wins
    caches = make_caches(NB, 2, 1, 64, torch.float16, seed=1)
    want = host(caches)
    n = 200 + extra
    ops.copy_blocks(caches[0], caches[1], _i32(np.arange(n)), _i32(1000 + np.arange(n) % 7), status=st)
    same(caches, moved(want, [(i, 1000 + i, 2) for i in range(7)]))


def test_copies_past_two_to_the_31(ops):
    """Pages whose byte and element offsets pass 2^31."""
    NB, BS, H, D = 33000, 128, 8, 64
    k, v = (torch.zeros(NB, BS, H, D, dtype=torch.int8, device="cuda") for _ in range(2))
    ks, vs = (torch.zeros(NB, BS, H, dtype=torch.float16, device="cuda") for _ in range(2))
    for t in (k, v, ks, vs):
        t[NB - 1] = 7
        t[1] = 3
    assert k.numel() > 2**31
    ops.copy_blocks(k, v, _i32([NB - 1, 1]), _i32([5, NB - 2]), ks, vs)
    for t in (k, v, ks, vs):
        assert (t[5] == 7).all() and (t[NB - 2] == 3).all() and (t[NB - 3] == 0).all() and (t[6] == 0).all()


def test_captured_copies_on_another_stream(ops):
    caches = make_caches(30, 16, 2, 64, torch.bfloat16, layers=2)
    src, dst = _i32([1, 2, 3]), _i32([11, 12, 13])
    st = torch.cuda.Stream()
    st.wait_stream(torch.cuda.current_stream())
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=st):
        ops.copy_blocks(caches[0], caches[1], src, dst)
    want = host(caches)
    dst.copy_(_i32([21, 22, 23]))
    torch.cuda.synchronize()
    with torch.cuda.stream(st):
        g.replay()
    torch.cuda.synchronize()
    same(caches, moved(want, [(1, 21, 16), (2, 22, 16), (3, 23, 16)]))


def test_copy_refusals_on_the_gpu(ops):
    caches = make_caches(6, 16, 2, 64, torch.float16, layers=2)
    k, v = caches[:2]
    i = _i32([1])
    for a in (([k[0], k[1][:4]], v, i, i), (k, [v[0], v[1].half()[..., :32]], i, i), (k[0].cpu(), v[0], i, i),
              (k[0], v[0].transpose(1, 3), i, i)):
        with pytest.raises((ValueError, RuntimeError)):
            ops.copy_blocks(*a)
    with pytest.raises(ValueError):
        ops.copy_blocks(k[0], v[0], i.cpu(), i)
    with pytest.raises(ValueError):
        ops.copy_blocks(k[0], v[0], i, i, status=torch.zeros(1, device="cuda"))
    with pytest.raises(ValueError):
        ops.copy_blocks(k[0].to(torch.int8), v[0].to(torch.int8), i, i)


# ---- compaction -------------------------------------------------------------------
def pool_arrays(ops, model, cols):
    """A model's state as device arrays; stale entries are filled with what must not be read."""
    table = np.full((len(model.rows), cols), -7)
    count = np.full(len(model.rows), -1)
    for i, r in enumerate(model.rows):
        if r is not None:
            table[i, :len(r)], count[i] = r, len(r)
    stack = np.full(model.NB, -9)
    stack[:len(model.stack)] = model.stack
    return ops.PoolState(_i32(stack), _i32([len(model.stack)]), _i32(table), _i32(count), _i32(model.ref),
                         torch.zeros(ops.pool_scratch_words(model.NB), dtype=torch.int32, device="cuda"))


def pool_equals(pool, model):
    top = pool.free_top.item()
    assert pool.free_stack[:top].tolist() == model.stack
    count, table = pool.count.tolist(), pool.table.cpu().numpy()
    assert [None if c < 0 else table[i, :c].tolist() for i, c in enumerate(count)] == model.rows
    assert pool.ref_count[:model.NB].tolist() == model.ref


def random_model(seed, NB, BS=16, seqs=20, cols=12, share=True):
    r = np.random.default_rng(seed)
    m = SharedPool(NB, seqs, cols, BS)
    for _ in range(80):
        s, what = int(r.integers(seqs)), r.random()
        if m.rows[s] is None and what < 0.5:
            m.allocate(s, int(r.integers(0, cols)))
        elif m.rows[s] is None and share:
            p = int(r.integers(seqs))
            if m.rows[p] is not None:
                m.fork(s, int(r.integers(0, BS * len(m.rows[p]) + 1)), p)
        elif what < 0.4:
            m.release(s)
    return m


@pytest.mark.parametrize("seed,NB", [(0, 40), (1, 100), (2, 5000), (3, 131), (4, 1), (5, 64), (6, 40000), (7, 65536), (8, 70001)])
@pytest.mark.parametrize("dtype,layers,layout", [(torch.int8, 2, "slots"), (torch.float16, 1, "heads"), (torch.float32, 66, "slots")])
def test_compaction(ops, seed, NB, dtype, layers, layout):
    if NB > 1000 and layers > 2:
        NB //= 20
    m = random_model(seed, NB)
    pool = pool_arrays(ops, m, 12)
    H, D, BS = (1, 64, 2) if NB > 1000 or layers > 2 else (3, 64, 16)
    caches = make_caches(NB, BS, H, D, dtype, layers, layout)
    want = host(caches)
    st = _i32([0])
    live = ops.compact_blocks(pool, *caches, status=st)
    n, moves = m.compact()
    m.check()
    assert live.tolist() == [n] and st.item() == 0
    pool_equals(pool, m)
    same(caches, moved(want, [(s, d, BS) for s, d in moves]))
    ops.compact_blocks(pool, *caches)  # nothing is left to do
    pool_equals(pool, m)
    same(caches, want)


def test_compaction_shrinks_and_refuses(ops):
    m = random_model(11, 80)
    used = sum(x > 0 for x in m.ref)
    pool = pool_arrays(ops, m, 12)
    caches = make_caches(80, 16, 1, 64, torch.float16)
    want = host(caches)
    before = [t.clone() for t in pool]
    st = _i32([0])
    live = ops.compact_blocks(pool, *caches, num_blocks=used - 1, status=st)  # too few: nothing changes
    assert st.item() == 128 and live.tolist() == [used]
    assert all(torch.equal(a, b) for a, b in zip(pool[:5], before[:5]))
    same(caches, want)
    ops.compact_blocks(pool, *caches, num_blocks=used + 2)
    n, moves = m.compact(used + 2)
    pool_equals(pool, m)
    same(caches, moved(want, [(s, d, 16) for s, d in moves]))
    with pytest.raises(ValueError):
        ops.compact_blocks(pool, *caches, num_blocks=81)
    with pytest.raises(ValueError):
        ops.compact_blocks(pool, *caches, num_blocks=-1)


def test_compaction_of_contradicting_arrays(ops):
    """A row that names an uncounted or impossible block keeps that entry and is reported; nothing else suffers."""
    m = random_model(12, 100)
    pool = pool_arrays(ops, m, 12)
    caches = make_caches(100, 2, 1, 64, torch.float16)
    free_high = max(b for b in range(100) if m.ref[b] == 0)
    row = next(i for i, r in enumerate(m.rows) if r is None)
    pool.count[row] = 2
    pool.table[row, :2] = _i32([free_high, 100])
    st = _i32([0])
    ops.compact_blocks(pool, *caches, status=st)
    live, _ = m.compact()
    assert st.item() == 1 | (128 if free_high >= live else 0)
    assert pool.table[row, :2].tolist() == [free_high, 100]
    pool.count[row] = -1
    pool_equals(pool, m)


def test_compiled_copies():
    """Through torch.compile, which traces the op on fake tensors."""
    from pie_b200 import _torch_ext

    op = _torch_ext.ops().copy_blocks
    k, v, _, _ = make_caches(9, 16, 2, 64, torch.float16, 2)
    want = moved(host((k, v)), [(1, 4, 16), (2, 7, 16)])
    src, dst = _i32([1, 2]), _i32([4, 7])

    def step(k0, k1, v0, v1, src, dst):
        op([k0, k1], [v0, v1], [], [], src, dst, None, None)
        return src

    got = torch.compile(step, fullgraph=True)(*k, *v, src, dst)
    assert got.tolist() == [1, 2]
    same((k, v), want)
