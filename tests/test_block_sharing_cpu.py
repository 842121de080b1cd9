"""Block sharing on the CPU: the host ledger against the list model, and what the entry points refuse."""
import ctypes
import os
import random
import subprocess

import numpy as np
import pytest
import torch

from conftest import ROOT
from oracle import beam_search as obs
from oracle.block_sharing import SUCCESS, SharedPool


def _apply(model, ops):
    for kind, slot, n, *parent in ops:
        st = (model.allocate(slot, n) if kind == 0 else model.release(slot) if kind == 1
              else model.fork(slot, n, parent[0])[0])
        assert st == SUCCESS


@pytest.mark.parametrize("seed", range(12))
def test_ledger_counts_like_the_list_model(seed):
    """Random allocations, forks and releases: the ledger's free count and decisions are the model's."""
    from pie_b200.block_pool import AllocStatus, BlockLedger

    r = random.Random(seed)
    NB, BS, seqs, cols = 60, 4, 12, 9
    led, model = BlockLedger(NB, seqs, cols), SharedPool(NB, seqs, cols, BS)
    nxt = 0
    for _ in range(400):
        live = list(led.blocks)
        what = r.random()
        if what < 0.4 and len(live) < seqs:
            led.allocate(nxt, r.randint(0, 4))
            nxt += 1
        elif what < 0.55 and live:
            s = r.choice(live)
            led.allocate(s, r.randint(0, min(2, cols - led.blocks[s])))
        elif what < 0.8 and live and len(live) < seqs:
            s = r.choice(live)
            st, _ = led.fork(s, nxt, r.randint(0, led.blocks[s] * BS), BS)
            assert st in (AllocStatus.SUCCESS, AllocStatus.INSUFFICIENT_SPACE)
            nxt += 1
        elif live:
            assert led.release(r.choice(live)) is AllocStatus.SUCCESS
        _apply(model, led.take_ops())
        model.check()
        assert led.free == len(model.stack)
        assert {led.slot[s]: n for s, n in led.blocks.items()} == {i: len(x) for i, x in enumerate(model.rows) if x is not None}


@pytest.mark.parametrize("seed", range(12))
def test_ledger_never_counts_more_free_blocks_than_beams_leave(seed):
    """Beams whose parents the host does not know: the ledger's free count stays at or below the model's, and meets it again."""
    from pie_b200.block_pool import AllocStatus, BlockLedger

    r = random.Random(100 + seed)
    NB, BS, seqs, cols = 90, 4, 14, 12
    led, model = BlockLedger(NB, seqs, cols), SharedPool(NB, seqs, cols, BS)
    groups, nxt = {}, 0  # first beam -> [slots, tokens]
    plain = {}

    def follow():
        _apply(model, led.take_ops())
        model.check()

    for _ in range(250):
        what = r.random()
        if what < 0.2 and len(led.blocks) < seqs:
            n = r.randint(1, 12)
            if led.allocate(nxt, -(-n // BS))[0] is AllocStatus.SUCCESS:
                plain[nxt] = n
            nxt += 1
        elif what < 0.3 and plain and len(led.blocks) < seqs:
            s = r.choice(list(plain))
            if led.fork(s, nxt, plain[s], BS)[0] is AllocStatus.SUCCESS:
                plain[nxt] = plain[s]
            nxt += 1
        elif what < 0.4 and plain and len(led.blocks) + 3 <= seqs:
            s = r.choice(list(plain))
            ids = [(s, k) for k in (1, 2, 3)]
            if led.fork_beams(s, ids, plain[s], BS) is AllocStatus.SUCCESS:
                groups[s] = [[led.slot[b] for b in (s, *ids)], plain.pop(s)]
                with pytest.raises(ValueError):
                    led.release(ids[0])
                with pytest.raises(ValueError):
                    led.fork(s, "x", 1, BS)
        elif what < 0.85 and groups:
            s = r.choice(list(groups))
            slots, n = groups[s]
            if n % BS == 0:
                if -(-(n + 1) // BS) > cols or led.allocate_beams(s, 1) is not AllocStatus.SUCCESS:
                    continue
                follow()
            new, _, freed = model.reorder(slots, [r.randrange(4) for _ in range(4)], n + 1)
            model.push(freed)
            groups[s] = [new, n + 1]
        elif what < 0.92 and groups:
            s = r.choice(list(groups))
            del groups[s]
            assert led.release_beams(s) is AllocStatus.SUCCESS
        elif plain:
            s = r.choice(list(plain))
            del plain[s]
            led.release(s)
        follow()
        assert led.free <= len(model.stack)
        if not groups:
            assert led.free == len(model.stack)


def test_ledger_refusals():
    from pie_b200.block_pool import AllocStatus, BlockLedger

    led = BlockLedger(10, 3, 8)
    led.allocate(0, 3)
    assert led.fork(5, 1, 4, 4)[0] is AllocStatus.FAILURE  # no such parent
    assert led.fork(0, 0, 4, 4)[0] is AllocStatus.FAILURE  # the child exists
    with pytest.raises(ValueError):
        led.fork(0, 1, 13, 4)                              # more tokens than blocks
    with pytest.raises(ValueError):
        led.fork(0, 1, -1, 4)
    with pytest.raises(ValueError):
        led.fork_beams(0, [1, 1], 12, 4)
    with pytest.raises(ValueError):
        led.fork_beams(0, [1], 8, 4)                       # an unused block
    with pytest.raises(RuntimeError):
        led.fork_beams(0, [1, 2, 3], 12, 4)                # three rows in all
    assert led.release_beams(0) is AllocStatus.FAILURE
    led.allocate(1, 7)
    assert led.fork(0, 2, 11, 4)[0] is AllocStatus.INSUFFICIENT_SPACE
    assert led.fork_beams(0, [2], 11, 4) is AllocStatus.INSUFFICIENT_SPACE
    assert led.fork_beams(0, [2], 12, 4) is AllocStatus.SUCCESS
    led.dissolve_beams(0)
    assert led.blocks == {0: 3, 1: 7} and led.free == 0
    led.release(0)
    led.release(1)
    assert led.free == 10


def test_struct_layouts_match_header(tmp_path):
    from pie_b200 import _lib

    structs = {"pa_block_share_t": _lib.PaBlockShare, "pa_beam_select_t": _lib.PaBeamSelect}
    lines = ['#include <stdio.h>', '#include <stddef.h>', '#include "paged_attn_b200.h"', "int main(void) {"]
    for cname, py in structs.items():
        lines.append(f'printf("{cname} sizeof %zu\\n", sizeof({cname}));')
        lines += [f'printf("{cname} {f} %zu\\n", offsetof({cname}, {f}));' for f, _ in py._fields_]
    lines.append("return 0; }")
    (tmp_path / "layout.c").write_text("\n".join(lines))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(tmp_path / "layout.c"), "-o", str(exe)], check=True)
    for ln in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.splitlines():
        cname, field, val = ln.split()
        py = structs[cname]
        assert int(val) == (ctypes.sizeof(py) if field == "sizeof" else getattr(py, field).offset), ln


def _cache(n=1, dtype=0, blocks=8):
    from pie_b200 import _lib

    c = (_lib.PaKvCache * n)()
    for kv in c:
        kv.k = kv.v = 1 << 20
        kv.dtype = dtype
        kv.num_blocks, kv.block_size, kv.num_kv_heads, kv.head_dim = blocks, 16, 2, 64
        kv.k_stride_block = kv.v_stride_block = 16 * 128
        kv.k_stride_slot = kv.v_stride_slot = 128
        kv.k_stride_head = kv.v_stride_head = 64
    return c


def test_copy_blocks_validates_without_gpu():
    from pie_b200 import _lib

    lib, p = _lib.load(), 1 << 21
    c = _cache(2)
    assert lib.kv_copy_blocks(c, 2, p, p, None, 0, None, None) == _lib.PA_OK  # nothing to do
    assert lib.kv_copy_blocks(None, 1, p, p, None, 1, None, None) == _lib.PA_ERR_INVALID
    assert lib.kv_copy_blocks(c, 0, p, p, None, 1, None, None) == _lib.PA_ERR_INVALID
    assert lib.kv_copy_blocks(c, 2, p, p, None, -1, None, None) == _lib.PA_ERR_INVALID
    assert lib.kv_copy_blocks(c, 2, None, p, None, 1, None, None) == _lib.PA_ERR_INVALID
    for field in ("k_stride_slot", "num_blocks", "num_kv_heads", "dtype"):
        c = _cache(2)
        setattr(c[1], field, 16 * getattr(c[1], field) + (1 if field == "dtype" else 0))
        assert lib.kv_copy_blocks(c, 2, p, p, None, 1, None, None) == _lib.PA_ERR_INVALID, field
        assert b"layer 1" in lib.paged_attn_error_string()
    c = _cache(1, dtype=_lib.PA_DTYPE_I8)  # no scales
    assert lib.kv_copy_blocks(c, 1, p, p, None, 1, None, None) == _lib.PA_ERR_INVALID


def test_shared_pool_calls_validate_without_gpu():
    from pie_b200 import _lib
    from pie_b200.block_pool import PaBlockPool
    from pie_b200.ops import pool_scratch_words

    lib, p = _lib.load(), 1 << 21
    d = PaBlockPool(p, p, p, p, 8, 16, 8, 8, 0)
    words = lib.block_pool_scratch_words(16)
    assert words == pool_scratch_words(16)
    s, B = _lib.PaBlockShare(p, p, words), ctypes.byref
    assert lib.block_pool_init_shared(B(d), B(_lib.PaBlockShare(None, p, words)), None) == _lib.PA_ERR_INVALID
    assert lib.block_pool_init_shared(B(d), B(_lib.PaBlockShare(p, p, words - 1)), None) == _lib.PA_ERR_WORKSPACE
    assert lib.block_pool_apply_shared(B(d), B(s), None, 1, 16, None, None, None, None, None) == _lib.PA_ERR_INVALID
    assert lib.block_pool_apply_shared(B(d), B(s), p, 1, 0, None, None, None, None, None) == _lib.PA_ERR_INVALID
    assert lib.block_pool_apply_shared(B(d), B(s), p, 1, 16, None, p, None, None, None) == _lib.PA_ERR_INVALID
    assert lib.block_pool_apply_shared(B(d), B(s), p, 0, 16, None, None, None, None, None) == _lib.PA_OK
    c = _cache(1, blocks=16)

    def reorder(groups=1, beams=4, out=p + 64, caches=c, slots=p):
        return lib.block_pool_reorder(B(d), B(s), slots, p, p, groups, beams, out, caches, 1, None, None)

    assert reorder(groups=0) == _lib.PA_OK
    assert reorder(groups=-1) == _lib.PA_ERR_INVALID
    assert reorder(beams=0) == reorder(beams=33) == _lib.PA_ERR_UNSUPPORTED
    assert reorder(out=p) == reorder(out=None) == reorder(slots=None) == _lib.PA_ERR_INVALID
    assert reorder(caches=_cache(1, blocks=15)) == _lib.PA_ERR_INVALID
    for after in (-1, 17):
        assert lib.block_pool_compact(B(d), B(s), after, None, c, 1, None, None) == _lib.PA_ERR_INVALID
    assert lib.block_pool_compact(B(d), B(s), 16, None, None, 1, None, None) == _lib.PA_ERR_INVALID


@pytest.mark.parametrize("change,code", [
    (dict(dtype=2), -1), (dict(dtype=9), -1), (dict(vocab=0), -1), (dict(num_seqs=-1), -1), (dict(num_beams=0), -2),
    (dict(num_beams=33), -2), (dict(num_out=0), -2), (dict(num_out=33), -2), (dict(vocab=7), -1), (dict(eos_id=100), -1),
    (dict(eos_id=-1), -1), (dict(stride_seq=-4), -1), (dict(vocab=2**31 - 1), -2),
])
def test_beam_select_validates_without_gpu(change, code):
    from pie_b200 import _lib

    lib, n = _lib.load(), ctypes.c_size_t(0)
    args = dict(logits=1 << 20, scores=1 << 20, finished=1 << 20, stride_seq=400, stride_beam=100, dtype=3, num_seqs=2,
                num_beams=4, vocab=100, eos_id=3, num_out=32)
    a = _lib.PaBeamSelect(**args)
    assert lib.beam_select_workspace_size(a, ctypes.byref(n)) == 0 and n.value >= 2 * 4 * (32 * 8 + 8)
    assert lib.beam_select(a, None, 0, None) == _lib.PA_ERR_INVALID  # no outputs
    a.out_scores = a.out_tokens = a.out_parents = 1 << 22
    assert lib.beam_select(a, None, 0, None) == _lib.PA_ERR_WORKSPACE
    for k, v in change.items():
        setattr(a, k, v)
    assert lib.beam_select(a, 1 << 23, 1 << 40, None) == code
    assert lib.paged_attn_error_string()


def test_front_end_refusals_without_gpu():
    from pie_b200 import ops

    x, s = torch.zeros(2, 3, 50), torch.zeros(2, 3)
    for bad in (dict(logits=x[0]), dict(logits=x.double()), dict(num_out=0), dict(num_out=151),
                dict(finished=torch.zeros(2, 3, dtype=torch.bool)), dict(logits=x[..., :0]),
                dict(finished=torch.zeros(2, 3, dtype=torch.bool), eos_id=50)):
        a = dict(logits=x, beam_scores=s, num_out=4, finished=None, eos_id=None) | bad
        with pytest.raises(ValueError):
            ops.beam_select(a["logits"], a["beam_scores"], a["num_out"], finished=a["finished"], eos_id=a["eos_id"])
    K = torch.zeros(5, 16, 2, 64, dtype=torch.float16)
    i = torch.zeros(3, dtype=torch.int32)
    with pytest.raises(ValueError):
        ops.copy_blocks([], [], i, i)
    with pytest.raises(ValueError):
        ops.copy_blocks(K, K, i, i[:2])
    with pytest.raises(ValueError):
        ops.copy_blocks(K, K, i, i, num_slots=i[:1])
    with pytest.raises(ValueError):
        ops.layer_descs([K, K], [K])
    with pytest.raises(ValueError):
        ops.layer_descs(K.to(torch.int8), K.to(torch.int8))
    with pytest.raises(ValueError):
        ops.compact_blocks(None, K, K, num_blocks=-1)
    for name in ("copy_blocks", "reorder_beams", "compact_blocks", "beam_select"):
        with pytest.raises(Exception):  # no CPU path
            if name == "beam_select":
                ops.beam_select(x, s, 4)
            elif name == "copy_blocks":
                ops.copy_blocks(K, K, i, i)
            else:
                pool = ops.PoolState(*[torch.zeros(5, dtype=torch.int32)] * 2, torch.zeros(4, 5, dtype=torch.int32),
                                     torch.zeros(4, dtype=torch.int32), torch.zeros(5, dtype=torch.int32),
                                     torch.zeros(ops.pool_scratch_words(5), dtype=torch.int32))
                if name == "reorder_beams":
                    ops.reorder_beams(pool, i[None], i[None], i[:1], K, K)
                else:
                    ops.compact_blocks(pool, K, K)


def test_meta_kernels_give_the_shapes():
    from pie_b200 import _torch_ext

    ops = _torch_ext.ops()
    m = dict(device="meta")
    x = torch.empty(3, 4, 100, dtype=torch.bfloat16, **m)
    s, t, p = ops.beam_select(x, torch.empty(3, 4, **m), 7, None, -1)
    assert s.shape == t.shape == p.shape == (3, 7) and s.dtype == torch.float32 and t.dtype == p.dtype == torch.int32


def test_selection_oracle_on_known_values():
    """Two beams of three tokens, by hand: log-probabilities of [0, ln 2, 0] are ln 1/4, ln 1/2, ln 1/4."""
    x = np.array([[[0.0, np.log(2.0), 0.0], [0.0, 0.0, -np.inf]]])
    s, t, p = obs.select(x, np.array([[0.0, np.log(0.5)]]), 5)
    assert t.tolist() == [[1, 0, 2, 0, 1]] and p.tolist() == [[0, 0, 0, 1, 1]]
    np.testing.assert_allclose(s, [np.log([0.5, 0.25, 0.25, 0.25, 0.25])])


def _host_manager(ledger):
    """A manager without its device half: what it refuses before it touches the device."""
    from pie_b200.block_pool import DeviceBlockManager

    dm = DeviceBlockManager.__new__(DeviceBlockManager)
    dm.ledger, dm.block_size, dm.num_blocks, dm._copies = ledger, 4, ledger.num_blocks, set()
    return dm


def test_beams_have_no_rows_here_once_the_device_has_permuted_them():
    """Rows [0, 1, 2] and parents [1, 1, 0] give the beams the rows [1, 2, 0]: a beam's id would name another's row."""
    from pie_b200.block_pool import BlockLedger

    led = BlockLedger(40, 8, 6)
    model = SharedPool(40, 8, 6, 4)
    for s in (7, 8, 9):
        led.allocate(s, 2)
    assert led.fork_beams(7, ["a", (7, 2)], 8, 4).value == 0 and led.fork_beams(8, ["c"], 8, 4).value == 0
    _apply(model, led.take_ops())
    before = [led.row(s) for s in (7, "a", (7, 2))]
    assert model.reorder(before, [1, 1, 0], 8)[0] == [before[1], before[2], before[0]]
    dm = _host_manager(led)
    assert dm.slot_of("a") == before[1]  # as fork_beams made them
    led.beams_moved()
    for s in (7, "a", (7, 2), 8, "c"):
        with pytest.raises(ValueError, match="beam of"):
            dm.slot_of(s)
        with pytest.raises(ValueError, match="beam of"):
            dm.step_inputs([9, s], [1, 1], [8, 8])
        with pytest.raises(ValueError, match="beam of"):
            led.none_is_a_beam([9, s])
    with pytest.raises(ValueError, match="beam of"):
        dm.beam_slots([7])
    with pytest.raises(ValueError, match="beam of"):
        dm.block_table
    assert dm.slot_of(9) == led.slot[9]
    led.none_is_a_beam([9])
    led.release_beams(7)
    led.release_beams(8)
    led.allocate(7, 1)  # the id is an ordinary one again
    assert dm.slot_of(7) == led.slot[7] and not led.moved
    led.none_is_a_beam([7, 9])


def test_the_decode_step_takes_no_beam():
    from pie_b200.block_pool import BlockLedger
    from pie_b200.decode_step import DecodeStepGraph

    led = BlockLedger(40, 8, 6)
    led.allocate(0, 2)
    led.allocate(1, 2)
    led.fork_beams(0, [(0, 1)], 8, 4)
    graph = DecodeStepGraph.__new__(DecodeStepGraph)
    graph.pool, graph.S = _host_manager(led), 4
    for ids in ([0], [(0, 1)], [1, 0], [np.int64(0)]):
        with pytest.raises(ValueError, match="beam of"):
            graph.step(ids, [9] * len(ids), None, None, None)
    assert len(led.take_ops()) == 3  # nothing was queued


def test_every_op_has_a_meta_kernel():
    """On meta tensors: ops that return nothing leave their arguments alone, the others give their outputs' shapes."""
    from pie_b200 import _torch_ext

    ops = _torch_ext.ops()

    def t(*shape, dtype=torch.int32):
        return torch.empty(*shape, dtype=dtype, device="meta")

    half = torch.float16
    kv = [t(10, 16, 2, 64, dtype=half)]
    pool = (t(10), t(1), t(6, 5), t(6), t(10), t(60))
    assert ops.copy_blocks(kv, kv, [], [], t(3), t(3), None, None) is None
    assert ops.copy_blocks(kv * 2, kv * 2, [], [], t(3), t(3), t(3), t(1)) is None
    assert ops.write_kv(t(4, 2, 64, dtype=half), t(4, 2, 64, dtype=half), t(2, 5), t(4), t(4), kv[0], kv[0], None, None,
                        None) is None
    assert ops.project_write_kv(t(4, 256, dtype=half), t(256, 256, dtype=half), None, t(2, 5), t(4), t(4), kv[0], kv[0],
                                None, None, None) is None
    q, lse = t(2, 4, 1, 64, dtype=half), t(2, 4, 1, dtype=half)
    assert ops.paged_attention_out(q, kv[0], kv[0], t(2), t(2, 5), t(2), t(2), None, None, False, 0.0, 0, None, q, lse) is None
    q, lse = t(7, 4, 64, dtype=half), t(7, 4, dtype=half)
    assert ops.paged_attention_varlen_out(q, t(3), t(2), 5, kv[0], kv[0], t(2, 5), t(2), t(2), None, None, False, 0.0, None,
                                          q, lse) is None
    assert ops.reorder_beams(*pool, t(2, 3), t(2, 3), t(2), kv, kv, [], [], None).shape == (2, 3)
    assert ops.compact_blocks(*pool, -1, kv, kv, [], [], None).shape == (1,)


def test_a_reordering_inside_a_shared_block_would_write_others_tokens():
    """Tokens rolled back into a block that an earlier reordering shared: on the model, two copies have one target."""
    m = SharedPool(20, 4, 4, 4)
    m.allocate(0, 1)
    for s in (1, 2):
        m.fork(s, 4, 0)
    for s in range(3):
        m.allocate(s, 1)
    assert m.may_reorder([0, 1, 2], 6)
    m.push(m.reorder([0, 1, 2], [1, 1, 1], 8)[2])  # the second block is full: all three hold beam 1's
    assert m.may_reorder([0, 1, 2], 8) and not m.may_reorder([0, 1, 2], 6)
    copies = m.reorder([0, 1, 2], [0, 0, 0], 6)[1]
    assert len({d for _, d, _ in copies}) == 1 < len(copies)


def test_beams_do_not_start_inside_a_shared_block():
    """A fork of a whole block, taken as holding fewer tokens: beam 0 would append into the block of its parent."""
    from pie_b200.block_pool import AllocStatus, BlockLedger

    led = BlockLedger(20, 8, 4)
    led.allocate(0, 2)
    led.fork(0, 1, 8, 4)
    for tokens in (5, 7):
        with pytest.raises(ValueError, match="another sequence holds"):
            led.fork_beams(1, ["a"], tokens, 4)
    with pytest.raises(ValueError, match="another sequence holds"):
        led.fork_beams(0, ["a"], 6, 4)  # the parent neither
    assert led.shared_columns(0) == led.shared_columns(1) == 2 and not led.beams and len(led.take_ops()) == 2
    led.fork(1, 2, 6, 4)                # a copy of the last block is its own
    assert led.shared_columns(2) == 1 and led.fork_beams(2, ["a"], 6, 4) is AllocStatus.SUCCESS
    assert led.fork_beams(1, ["b"], 8, 4) is AllocStatus.SUCCESS  # whole blocks: the next token opens a new one
    led.release_beams(1)
    led.release_beams(2)
    assert led.shared_columns(0) == 0 and led.fork_beams(0, ["a"], 6, 4) is AllocStatus.SUCCESS  # alone again


@pytest.mark.parametrize("dtype,part", [(3, 2**17), (0, 2**18), (1, 2**18)])
@pytest.mark.parametrize("beams,out", [(32, 32), (4, 8), (1, 1), (8, 16), (3, 7)])
def test_parts_are_short_enough_for_the_sums(dtype, part, beams, out):
    """A thread's fp32 sum takes one addition, and perhaps one rescaling, for each unit of its part: 32 at most."""
    from pie_b200 import _lib

    lib, n = _lib.load(), ctypes.c_size_t(0)
    most = min(2**30, 8192 // (beams * out) * part)
    for seqs in (1, 700):
        for vocab in (out, 50257, 131072, 262144, part + 1, 5 * part, most - 1, most):
            if vocab > most:
                continue
            a = _lib.PaBeamSelect(dtype=dtype, num_seqs=seqs, num_beams=beams, vocab=vocab, num_out=out, eos_id=-1)
            assert lib.beam_select_workspace_size(a, ctypes.byref(n)) == _lib.PA_OK
            parts, rest = divmod(n.value, seqs * beams * (8 * out + 8))
            assert rest == 0 and -(-vocab // part) <= parts <= 8192 // (beams * out), (vocab, parts)
    if most < 2**30:
        for vocab in (most + 1, 2**30):
            a = _lib.PaBeamSelect(dtype=dtype, num_seqs=1, num_beams=beams, vocab=vocab, num_out=out, eos_id=-1)
            assert lib.beam_select_workspace_size(a, ctypes.byref(n)) == _lib.PA_ERR_UNSUPPORTED
            assert str(most).encode() in lib.paged_attn_error_string()


def test_only_batches_that_meet_shared_blocks_are_counted():
    """A scheduler that shares nothing keeps the plain pool's launch: the ledger says which batches need the counts."""
    from pie_b200.block_pool import BlockLedger

    led = BlockLedger(60, 12, 6)

    def counted():
        flag, _ = led.counted, led.take_ops()
        return flag

    for s in range(4):
        led.allocate(s, 2)
    led.release(3)
    assert not counted()
    led.fork(0, 10, 8, 4)
    assert counted()
    led.allocate(10, 1)           # a block of its own
    led.release(2)
    assert not counted()
    led.release(0)                # the fork still holds its blocks
    assert counted()
    led.release(10)               # nobody else does any more
    assert not counted()
    led.fork_beams(1, ["b"], 8, 4)
    assert counted()
    led.allocate_beams(1, 1)
    assert not counted()
    led.release_beams(1)
    assert counted()
    led.allocate(1, 2)
    led.fork_beams(1, ["b"], 8, 4)
    led.take_ops()
    led.dissolve_beams(1)
    assert counted()
    led.release(1)
    assert not counted() and led.free == 60


def test_sole_batches_validate_without_gpu():
    from pie_b200 import _lib
    from pie_b200.block_pool import PaBlockPool

    lib, p, B = _lib.load(), 1 << 21, ctypes.byref
    d = PaBlockPool(p, p, p, p, 8, 16, 8, 8, 0)
    s = _lib.PaBlockShare(p, p, lib.block_pool_scratch_words(16))
    assert lib.block_pool_apply_sole(B(d), B(_lib.PaBlockShare(None, p, 999)), p, 1, None, None) == _lib.PA_ERR_INVALID
    assert lib.block_pool_apply_sole(B(d), B(s), None, 1, None, None) == _lib.PA_ERR_INVALID
    assert lib.block_pool_apply_sole(B(d), B(s), p, -1, None, None) == _lib.PA_ERR_INVALID
    assert lib.block_pool_apply_sole(B(d), B(s), p, 0, None, None) == _lib.PA_OK


def _recount(led, model):
    for s in led.beams:
        first, last = led.private_columns(s)
        rows = [model.rows[led.slot[b]] for b in led.beams[s]]
        assert all(len(r) == last for r in rows) and len({tuple(r[:first]) for r in rows}) == 1
        led.count_beams(s, len({b for r in rows for b in r[first:last]}))


def test_ledger_learns_what_reorderings_freed():
    """One search of 4 beams over 512 new tokens that follow one line: 34 blocks in use, 129 counted before."""
    from pie_b200.block_pool import AllocStatus, BlockLedger

    NB, BS = 160, 16
    led, model = BlockLedger(NB, 8, 64), SharedPool(NB, 8, 64, BS)
    led.allocate(0, 1)
    led.fork_beams(0, [1, 2, 3], 16, BS)
    _apply(model, led.take_ops())
    slots = [led.slot[b] for b in led.beams[0]]
    for n in range(16, 16 + 512):
        if n % BS == 0:
            assert led.allocate_beams(0, 1) is AllocStatus.SUCCESS
            _apply(model, led.take_ops())
        slots, _, freed = model.reorder(slots, [0, 0, 0, 0], n + 1)
        model.push(freed)
    assert NB - led.free == 129
    assert led.allocate("other", 60)[0] is AllocStatus.INSUFFICIENT_SPACE
    _recount(led, model)
    assert NB - led.free == NB - len(model.stack) == 33
    assert led.allocate("other", 60)[0] is AllocStatus.SUCCESS
    led.release_beams(0)
    _apply(model, led.take_ops())
    model.check()
    assert led.free == len(model.stack) == NB - 60 and not led.regained


@pytest.mark.parametrize("seed", range(16))
def test_recounted_ledger_is_the_model_and_never_above_it(seed):
    """Searches that start, share prompts, grow, reorder, are recounted and end at any time, beside plain sequences."""
    from pie_b200.block_pool import AllocStatus, BlockLedger

    r = random.Random(500 + seed)
    NB, BS, seqs, cols = 120, 4, 20, 12
    led, model = BlockLedger(NB, seqs, cols), SharedPool(NB, seqs, cols, BS)
    groups, plain, nxt = {}, {}, 0
    for _ in range(400):
        what = r.random()
        if what < 0.15 and len(led.blocks) < seqs:
            n = r.randint(0, 14)
            if led.allocate(nxt, -(-n // BS))[0] is AllocStatus.SUCCESS:
                plain[nxt] = n
            nxt += 1
        elif what < 0.3 and plain and len(led.blocks) < seqs:
            s = r.choice(list(plain))
            n = r.randint(0, plain[s])
            if led.fork(s, nxt, n, BS)[0] is AllocStatus.SUCCESS:
                plain[nxt] = n
            nxt += 1
        elif what < 0.4 and plain:
            s, k = r.choice(list(plain)), r.randint(1, 5)
            if len(led.blocks) + k - 1 <= seqs and (plain[s] % BS == 0 or led.shared_columns(s) <= plain[s] // BS):
                ids = [(s, j) for j in range(1, k)]
                if led.fork_beams(s, ids, plain[s], BS) is AllocStatus.SUCCESS:
                    groups[s] = [[led.slot[b] for b in (s, *ids)], plain.pop(s)]
        elif what < 0.8 and groups:
            s = r.choice(list(groups))
            slots, n = groups[s]
            if n % BS == 0:
                if n // BS >= cols or led.allocate_beams(s, 1) is not AllocStatus.SUCCESS:
                    continue
                _apply(model, led.take_ops())
            new, _, freed = model.reorder(slots, [r.randrange(len(slots)) for _ in slots], n + 1)
            model.push(freed)
            groups[s] = [new, n + 1]
        elif what < 0.85 and groups:
            s = r.choice(list(groups))
            del groups[s]
            led.release_beams(s)
        elif what < 0.92:
            _apply(model, led.take_ops())
            _recount(led, model)
            assert led.free == len(model.stack)
        elif plain:
            s = r.choice(list(plain))
            del plain[s]
            led.release(s)
        _apply(model, led.take_ops())
        model.check()
        assert 0 <= led.free <= len(model.stack)
        assert groups or led.free == len(model.stack)


@pytest.mark.parametrize("shape,layers,why", [
    ((20, 12, 2, 64), None, "power of two"), ((20, 4, 2, 96), None, "head_dim"), ((20, 4, 2, 64), (20, 4, 4, 64), "layer 1"),
    ((20, 4, 2, 64), (20, 4, 2, 128), "layer 1"), ((20, 4, 2, 67), None, "strides")])
def test_caches_that_cannot_be_copied_are_refused_when_attached(shape, layers, why):
    """Not at the flush, which had applied the fork on the device and then could not copy its page."""
    from pie_b200 import _lib
    from pie_b200.block_pool import BlockLedger

    dm = _host_manager(BlockLedger(20, 8, 4))
    dm.block_size, dm.caches, dm._cache_descs = shape[1], None, None
    dm.free_top = torch.zeros(1, dtype=torch.int32)

    def pool(s):
        t = torch.zeros(s, dtype=torch.float16)
        return t[..., :64] if s[-1] == 67 else t

    k = [pool(shape)] + ([pool(layers)] if layers else [])
    with pytest.raises((_lib.PagedAttnError, ValueError), match=why):
        dm.attach_caches(k, [t.clone() if t.is_contiguous() else t for t in k])
    assert dm.caches is None and dm._cache_descs is None
    with pytest.raises(ValueError, match="attach_caches"):
        dm.fork(0, 1, 5)


def test_the_decode_step_writes_no_shared_block():
    """A sequence rolled back below the point at which it was forked: its next token would be its fork's too."""
    from pie_b200.block_pool import BlockLedger
    from pie_b200.decode_step import DecodeStepGraph

    led = BlockLedger(40, 8, 6)
    led.allocate(0, 3)
    led.allocate(1, 1)
    led.fork(0, 5, 9, 4)  # two whole blocks shared, the third copied
    graph = DecodeStepGraph.__new__(DecodeStepGraph)
    graph.pool, graph.S, graph.BS = _host_manager(led), 4, 4
    graph.pool.flush = lambda: (_ for _ in ()).throw(KeyError("the device"))  # what the host lets pass ends here
    graph.graphs, graph.pool.max_blocks_per_seq = (), 6
    for ids, lens in (([0], [8]), ([5], [1]), ([1, 5], [4, 7]), ([1, 0], [3, 5])):
        with pytest.raises(ValueError, match="another sequence holds"):
            graph.step(ids, lens, None, None, None)
    for ids, lens in (([0], [9]), ([5], [10]), ([1], [1]), ([0, 5, 1], [12, 9, 2])):
        with pytest.raises(KeyError, match="the device"):
            graph.step(ids, lens, None, None, None)
    led.release(0)
    with pytest.raises(KeyError, match="the device"):
        graph.step([5], [3], None, None, None)  # alone again


def test_only_the_searches_that_moved_lose_their_rows():
    from pie_b200.block_pool import BlockLedger

    led = BlockLedger(40, 8, 6)
    for s in (0, 1):
        led.allocate(s, 2)
        led.fork_beams(s, [(s, 1)], 8, 4)
    led.beams_moved([0, 77])
    dm = _host_manager(led)
    assert dm.slot_of(1) == led.slot[1] and dm.slot_of((1, 1)) == led.slot[(1, 1)]
    for s in (0, (0, 1)):
        with pytest.raises(ValueError, match="beam of"):
            dm.slot_of(s)
    led.release_beams(0)
    assert not led.moved
