"""CPU: shared prefixes: the ledger's groups, what the entry points refuse, and the descriptor's layout."""
import ctypes
import os
import random
import subprocess

import pytest
import torch

from conftest import ROOT
from oracle.block_sharing import SharedPool
from test_capi_cpu import _descs


@pytest.mark.parametrize("seed", range(10))
def test_groups_share_what_they_say(seed):
    """Random forks and releases: the columns that a group is said to share hold the same blocks in the list model's rows."""
    from pie_b200.block_pool import AllocStatus, BlockLedger

    r = random.Random(seed)
    NB, BS, seqs, cols = 80, 4, 14, 9
    led, model = BlockLedger(NB, seqs, cols), SharedPool(NB, seqs, cols, BS)
    nxt, most = 0, 0
    for step in range(250):
        live = list(led.blocks)
        what = r.random()
        if what < 0.25 and len(live) < seqs:
            led.allocate(nxt, r.randint(0, 5))
            nxt += 1
        elif what < 0.35 and live:
            s = r.choice(live)
            led.allocate(s, r.randint(0, min(2, cols - led.blocks[s])))
        elif what < 0.8 and live and len(live) < seqs:
            s = r.choice(live)
            if led.fork(s, nxt, r.randint(0, led.blocks[s] * BS), BS)[0] is AllocStatus.SUCCESS:
                nxt += 1
        elif live:
            led.release(r.choice(live))
        for kind, slot, n, *parent in led.take_ops():
            model.allocate(slot, n) if kind == 0 else model.release(slot) if kind == 1 else model.fork(slot, n, parent[0])
        order = list(led.blocks)
        r.shuffle(order)
        order = sorted(order) if step % 3 else order
        starts, columns = led.shared_runs(order)
        assert starts[0] == 0 and starts[-1] == len(order) and len(columns) == len(starts) - 1
        assert all(a < b for a, b in zip(starts, starts[1:]))
        for a, b, c in zip(starts, starts[1:], columns):
            rows = [model.rows[led.slot[s]] for s in order[a:b]]
            assert all(len(x) >= c and x[:c] == rows[0][:c] for x in rows)
            assert b - a > 1 or c == 0
            most = max(most, (b - a) * c)
    assert most >= 2  # some group shared some column


def test_groups_of_a_tree():
    """Forks of forks: a neighbour joins while the group reads no fewer columns together than without it."""
    from pie_b200.block_pool import BlockLedger

    led = BlockLedger(100, 10, 12)
    led.allocate(0, 8)
    led.fork(0, 1, 32, 4)
    led.fork(0, 2, 32, 4)
    led.fork(0, 3, 4, 4)
    led.fork(3, 4, 4, 4)
    led.allocate(5, 3)
    assert led.shared_runs([0, 1, 2]) == ([0, 3], [8])
    assert led.shared_runs([0, 1, 2, 3, 4, 5]) == ([0, 3, 5, 6], [8, 1, 0])  # 8 columns of three, not 1 of four
    assert led.shared_runs([0, 3]) == ([0, 2], [1])
    assert led.shared_runs([0, 5, 1]) == ([0, 1, 2, 3], [0, 0, 0])
    assert led.shared_runs([1, 1]) == ([0, 2], [8])
    assert led.shared_runs([]) == ([0], [])


def _args(num_groups=1):
    from pie_b200 import _lib

    io, kv, pg = _descs()
    io.max_q_len, io.lse = 1, None
    io.q_stride_seq = io.o_stride_seq = 8 * 128
    io.q_stride_head = io.o_stride_head = 128
    return io, kv, pg, _lib.PaGroups(1 << 23, 1 << 23, num_groups, 0)


@pytest.mark.parametrize("mutate,code,msg", [
    (lambda io, kv, pg, g: setattr(io, "max_q_len", 5), -2, b"<= 16"),
    (lambda io, kv, pg, g: setattr(io, "num_q_heads", 34), -2, b"<= 16"),
    (lambda io, kv, pg, g: setattr(io, "causal_top_left", 1), -1, b"bottom-right"),
    (lambda io, kv, pg, g: setattr(kv, "dtype", 3), -2, b"fp16, bf16 or int8"),
    (lambda io, kv, pg, g: setattr(kv, "dtype", 2), -1, b"k_scale"),
    (lambda io, kv, pg, g: setattr(kv, "head_dim", 96), -2, b"head_dim"),
    (lambda io, kv, pg, g: setattr(pg, "num_seqs", 4097), -2, b"4096"),
    (lambda io, kv, pg, g: setattr(g, "num_groups", 4097), -2, b"4096"),
    (lambda io, kv, pg, g: setattr(g, "num_groups", -1), -1, b"num_groups"),
    (lambda io, kv, pg, g: setattr(g, "group_start", None), -1, b"NULL"),
    (lambda io, kv, pg, g: setattr(g, "prefix_len", None), -1, b"NULL"),
    (lambda io, kv, pg, g: setattr(pg, "bt_cols", 1 << 28), -2, b"keys"),
])
def test_shared_prefix_arguments(mutate, code, msg):
    from pie_b200 import _lib

    lib = _lib.load()
    args = _args()
    mutate(*args)
    n = ctypes.c_size_t(0)
    assert lib.shared_prefix_workspace_size(*args, ctypes.byref(n)) == code, lib.paged_attn_error_string()
    assert msg in lib.paged_attn_error_string()
    assert lib.shared_prefix_attn(*args, None, 0, None, None) == code


def test_shared_prefix_needs_its_groups():
    from pie_b200 import _lib

    lib = _lib.load()
    args = _args()
    assert lib.shared_prefix_attn(*args[:3], None, None, 0, None, None) == _lib.PA_ERR_INVALID
    assert b"groups" in lib.paged_attn_error_string()


@pytest.mark.parametrize("kw,msg", [
    (dict(Q=torch.zeros(2, 4, 64)), "num_seqs, num_q_heads"),
    (dict(Q=torch.zeros(2, 4, 1, 128)), "head_dim of Q"),
    (dict(K=torch.zeros(4, 8, 2, 64), V=torch.zeros(4, 8, 2, 64)), "block_size"),
    (dict(block_table=torch.zeros(3, 3, dtype=torch.int32)), "block_table"),
    (dict(group_start=torch.zeros(3, dtype=torch.int32)), "group_start"),
    (dict(group_start=torch.zeros(0, dtype=torch.int32), prefix_len=torch.zeros(0, dtype=torch.int32)), "group_start"),
    (dict(prefix_len=torch.zeros(1, 1, dtype=torch.int32)), "group_start"),
    (dict(out=torch.zeros(2, 4, 1, 64)), "out must be"),
    (dict(out=torch.zeros(2, 4, 2, 64).half()), "out must be"),
    (dict(lse=torch.zeros(2, 4, 1)), "lse must be"),
])
def test_shared_prefix_front_end(kw, msg):
    from pie_b200 import ops

    one = torch.ones(2, dtype=torch.int32)
    args = dict(Q=torch.zeros(2, 4, 1, 64), K=torch.zeros(4, 16, 2, 64), V=torch.zeros(4, 16, 2, 64), q_len_per_seq=one,
                block_table=torch.zeros(2, 3, dtype=torch.int32), num_blocks_per_seq=one, block_size=16, kv_len_per_seq=one,
                group_start=torch.tensor([0, 2], dtype=torch.int32), prefix_len=torch.zeros(1, dtype=torch.int32))
    with pytest.raises(ValueError, match=msg):
        ops.shared_prefix_attention(**{**args, **kw})


def test_groups_layout_matches_header(tmp_path):
    from pie_b200 import _lib

    names = [f for f, _ in _lib.PaGroups._fields_]
    src = tmp_path / "layout.c"
    src.write_text("\n".join(['#include <stdio.h>', '#include <stddef.h>', '#include "paged_attn_b200.h"', "int main(void) {",
                              'printf("%zu", sizeof(pa_groups_t));']
                             + [f'printf(" %zu", offsetof(pa_groups_t, {f}));' for f in names] + ["return 0; }"]))
    exe = tmp_path / "layout"
    subprocess.run(["gcc", "-I", os.path.join(ROOT, "include"), str(src), "-o", str(exe)], check=True)
    got = [int(x) for x in subprocess.run([str(exe)], capture_output=True, text=True, check=True).stdout.split()]
    assert got == [ctypes.sizeof(_lib.PaGroups)] + [getattr(_lib.PaGroups, f).offset for f in names]
