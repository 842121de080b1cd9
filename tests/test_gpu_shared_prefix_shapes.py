"""GPU: shared prefixes of shapes that the plan treats apart: more rows than the GPU holds at once, large groups beside small ones, blocks
longer than a tile, blocks past 32-bit offsets.  By the 2-norm of a head's error (tests/test_gpu_shared_prefix_norms.py)."""
import numpy as np
import pytest
import torch

from test_gpu_shared_prefix import POOLS, Problem
from test_gpu_shared_prefix_norms import check_norms, parts

pytestmark = pytest.mark.gpu


def run(p, shared, rows):
    from pie_b200 import ops

    status = torch.zeros(1, dtype=torch.int32, device="cuda")
    O, L = ops.shared_prefix_attention(*p.args(), status=status)
    assert status.item() == 0
    check_norms(p, O, L, shared, True, rows=rows)
    again = ops.shared_prefix_attention(*p.args())
    assert torch.equal(O, again[0]) and torch.equal(L, again[1])


@pytest.mark.parametrize("pool", POOLS)
def test_more_rows_than_a_pass_holds(pool):
    """2500 sequences of 16 heads on one KV head: 157 pairs of row tiles, more than SMs, so that K and V are passed over twice."""
    rng = np.random.default_rng(1)
    p = Problem([(2500, 400)], [rng.integers(1, 20, 2500).tolist()], Hq=16, Hkv=1, pool=pool, seed=1)
    run(p, parts([(2500, 400)], 16), sorted({0, 1, 15, 16, 2367, 2368, 2369, 2499, *rng.integers(0, 2500, 30).tolist()}))


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("D", [64, 128])
def test_large_and_small_groups(pool, D):
    """Groups of one row tile, of one pair and of ten in one call, with short and long prefixes, and sequences of none."""
    rng = np.random.default_rng(2)
    groups = [(2, 5000), (300, 2048), (40, 1000), (3, 130), (33, 64), (1, 500), (9, 3000)]
    p = Problem(groups, [rng.integers(1, 50, n).tolist() for n, _ in groups], alone=[1, 700, 20], Hq=16, Hkv=2, D=D, pool=pool, seed=2)
    run(p, parts(groups, 16, 3), sorted({0, 1, 2, 33, 34, 35, 301, 302, 341, 342, 345, 378, 387, 390, *rng.integers(0, 391, 10).tolist()}))


@pytest.mark.parametrize("pool", POOLS)
@pytest.mark.parametrize("BS", [128, 512])
def test_long_blocks(pool, BS):
    groups = [(20, 1024), (5, 3 * BS)]
    rng = np.random.default_rng(3)
    p = Problem(groups, [rng.integers(1, 2 * BS, n).tolist() for n, _ in groups], alone=[BS + 1], BS=BS, pool=pool, seed=3, spare=2)
    run(p, parts(groups, BS, 1), [0, 7, 19, 20, 24, 25])


@pytest.mark.parametrize("pool", POOLS)
def test_blocks_past_32_bit_offsets(pool):
    """A pool of more than 2^32 bytes (2^31 elements), of which the last blocks are used."""
    NB = (1 << 31) // (16 * 8 * 128) + 4000
    p = Problem([(24, 1600), (3, 800)], [[9] * 24, [40] * 3], Hq=32, Hkv=8, pool=pool, seed=4)
    n = p.K.shape[0]
    far = torch.empty(2, NB, 16, 8, 128, dtype=pool, device="cuda")
    far[:, NB - n:] = torch.stack([p.K, p.V])
    p.K, p.V = far[0], far[1]
    if p.ks is not None:
        p.ks, p.vs = (torch.cat([torch.zeros(NB - n, *s.shape[1:], dtype=s.dtype, device="cuda"), s]) for s in (p.ks, p.vs))
    p.table[p.table < n] += NB - n
    run(p, parts([(24, 1600), (3, 800)], 16), [0, 11, 23, 24, 26])
    del far
    torch.cuda.empty_cache()
