"""CPU: the 2-norm bound of tests/test_gpu_shared_prefix_norms.py passes a row computed with the kernels' roundings, and none with a mistake."""
import math

import pytest
import torch

from oracle.shared_prefix import attend, lse_bound, norm_bound


def rows(pool, n, D, seed):
    g = torch.Generator().manual_seed(seed)
    H = 6  # rows and heads together: the fewest of a GPU test
    q = (torch.randn(H, D, generator=g) * 1.5).to(torch.bfloat16 if pool == torch.bfloat16 else torch.float16).double()
    if pool == torch.int8:
        codes = torch.randint(-127, 128, (2, n, H, D), generator=g).double()
        scales = (torch.rand(2, n, H, 1, generator=g) * 0.02 + 0.005).half().double()
        return q, codes, scales
    return q, torch.randn(2, n, H, D, generator=g).to(pool).double(), torch.ones(2, n, H, 1, dtype=torch.float64)


def as_a_kernel(q, k, v, scale, operand):
    """o in fp16: logits and sums in 32 bits, probabilities rounded to the operand type against the largest so far, tile by tile."""
    s = (torch.einsum("hd,nhd->hn", q.float(), k.float()) * scale)
    o, l, m = torch.zeros(q.shape), torch.zeros(q.shape[0]), torch.full((q.shape[0],), -math.inf)
    for t in range(0, s.shape[1], 128):
        new = torch.maximum(m, s[:, t:t + 128].amax(1))
        o, l, m = o * (m - new).exp()[:, None], l * (m - new).exp(), new
        p = (s[:, t:t + 128] - m[:, None]).exp()
        l = l + p.sum(1)
        o = o + torch.einsum("hn,nhd->hd", p.to(operand).float(), v[t:t + 128].float())
    return (o / l[:, None]).half().double(), (m + l.log()).half().double()


@pytest.mark.parametrize("pool", [torch.float16, torch.bfloat16, torch.int8])
@pytest.mark.parametrize("n", [200, 2100, 20000])
def test_what_the_bound_passes(pool, n):
    D, scale = 128, 1 / math.sqrt(128)
    operand = torch.float16 if pool == torch.int8 else pool
    unit = torch.finfo(operand).eps / 2
    for seed in range(1 if n > 10000 else 3):
        q, kv, scales = rows(pool, n, D, seed)
        k, v = (kv * scales).half().double() if pool == torch.int8 else kv
        o, lse, w = attend(q, k, v, scale)
        bound, lse_most = norm_bound(q, k, v, scale, o, w, unit), lse_bound(q, k, scale, lse)
        got, got_lse = as_a_kernel(q, k, v, scale, operand)
        off = (got - o).norm(dim=1)
        assert bool((off <= bound).all()) and bool(((got_lse - lse).abs() <= lse_most).all())

        def passes(x):
            return bool(((x - o).norm(dim=1) <= bound).all())

        assert not passes(torch.zeros_like(o))
        for t in range(0, n - 127, max(128, n // 10 // 128 * 128)):
            keep = torch.ones(n, dtype=torch.bool)
            keep[t:t + 128] = False
            assert not passes(as_a_kernel(q, k[keep], v[keep], scale, operand)[0])  # a tile left out
            other = torch.randint(0, n - 128, (1,), generator=torch.Generator().manual_seed(t)).item()
            x = v.clone()
            x[t:t + 128] = v[other:other + 128] if abs(other - t) > 16 else v[t:t + 128].flip(0)
            assert not passes(as_a_kernel(q, k, x, scale, operand)[0])  # a tile of values from elsewhere
            if pool == torch.int8:
                for which in (0, 1):
                    sc = scales.clone()
                    sc[which, t:t + 128] = scales[which, t:t + 128].flip(0)
                    k2, v2 = (kv * sc).half().double()
                    assert not passes(as_a_kernel(q, k2, v2, scale, operand)[0])  # a tile with other keys' scales
