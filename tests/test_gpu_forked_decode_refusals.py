"""GPU: what beam search and the captured step refuse before anything is written."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def search(B, K, V=40):
    from pie_b200.beam import BeamSearch
    from pie_b200.block_pool import DeviceBlockManager

    k, v = (torch.zeros(40, 4, 1, 64, dtype=torch.float16, device="cuda") for _ in range(2))
    pool = DeviceBlockManager(40, 4, 20, 8)
    pool.attach_caches(k, v)
    for s in range(B):
        pool.allocate(s, 2)
    return BeamSearch(pool, list(range(B)), [7] * B, torch.zeros(B, V, device="cuda"), K, 0, 5)


def words(*keep):
    """A mask's words for the tokens in ``keep``, of a vocabulary of 40."""
    bits = [0, 0]
    for t in keep:
        bits[t // 32] |= 1 << t % 32
    return torch.tensor([b - (1 << 32) if b >> 31 else b for b in bits], dtype=torch.int32)


@pytest.mark.parametrize("shape", [(1, 2, 2), (2, 3, 2), (4, 1, 2), (1, 4, 2), (2, 2, 2, 2)])
def test_masks_of_another_shape(shape):
    """Three dimensions are [B, K, words], or 1 for the beams or both; rows of another order are not taken for those."""
    s = search(2, 2)
    s.step_inputs()
    before = s.tokens.clone()
    with pytest.raises(ValueError, match="mask"):
        s.advance(torch.zeros(2, 2, 40, device="cuda"), torch.full(shape, -1, dtype=torch.int32, device="cuda"))
    assert torch.equal(s.tokens, before)
    s.advance(torch.zeros(2, 2, 40, device="cuda"))  # the search goes on
    s.finish()


def test_masks_of_each_shape():
    """Beam by beam, sequence by sequence, and one for all."""
    a, b = words(3, 9), words(5, 33)
    for mask, allowed in ((torch.stack([torch.stack([a, a]), torch.stack([b, b])]), [{3, 9}, {5, 33}]), (torch.stack([a, b]), [{3, 9}, {5, 33}]),
                          (torch.stack([a, b]).unsqueeze(1), [{3, 9}, {5, 33}]), (a, [{3, 9}] * 2), (b.view(1, 2), [{5, 33}] * 2),
                          (b.view(1, 1, 2), [{5, 33}] * 2), (torch.stack([a, a, b, b]), [{3, 9}, {5, 33}])):
        s = search(2, 2)
        s.step_inputs()
        got = s.advance(torch.randn(2, 2, 40, device="cuda"), mask.cuda()).tolist()
        for seq in range(2):
            assert set(got[seq]) <= allowed[seq] | {0}, (tuple(mask.shape), got)  # (a finished beam goes on with 0)
        s.finish()


def test_a_step_beyond_the_rotation_table():
    """A position without a row of the table would leave the token out and attend to what its slot held."""
    from pie_b200 import ops
    from pie_b200.block_pool import DeviceBlockManager
    from pie_b200.decode_step import DecodeStepGraph

    BS, H, D, NB = 4, 1, 64, 20
    k, v = (torch.zeros(NB, BS, H, D, dtype=torch.float16, device="cuda") for _ in range(2))
    pool = DeviceBlockManager(NB, BS, 4, 12)
    pool.attach_caches(k, v)
    graph = DecodeStepGraph(pool, k, v, None, None, 2, 2, rope=ops.rope_table(9, D, device="cuda"), share_prefixes=True)
    pool.allocate(0, 2)
    pool.allocate(1, 2)
    q, kn, vn = (torch.randn(2, h, D, device="cuda").half() for h in (2, 1, 1))
    graph.step([0, 1], [8, 9], q, kn, vn)
    free, cache = pool.num_free_blocks(), k.clone()
    with pytest.raises(ValueError, match="rope"):
        graph.step([0, 1], [9, 10], q, kn, vn)
    assert pool.num_free_blocks() == free and torch.equal(k, cache)
    graph.step([0], [9], q[:1], kn[:1], vn[:1])
    graph.check()
