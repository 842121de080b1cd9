"""CPU: the captured step's check of positions against its rotation table, before the pool is asked for anything."""
import pytest
import torch


def test_positions_that_the_table_does_not_hold():
    from pie_b200.block_pool import BlockLedger
    from pie_b200.decode_step import DecodeStepGraph
    from test_block_sharing_cpu import _host_manager

    led = BlockLedger(40, 8, 6)
    led.allocate(0, 3)
    led.allocate(1, 3)
    graph = DecodeStepGraph.__new__(DecodeStepGraph)
    graph.pool, graph.S, graph.BS = _host_manager(led), 4, 4
    graph.pool.flush = lambda: (_ for _ in ()).throw(KeyError("the device"))
    graph.graphs, graph.pool.max_blocks_per_seq = (), 6
    for rope, lens in ((None, [9, 12]), (torch.zeros(12, 16), [9, 12])):
        graph.rope = rope
        with pytest.raises(KeyError, match="the device"):  # what the host lets pass
            graph.step([0, 1], lens, None, None, None)
    graph.rope = torch.zeros(11, 16)
    with pytest.raises(ValueError, match="rope holds 11 positions"):
        graph.step([0, 1], [9, 12], None, None, None)
