"""CPU: how a step's order is cut into groups that share a prefix: as many columns saved as any cuts save."""
import itertools
import random

import pytest


def ledger():
    from pie_b200.block_pool import BlockLedger

    return BlockLedger(100000, 5000, 5000)


def two_documents():
    """A system prompt of 1 block; sequence 100 asks about document A, 200 to 231 about document B, both of 1024 blocks."""
    led = ledger()
    led.allocate(0, 1)
    for doc, first, n in ((1, 100, 1), (2, 200, 32)):
        led.fork(0, doc, 4, 4)
        led.allocate(doc, 1024)
        for s in range(first, first + n):
            led.fork(doc, s, 1025 * 4, 4)
    return led


@pytest.mark.parametrize("order,want", [
    ([100, *range(200, 232)], ([0, 1, 33], [0, 1025])),
    ([*range(200, 232), 100], ([0, 32, 33], [1025, 0])),
    ([*range(200, 232)], ([0, 32], [1025])),
    ([*range(200, 216), 100, *range(216, 232)], ([0, 16, 17, 33], [1025, 0, 1025])),
    ([100, 200], ([0, 2], [1])),
])
def test_a_neighbour_does_not_cost_the_others_their_prefix(order, want):
    assert two_documents().shared_runs(order) == want


def common(led, a, b):
    paths = []
    for s in (a, b):
        path, node = [], led.prefix.get(s)
        while node is not None:
            path.append(node)
            node = node.up
        paths.append(path[::-1])
    return sum(x.n for x, y in itertools.takewhile(lambda p: p[0] is p[1], zip(*paths)))


def saved(led, order, starts, pairs=lambda run: itertools.combinations(run, 2)):
    return sum((b - a - 1) * min((common(led, x, y) for x, y in pairs(order[a:b])), default=0) for a, b in zip(starts, starts[1:]))


@pytest.mark.parametrize("seed", range(40))
def test_no_cuts_save_more(seed):
    """Random trees of forks, in random orders (a sequence twice, too), against all cuts."""
    r = random.Random(seed)
    led = ledger()
    led.allocate(0, r.randint(1, 9))
    for s in range(1, 12):
        parent = r.randrange(s) if r.random() < 0.9 else None
        if parent is None:
            led.allocate(s, r.randint(0, 9))
            continue
        led.fork(parent, s, r.randint(0, led.blocks[parent]) * 4, 4)
        led.allocate(s, r.randint(0, 4))
    for _ in range(5):
        order = [r.randrange(12) for _ in range(r.randint(1, 9))]
        order = sorted(order) if r.random() < 0.5 else order
        starts, columns = led.shared_runs(order)
        assert starts[0] == 0 and starts[-1] == len(order) and len(columns) == len(starts) - 1
        for a, b, c in zip(starts, starts[1:], columns):
            assert a < b and c == (min(common(led, x, y) for x, y in itertools.combinations(order[a:b], 2)) if b - a > 1 else 0)
        most = max(saved(led, order, [0, *cut, len(order)]) for n in range(len(order)) for cut in itertools.combinations(range(1, len(order)), n))
        assert saved(led, order, starts) == most, (order, starts, columns)


def test_many_widths():
    """A chain in which every sequence was forked later than the one before: hundreds of widths, of which some are weighed."""
    led = ledger()
    led.allocate(0, 1)
    for s in range(1, 600):
        led.fork(s - 1, s, led.blocks[s - 1] * 4, 4)
        led.allocate(s, 1)
    order = list(range(600))
    starts, columns = led.shared_runs(order)
    for a, b, c in zip(starts, starts[1:], columns):
        assert c == (common(led, order[a], order[a + 1]) if b - a > 1 else 0)  # in this chain the first two share the least
    mine, halves, one = (saved(led, order, cuts, itertools.pairwise) for cuts in (starts, [0, 300, 600], [0, 600]))
    assert mine > halves > one
