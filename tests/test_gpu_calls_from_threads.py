"""GPU: calls of different sizes from several host threads at once: every one launches, and its outputs are those of the call alone."""
import threading

import pytest
import torch

from test_gpu_shared_prefix import Problem

pytestmark = pytest.mark.gpu


def race(calls, times):
    """Each of ``calls`` in its own thread and on its own stream, ``times`` times; the last outputs, and what was raised."""
    last, raised = [None] * len(calls), []
    gate = threading.Barrier(len(calls))

    def work(i):
        stream = torch.cuda.Stream()
        gate.wait()
        try:
            with torch.cuda.stream(stream):
                for _ in range(times):
                    last[i] = calls[i]()
            stream.synchronize()
        except Exception as e:  # noqa: BLE001
            raised.append(e)

    torch.cuda.synchronize()
    threads = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    torch.cuda.synchronize()
    return last, raised


@pytest.mark.parametrize("backend", ["torch", "ctypes"])
def test_batches_of_different_sizes(monkeypatch, backend):
    """The work lists' share of a launch's shared memory goes by the batch: no call may lower what another is about to launch with."""
    from pie_b200 import ops

    monkeypatch.setattr(ops, "BACKEND", backend)
    ps = [Problem([(2, 64)] * n, [[3, 5]] * n, Hq=2, Hkv=1, D=64, seed=n) for n in (1, 40, 300, 700)]
    calls = [lambda p=p: ops.shared_prefix_attention(*p.args()) for p in ps]
    want = [c() for c in calls]
    got, raised = race(calls, 1500)
    assert not raised, raised[0]
    for (o, l), (o2, l2) in zip(want, got):
        assert torch.equal(o, o2) and torch.equal(l, l2)


@pytest.mark.parametrize("backend", ["torch", "ctypes"])
def test_decode_batches_of_different_sizes(monkeypatch, backend):
    """The same of paged_attention's split-K kernel."""
    from pie_b200 import ops

    monkeypatch.setattr(ops, "BACKEND", backend)
    ps = [Problem([(1, 16)] * n, [[3]] * n, Hq=2, Hkv=1, D=64, seed=n) for n in (1, 33, 65, 97, 600, 900)]
    calls = [lambda p=p: ops.paged_attention(*p.args()[:8], mode="decode") for p in ps]
    want = [c() for c in calls]
    got, raised = race(calls, 6000)
    assert not raised, raised[0]
    for (o, l), (o2, l2) in zip(want, got):
        assert torch.equal(o, o2) and torch.equal(l, l2)


def test_large_batches_of_groups():
    """The plan of more than some 1500 sequences and groups takes more shared memory than a kernel has by default."""
    from pie_b200 import ops

    ps = [Problem([(2, 16)] * n, [[1, 2]] * n, Hq=1, Hkv=1, D=64, seed=n) for n in (2, 1400, 1800, 2048)]
    calls = [lambda p=p: ops.shared_prefix_attention(*p.args()) for p in ps]
    want = [c() for c in calls]
    got, raised = race(calls, 800)
    assert not raised, raised[0]
    for (o, l), (o2, l2) in zip(want, got):
        assert torch.equal(o, o2) and torch.equal(l, l2)
