"""Whose scratch a call gets: every thread has its own on a stream, and takes over what an ended one has left there."""

from __future__ import annotations

import threading

import pytest
import torch

from conftest import seeded


@pytest.fixture
def table(monkeypatch):
    """The table of eager workspaces, empty, with tensors on the CPU and a stream that the test names."""
    from phyai_amd import ops

    zeros = torch.zeros
    stream = {"now": 7}
    monkeypatch.setattr(ops, "_workspaces", {})
    monkeypatch.setattr(ops, "_retired", [])
    monkeypatch.setattr(ops, "_stream_ptr", lambda: stream["now"])
    monkeypatch.setattr(torch, "zeros", lambda *a, device=None, **kw: zeros(*a, **kw))
    return ops, stream


def reserve(ops, nbytes=100):
    return ops.reserve_workspace(nbytes, torch.device("cuda", 0))


def test_threads_of_one_stream_share_nothing(table):
    ops, _ = table
    mine, got, inside, leave = reserve(ops), [], threading.Barrier(3), threading.Event()

    def work():
        got.append(reserve(ops))
        inside.wait(20)
        leave.wait(20)
        got.append(reserve(ops))

    threads = [threading.Thread(target=work) for _ in range(2)]
    for t in threads:
        t.start()
    inside.wait(20)
    assert len({t.data_ptr() for t in [mine, *got]}) == 3 and len(ops._workspaces) == 3
    leave.set()
    for t in threads:
        t.join(20)
    assert len({t.data_ptr() for t in [mine, *got]}) == 3       # each met its own again
    assert reserve(ops) is mine and not ops._retired


def test_an_ended_thread_leaves_its_workspaces_to_the_next_on_the_stream(table):
    ops, stream = table
    seen = []
    for now in (7, 7, 8, 7, 8):
        stream["now"] = now
        t = threading.Thread(target=lambda: seen.append(reserve(ops)))
        t.start()
        t.join(20)
    assert seen[0] is seen[1] is seen[3] and seen[2] is seen[4] and seen[0] is not seen[2]
    assert len(ops._workspaces) == 2
    stream["now"] = 7
    bigger = reserve(ops, seen[0].numel() + 1)                  # taken over, then outgrown: kept, as anyone's is
    assert ops._retired == [seen[0]] and bigger.numel() > seen[0].numel() and len(ops._workspaces) == 2


@pytest.mark.gpu
def test_threads_of_one_stream_at_once(dev):
    """Two-launch linears and split attention from three threads on the default stream: the results of calls made alone."""
    import layer_oracle as oracle
    from phyai_amd import ops
    from test_gpu_layer_ops import attend_case

    gen = torch.Generator().manual_seed(5)
    w, ws = (t.to(dev) for t in oracle.block_weight(512, 512, gen))
    wq, wscale = ops.fp8_weight_quant(seeded((512, 512), 6).to(dev))
    kinds = []
    for i in range(3):
        x = seeded((1500 + 100 * i, 512), i).to(dev)
        q, k, v, table, offsets, lens, kw = attend_case(([2, 1], [900 - 50 * i, 700], 16, 8, 1, 256, True, None), torch.bfloat16, dev, seed=i)
        args = [t.to(dev) for t in (q, k, v, table, offsets, lens)]
        kinds.append([lambda x=x: ops.fp8_block_linear(x, w, ws), lambda args=args, kw=kw: ops.paged_attention(*args, **kw),
                      lambda x=x: ops.fp8_linear(x, wq, wscale)])
    alone = [[call() for call in calls] for calls in kinds]
    torch.cuda.synchronize()
    wrong, used, start = [], [], threading.Barrier(3)

    def work(i):
        start.wait(20)
        results = [[call() for call in kinds[i]] for _ in range(40)]
        used.append(ops.reserve_workspace(1).data_ptr())
        start.wait(20)
        torch.cuda.synchronize()
        wrong.extend((i, n) for r in results for n, (a, b) in enumerate(zip(r, alone[i])) if not torch.equal(a, b))

    threads = [threading.Thread(target=work, args=(i,)) for i in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(60)
    assert not wrong and len(set(used)) == 3
