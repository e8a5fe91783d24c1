"""Operators of several launches called from two threads at once on one stream, and captured ones replayed side by side:
every result is that of the call by itself, bit for bit."""

import threading

import pytest
import torch

import fast_route_b200 as fr
from fast_route_b200 import synth

pytestmark = pytest.mark.gpu


def _matrix(seed, rows, k, block, dev):
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8)
    lo, hi, dt = (0x20, 0x50, torch.float8_e4m3fn) if block == 16 else (118, 136, torch.float8_e8m0fnu)
    s = torch.randint(lo, hi, (rows, k // block), generator=g, dtype=torch.uint8).view(dt)
    return q.to(dev), s.to(dev)


def _calls(dev, which):
    """Calls of one thread: products of more than 128 tokens and matrices quantised in two launches, sizes in turn."""
    calls = []
    for i, (m, n, k, block) in enumerate([(200, 600, 2080, 16), (1000, 264, 544, 32), (333, 1399, 1056, 16), (3000, 512, 256, 32)]):
        a, b = _matrix(10 * which + i, m, k, block, dev), _matrix(100 + 10 * which + i, n, k, block, dev)
        calls.append(lambda a=a, b=b: (fr.matmul_fp4(*a, *b),))
        x = torch.randn(m, 512, generator=torch.Generator().manual_seed(which * 31 + i)).to(dev) * 10.0 ** (3 * which + i)
        calls.append(lambda x=x: fr.quantize_fp4(x))
    return calls


def _same(a, b):
    return all(torch.equal(x.view(torch.uint8), y.view(torch.uint8)) for x, y in zip(a, b))


@pytest.mark.parametrize("m", [3, 200])
def test_the_first_call_of_a_thread(dev, m):
    """A thread that has not used the GPU before: its first call makes tensor maps, which need a context."""
    a, b = _matrix(1, m, 512, 16, dev), _matrix(2, 300, 512, 16, dev)
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(m, 256, 128, 4, seed=1, dtype=torch.bfloat16, weight_std=0.05))
    calls = [lambda: fr.matmul_fp4(*a, *b), lambda: fr.fused_moe(x, gate, w1, w2, 2)]
    want = [c() for c in calls]
    torch.cuda.synchronize()
    got = [None, None]

    def go(i):
        got[i] = calls[i]()
    for i in range(2):
        t = threading.Thread(target=go, args=(i,))
        t.start()
        t.join()
    assert all(g is not None and torch.equal(g, w) for g, w in zip(got, want))


def test_two_threads_on_one_stream(dev):
    calls = [_calls(dev, 0), _calls(dev, 1)]
    want = [[c() for c in mine] for mine in calls]
    torch.cuda.synchronize()
    wrong, errors = [], []
    start = threading.Barrier(2, timeout=60)

    def go(which):
        try:
            start.wait()
            got = []
            for _ in range(40):
                got += [(i, c()) for i, c in enumerate(calls[which])]
            wrong.extend((which, i) for i, r in got if not _same(r, want[which][i]))
        except BaseException as e:      # noqa: BLE001  (reported below)
            errors.append(e)
    threads = [threading.Thread(target=go, args=(w,)) for w in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert not wrong, wrong[:5]


def test_captured_calls_replayed_side_by_side(dev):
    calls = [_calls(dev, 0), _calls(dev, 1)]
    want = [[c() for c in mine] for mine in calls]
    graphs, got = [], []
    for mine in calls:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got.append([c() for c in mine])
        graphs.append(graph)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(5):
        for results in got:
            for r in results:
                for t in r:
                    t.view(torch.uint8).zero_()
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        eager = [c() for c in calls[0]]
        torch.cuda.synchronize()
        assert all(_same(r, w) for results, wants in zip(got, want) for r, w in zip(results, wants))
        assert all(_same(r, w) for r, w in zip(eager, want[0]))
