"""Operators called from several threads: every result is that of the call by itself, bit for bit."""

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
