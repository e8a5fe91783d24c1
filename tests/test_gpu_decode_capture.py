"""Captured few-token layers whose workspace holds other data than zeros where the layer needs none."""

import pytest
import torch

import fast_route_b200 as fr
from fast_route_b200 import synth

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,H,I,E,k", [(1, 256, 512, 8, 2), (16, 512, 96, 32, 6), (9, 64, 1024, 200, 4)])
def test_replays_over_memory_that_was_used(dev, M, H, I, E, k):
    """The graph's pool is filled with NaN bit patterns between the replays; layers of one graph also use it in turn."""
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=M, dtype=torch.bfloat16, weight_std=0.05))
    q = fr.quantize_experts_fp4(w1, w2)
    run = lambda: (fr.fused_moe_decode(x, gate, w1, w2, k),  # noqa: E731
                   fr.fused_moe_decode_fp4(x, gate, q[0], q[1], q[3], q[4], k, w1_global=q[2], w2_global=q[5]))
    want = run()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        junk = torch.full((16 << 20,), -1, dtype=torch.int8, device=dev)       # freed: the layers' workspaces come from here
        del junk
        first = run()
        junk = torch.full((16 << 20,), -1, dtype=torch.int8, device=dev)
        del junk
        second = run()
    for _ in range(4):
        for t in first + second:
            t.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(first + second, want + want))
