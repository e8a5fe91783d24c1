"""The few-token layer beside ``fused_moe``, with infinities at ragged row ends, at large sizes, from two threads, and with
waits that run out in some thread blocks only."""

import threading

import numpy as np
import pytest
import torch

import fast_route_b200 as fr
from fast_route_b200 import synth
from oracle import fp4 as o

pytestmark = pytest.mark.gpu


def _np(t):
    return t.detach().cpu().double().numpy()


def _values(q, s, g, block):
    return o.values(q.cpu().numpy(), s.view(torch.uint8).cpu().numpy(), None if g is None else _np(g), block)


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,H,I,E,k", [(1, 256, 256, 8, 2), (5, 512, 1408, 64, 6), (9, 64, 64, 4, 2), (16, 264, 520, 60, 8),
                                       (16, 1024, 1536, 8, 2), (3, 2048, 352, 16, 4)])
def test_same_layer_as_fused_moe(dev, M, H, I, E, k, dt):
    """Where both choose the same experts: weights from logits that are each within fp32 accumulation of the exact ones, and
    outputs within the sum of both layers' bounds, each for its own routing weights.  fused_moe may also round every
    expert's share to the 16-bit type before it adds them up."""
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=M + I, dtype=dt, weight_std=0.05))
    a, aw, ai = fr.fused_moe_decode(x, gate, w1, w2, k, return_routing=True)
    b, bw, bi = fr.fused_moe(x, gate, w1, w2, k, return_routing=True)
    agree = (ai == bi).all(1).cpu().numpy()
    assert agree.mean() > 0.9
    slack = 2 * (H + 8) * 2.0 ** -24 * (np.abs(_np(x)) @ np.abs(_np(gate))).max(1, keepdims=True)
    aw, bw = _np(aw), _np(bw)
    assert (np.abs(aw - bw) <= (4 * slack + 2 * (E + 16) * 2.0 ** -24) * bw + 1e-37)[agree].all()
    eps, tiny = torch.finfo(dt).eps, float(torch.finfo(dt).smallest_normal)
    ids = ai.cpu().numpy()
    ref_a, err_a = o.layer_with_bound(_np(x), _np(w1), _np(w2), ids, aw, eps)
    ref_b, err_b = o.layer_with_bound(_np(x), _np(w1), _np(w2), ids, bw, eps)
    share = np.zeros_like(ref_b)
    for j in range(k):
        r, e = o.layer_with_bound(_np(x), _np(w1), _np(w2), ids[:, j:j + 1], bw[:, j:j + 1], eps)
        share += eps / 2 * (np.abs(r) + e) * (1 + eps)
    bound = err_a + err_b + share + np.abs(ref_a - ref_b) + 4 * tiny * (1 + np.abs(ref_a).max())
    assert (np.abs(_np(a) - _np(b)) <= bound)[agree].all()


@pytest.mark.parametrize("M", [3, 9, 16])
@pytest.mark.parametrize("H,I", [(288, 352), (416, 544), (352, 1408), (1056, 288)])
@pytest.mark.parametrize("block,dt", [(0, torch.bfloat16), (0, torch.float16), (16, torch.bfloat16), (16, torch.float16),
                                      (32, torch.bfloat16)])
def test_infinite_tokens_at_ragged_row_ends(dev, M, H, I, block, dt):
    """Row lengths that end in the first and in the second half of a step, all weights positive: an infinite token's outputs
    are infinite, not NaN from the filling past the row's end, and the others as if it were finite, bit for bit."""
    E, k = 2, 2
    g = torch.Generator().manual_seed(M + H)
    gate = torch.zeros(H, E, dtype=dt, device=dev)                     # both experts, half each
    x = torch.rand(M, H, generator=g).to(dt)
    if block == 0:
        w1 = (torch.rand(E, 2 * I, H, generator=g) * 0.01 + 0.01).to(dt).to(dev)
        w2 = (torch.rand(E, H, I, generator=g) * 0.01 + 0.01).to(dt).to(dev)
        run = lambda v: fr.fused_moe_decode(v.to(dev), gate, w1, w2, k)  # noqa: E731
    else:
        def matrix(rows, cols):
            code = torch.randint(1, 8, (E, rows, cols), generator=g, dtype=torch.uint8)
            lo, hi, sdt = (0x10, 0x18, torch.float8_e4m3fn) if block == 16 else (119, 121, torch.float8_e8m0fnu)
            s = torch.randint(lo, hi, (E, rows, cols // block), generator=g, dtype=torch.uint8)
            return (code[..., 0::2] | (code[..., 1::2] << 4)).to(dev), s.view(sdt).to(dev)
        (q1, s1), (q2, s2) = matrix(2 * I, H), matrix(H, I)
        run = lambda v: fr.fused_moe_decode_fp4(v.to(dev), gate, q1, s1, q2, s2, k)  # noqa: E731
    clean = run(x)
    # Finite, but where the exact result is past fp16: with weights of `mean` on average the first product is H / 2 * mean, an
    # activation its square (silu(h) * h, h > 4), and I of them make I * mean as much: H = 352, I = 1408, blocks of 16:
    # (352 / 2 * 0.117)^2 * 1408 * 0.117 = 70000 > 65504.
    mean = {0: 0.015, 16: 0.117, 32: 0.016}[block]
    assert not torch.isnan(clean).any()
    assert torch.isfinite(clean).all() or (H / 2 * mean) ** 2 * I * mean > torch.finfo(dt).max / 2
    for bad in {1, M - 1}:
        for at in (5, H - 3):
            y = x.clone()
            y[bad, at] = float("inf")
            out = run(y)
            rest = [t for t in range(M) if t != bad]
            assert torch.equal(out[rest], clean[rest])
            assert (out[bad] == float("inf")).all()


@pytest.mark.parametrize("M,H,I,E,k", [(16, 8200, 264, 3, 2), (2, 264, 14336, 2, 1), (16, 2048, 1408, 6, 3), (5, 4096, 2816, 2, 2)])
@pytest.mark.parametrize("block", [0, 16, 32])
def test_bound_at_large_sizes(dev, M, H, I, E, k, block):
    if block:
        H, I = -(-H // 32) * 32, -(-I // 32) * 32
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=H, dtype=torch.bfloat16, weight_std=0.03))
    if block == 0:
        out, tw, ti = fr.fused_moe_decode(x, gate, w1, w2, k, return_routing=True)
        e1, e2 = _np(w1), _np(w2)
    else:
        q1, s1, g1, q2, s2, g2 = fr.quantize_experts_fp4(w1, w2, block)
        out, tw, ti = fr.fused_moe_decode_fp4(x, gate, q1, s1, q2, s2, k, w1_global=g1, w2_global=g2, return_routing=True)
        e1, e2 = _values(q1, s1, g1, block), _values(q2, s2, g2, block)
    ref, err = o.layer_with_bound(_np(x), e1, e2, ti.cpu().numpy(), _np(tw), torch.finfo(torch.bfloat16).eps)
    assert (np.abs(_np(out) - ref) <= err).all()


def test_two_threads_on_one_stream(dev):
    """Layers of different sizes and formats from two threads, whose cached workspace grows meanwhile."""
    calls = []
    for i, (M, H, I, E, k) in enumerate([(1, 256, 512, 4, 2), (16, 512, 96, 32, 6), (3, 2048, 64, 8, 1), (16, 1024, 2816, 8, 8)]):
        x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=i, dtype=torch.bfloat16, weight_std=0.05))
        q = fr.quantize_experts_fp4(w1, w2)
        calls.append(lambda a=(x, gate, w1, w2, k): fr.fused_moe_decode(*a))
        calls.append(lambda x=x, gate=gate, q=q, k=k: fr.fused_moe_decode_fp4(x, gate, q[0], q[1], q[3], q[4], k,
                                                                              w1_global=q[2], w2_global=q[5]))
    want = [c() for c in calls]
    torch.cuda.synchronize()
    fr._lib._workspaces.clear()
    got, errors = [], []
    start = threading.Barrier(2, timeout=60)

    def go(which):
        try:
            start.wait()
            for r in range(30):
                got.extend((i, calls[i]()) for i in (range(len(calls)) if which else reversed(range(len(calls)))))
        except BaseException as e:      # noqa: BLE001  (reported below)
            errors.append(e)
    threads = [threading.Thread(target=go, args=(w,)) for w in (0, 1)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors, errors
    assert len(got) == 60 * len(calls) and all(torch.equal(r, want[i]) for i, r in got)


@pytest.mark.reads_status
def test_some_blocks_give_up_and_others_do_not(dev):
    """Poll budgets from one on upwards: with the smallest some waits run out, with the largest none, and between them some
    thread blocks report and others do not (one token: every block that gives up reports once).  The workspace serves
    the next call each time."""
    from fast_route_b200 import _lib
    M, H, I, E, k = 1, 256, 512, 8, 2
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=5, dtype=torch.bfloat16))
    lib = _lib.load()
    nbytes = lib.fr_moe_decode_workspace_bytes(M, H, I, E, k)
    ws = torch.zeros(nbytes + 1024, dtype=torch.uint8, device=dev)
    ws = ws[(-ws.data_ptr()) % 1024:][:nbytes]
    out = torch.empty_like(x)

    def call():
        """Number of blocks that gave up."""
        assert lib.fr_moe_decode(_lib.ptr(x), _lib.ptr(gate), gate.stride(0), gate.stride(1), _lib.ptr(w1), None, None,
                                 _lib.ptr(w2), None, None, 1, 0, M, H, I, E, k, 1, _lib.ptr(out), None, None,
                                 _lib.ptr(ws), nbytes, _lib.stream_ptr(dev)) == 0
        torch.cuda.synchronize()
        code, _, _, count = _lib.device_status()
        assert (code == 0) == (count == 0) and code in (0, 1)
        return count
    assert call() == 0
    want = out.clone()
    words = ws[:32].view(torch.int32)
    blocks = int(words[1])
    gave_up = {}
    for budget in [1 << i for i in range(12)] + [1 << 20]:
        for _ in range(10):
            words[3] = budget
            gave_up.setdefault(budget, []).append(call())
            words[3] = 0
            out.zero_()
            assert call() == 0 and torch.equal(out, want)
    assert max(gave_up[1]) > 0 and not any(gave_up[1 << 20])
    counts = [c for v in gave_up.values() for c in v]
    assert max(counts) <= blocks and any(0 < c < blocks for c in counts), gave_up
