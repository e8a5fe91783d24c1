"""The few-token layer against the layer evaluated in 64 bits, element by element, with a bound that is computed from
the kernel's rounding points (``oracle.fp4.layer_with_bound``)."""

import numpy as np
import pytest
import torch

import fast_route_b200 as fr
import oracle
from fast_route_b200 import synth
from oracle import fp4 as o

pytestmark = pytest.mark.gpu


def _d(t):
    return t.detach().cpu().double().numpy()


def _check_routing(x, gate, k, tw, ti, renormalize=True):
    """Ids and weights follow from logits that are within fp32 accumulation of the exact ones."""
    xd, gd = _d(x), _d(gate)
    logits = xd @ gd
    tol = (xd.shape[1] + 8) * 2.0 ** -24 * (np.abs(xd) @ np.abs(gd))
    ids, w = ti.cpu().numpy(), tw.cpu().double().numpy()
    for t in range(xd.shape[0]):
        assert len(set(ids[t])) == k and ids[t].min() >= 0 and ids[t].max() < gd.shape[1]
        sel = logits[t, ids[t]]
        slack = 2 * tol[t].max()
        assert (sel[:-1] >= sel[1:] - slack).all()                     # descending
        rest = np.delete(logits[t], ids[t])
        assert rest.size == 0 or rest.max() <= sel[-1] + slack         # nothing larger was left out
        den = np.exp((sel if renormalize else logits[t]) - sel[0]).sum()
        want = np.exp(sel - sel[0]) / den
        # logits off by `slack` at most, the recipe's exponential and sums a few fp32 roundings per term
        assert np.allclose(w[t], want, rtol=2 * slack + (gd.shape[1] + 16) * 2.0 ** -24, atol=1e-37)


def _check(x, gate, w1, w2, k, dev, run, w1_exact=None, w2_exact=None, renormalize=True):
    out, tw, ti = run()
    torch.cuda.synchronize()
    _check_routing(x, gate, k, tw, ti, renormalize)
    eps = torch.finfo(x.dtype).eps
    ref, err = o.layer_with_bound(_d(x), _d(w1) if w1_exact is None else w1_exact,
                                  _d(w2) if w2_exact is None else w2_exact, ti.cpu().numpy(), tw.cpu().double().numpy(), eps)
    off = np.abs(_d(out) - ref)
    tiny = torch.finfo(x.dtype).smallest_normal                        # subnormal outputs and activations
    assert (off <= err + tiny * (1 + np.abs(ref).max())).all(), float((off / (err + 1e-30)).max())
    return out, tw, ti


CASES = [(1, 256, 256, 8, 2), (2, 64, 32, 4, 1), (3, 2048, 352, 16, 4), (5, 512, 1408, 64, 6), (8, 1024, 96, 8, 8),
         (9, 8, 8, 4, 2), (16, 264, 520, 60, 8), (16, 4096, 128, 3, 3), (7, 40, 2056, 256, 5), (16, 128, 64, 128, 1),
         (1, 5128, 72, 2, 1), (13, 1000, 1000, 7, 3)]


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("M,H,I,E,k", CASES)
def test_decode_16bit(dev, M, H, I, E, k, dt):
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=M + H, dtype=dt, weight_std=0.05))
    first = _check(x, gate, w1, w2, k, dev, lambda: fr.fused_moe_decode(x, gate, w1, w2, k, return_routing=True))
    again = fr.fused_moe_decode(x, gate, w1, w2, k, return_routing=True)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    # the layer for any batch: same routing, outputs within the sum of both layers' rounding
    out, tw, ti = fr.fused_moe(x, gate, w1, w2, k, return_routing=True)
    assert (ti == first[2]).float().mean() > 0.97


@pytest.mark.parametrize("M,H,I,E,k", [(1, 256, 256, 8, 2), (4, 2048, 96, 16, 4), (16, 352, 1408, 64, 6), (9, 32, 32, 4, 2),
                                       (16, 4096, 160, 5, 5), (3, 1056, 544, 128, 7)])
@pytest.mark.parametrize("block,dt", [(16, torch.bfloat16), (16, torch.float16), (32, torch.bfloat16)])
def test_decode_fp4(dev, M, H, I, E, k, block, dt):
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=M + I, dtype=dt, weight_std=0.05))
    q1, s1, g1, q2, s2, g2 = fr.quantize_experts_fp4(w1, w2, block)
    u8 = lambda t: t.view(torch.uint8).cpu().numpy()  # noqa: E731
    gl = lambda g: None if g is None else g.cpu().double().numpy()  # noqa: E731
    e1, e2 = o.values(u8(q1), u8(s1), gl(g1), block), o.values(u8(q2), u8(s2), gl(g2), block)
    run = lambda: fr.fused_moe_decode_fp4(x, gate, q1, s1, q2, s2, k, w1_global=g1, w2_global=g2, return_routing=True)  # noqa: E731
    first = _check(x, gate, None, None, k, dev, run, e1, e2)
    assert all(torch.equal(a, b) for a, b in zip(first, run()))


@pytest.mark.parametrize("block,dt", [(16, torch.bfloat16), (16, torch.float16), (32, torch.bfloat16)])
def test_every_code_with_every_scale(dev, block, dt):
    """One-hot activations pick single weights: GEMM1 rows get every block scale, the columns every code, and w2 (ones on
    the diagonal) passes silu(weight) * 1 on, so each expanded weight is seen by itself."""
    n_scale = 127 if block == 16 else 94           # E4M3 0 .. 448; E8M0 2^-60 .. 2^33: the documented range
    H, I = 128, 128
    code = torch.arange(16, dtype=torch.uint8).repeat(H // 16)
    q1 = torch.zeros(1, 2 * I, H // 2, dtype=torch.uint8)
    q1[0, :I] = code[0::2] | (code[1::2] << 4)
    q1[0, I:] = 0x22                               # 1.0
    base = 0 if block == 16 else 67
    s1 = torch.zeros(1, 2 * I, H // block, dtype=torch.uint8)
    s1[0, :n_scale] = (torch.arange(n_scale, dtype=torch.uint8) + base).unsqueeze(1)
    s1[0, I:] = 0x38 if block == 16 else 127       # 1.0
    q2 = torch.zeros(1, H, I // 2, dtype=torch.uint8)
    for i in range(I):
        q2[0, i, i // 2] = 2 << (4 * (i & 1))
    s2 = torch.full((1, H, I // block), 0x38 if block == 16 else 127, dtype=torch.uint8)
    sdt = torch.float8_e4m3fn if block == 16 else torch.float8_e8m0fnu
    gate = torch.zeros(H, 1, dtype=dt, device=dev)
    for col0 in (0, 16, 112):
        x = torch.zeros(16, H, dtype=dt)
        for t in range(16):
            x[t, col0 + t] = 0.5
        out = fr.fused_moe_decode_fp4(x.to(dev), gate, q1.to(dev), s1.view(sdt).to(dev), q2.to(dev), s2.view(sdt).to(dev), 1)
        w = o.values(q1.numpy(), s1.numpy(), None, block)[0]
        g, u = w[:I, col0:col0 + 16].T * 0.5, 0.5
        act = g / (1 + np.exp(-np.minimum(np.maximum(g, -700), 700))) * u
        got = out.cpu().double().numpy()
        eps = torch.finfo(dt).eps
        big = torch.finfo(dt).max
        ok = np.abs(act) < big / 2
        assert ok.all() if block == 16 else ok.any()
        # half a step of rounding for each of the two products; the fast exponential is documented to be within
        # 2 + 1.173 |g| units in the last place (2^-23) and the fast division within 2; the division gives 0 where
        # 1 + exp(-g) passes 2^126, that is g < -87.3: what is lost there is at most 88 * 2^-126
        bound = (eps + (6 + 1.2 * np.minimum(np.abs(g), 90)) * 2.0 ** -23) * np.abs(act)
        bound += max(float(torch.finfo(dt).smallest_normal) * eps, 88 * 2.0 ** -126)
        assert (np.abs(got - act)[ok] <= bound[ok]).all()


def test_nan_and_infinite_weights_stay_with_their_expert(dev):
    M, H, I, E, k = 6, 256, 192, 8, 2
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=3, dtype=torch.bfloat16, weight_std=0.05))
    clean, tw, ti = fr.fused_moe_decode(x, gate, w1, w2, k, return_routing=True)
    victim = int(ti[0, 0])
    hit = (ti == victim).any(1)
    assert 0 < int(hit.sum()) < M
    for name, bad in (("w2", float("nan")), ("w2", float("inf")), ("w1", float("nan")), ("w1", float("-inf"))):
        a, b = w1.clone(), w2.clone()
        (a if name == "w1" else b)[victim, 5, 7] = bad
        out = fr.fused_moe_decode(x, gate, a, b, k)
        assert torch.equal(out[~hit], clean[~hit])
        assert not torch.isfinite(out[hit].float()).all()
    # an expert nobody chose
    idle = next(e for e in range(E) if not (ti == e).any())
    w1[idle], w2[idle] = float("nan"), float("nan")
    assert torch.equal(fr.fused_moe_decode(x, gate, w1, w2, k), clean)
    # one token's NaN stays with that token
    y = x.clone()
    y[2, 9] = float("nan")
    out = fr.fused_moe_decode(y, gate, w1.nan_to_num(0), w2.nan_to_num(0), k)
    keep = [t for t in range(M) if t != 2]
    assert torch.equal(out[keep], clean[keep])


@pytest.mark.parametrize("H,I", [(264, 200), (1000, 1000), (72, 520)])
def test_infinities_past_the_end_of_a_row(dev, H, I):
    """Row lengths that end inside a step, an infinity in the first elements: no NaN comes of a product with the filling."""
    M, E, k = 3, 2, 2
    g = torch.Generator().manual_seed(4)
    for dt in (torch.bfloat16, torch.float16):
        x = torch.rand(M, H, generator=g).to(dt)
        w1, w2 = torch.rand(E, 2 * I, H, generator=g).to(dt) * 0.01, torch.rand(E, H, I, generator=g).to(dt) * 0.01 + 0.01
        w1 += 0.01                                         # every weight positive: an infinity stays one
        x[1, 5] = float("inf")
        gate = torch.zeros(H, E, dtype=dt)                 # both experts, half each, for finite and infinite tokens alike
        gate[:, 0] = 0
        out = fr.fused_moe_decode(x.to(dev), gate.to(dev), w1.to(dev), w2.to(dev), k).cpu()
        assert torch.isfinite(out[[0, 2]]).all()
        assert torch.isinf(out[1]).all() and (out[1] > 0).all()


def test_nan_scales_stay_with_their_expert(dev):
    M, H, I, E, k = 6, 256, 192, 8, 2
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=3, dtype=torch.bfloat16, weight_std=0.05))
    for block in (16, 32):
        q1, s1, g1, q2, s2, g2 = fr.quantize_experts_fp4(w1, w2, block)
        run = lambda a, b: fr.fused_moe_decode_fp4(x, gate, q1, a, q2, b, k, w1_global=g1, w2_global=g2)  # noqa: E731
        clean = run(s1, s2)
        ti = fr.fused_moe_decode(x, gate, w1, w2, k, return_routing=True)[2]
        victim = int(ti[0, 0])
        hit = (ti == victim).any(1)
        for which in (0, 1):
            s = [s1.clone(), s2.clone()]
            s[which].view(torch.uint8)[victim, 3, 2] = 0x7F if block == 16 else 0xFF
            out = run(*s)
            assert torch.equal(out[~hit], clean[~hit])
            assert torch.isnan(out[hit].float()).any()


def test_ties_go_to_the_lower_expert(dev):
    """Equal logits: a gate of repeated columns, so that whole groups of experts tie exactly."""
    M, H, I, E, k = 5, 64, 32, 96, 7
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=5, dtype=torch.bfloat16, weight_std=0.05))
    gate = gate[:, :8].repeat(1, 12)
    _, tw, ti = fr.fused_moe_decode(x, gate, w1, w2, k, return_routing=True)
    logits = (x.double() @ gate.double()).cpu()
    want = torch.argsort(logits, dim=1, descending=True, stable=True)[:, :k]
    assert torch.equal(ti.cpu().long(), want)
    assert torch.allclose(tw.cpu(), torch.full_like(tw.cpu(), 1 / 7), rtol=1e-5)
    zero = fr.fused_moe_decode(torch.zeros_like(x), gate, w1, w2, k, return_routing=True)
    assert torch.equal(zero[2].cpu(), torch.arange(k, dtype=torch.int32).expand(M, k)) and not zero[0].any()


@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16])
def test_options(dev, dt):
    M, H, I, E, k = 4, 320, 224, 12, 3
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=9, dtype=dt, weight_std=0.05))
    base = fr.fused_moe_decode(x, gate, w1, w2, k)
    # a row-major gate, a gate with a pitch that is no multiple of 8, a gate off a 16-byte boundary
    wide = torch.zeros(H, E + 1, dtype=dt, device=dev)
    wide[:, :E] = gate
    odd = torch.zeros(E, H + 3, dtype=dt, device=dev)
    odd[:, 1:H + 1] = gate.t()
    for g in (gate.contiguous(), wide[:, :E], odd[:, 1:H + 1].t()):
        assert torch.equal(fr.fused_moe_decode(x, g, w1, w2, k), base)
    _check(x, gate, w1, w2, k, dev, lambda: fr.fused_moe_decode(x, gate, w1, w2, k, renormalize=False, return_routing=True),
           renormalize=False)
    y = x.clone()
    same = fr.fused_moe_decode(y, gate, w1, w2, k, inplace=True)
    assert same.data_ptr() == y.data_ptr() and torch.equal(y, base)
    assert fr.fused_moe_decode(x[:0], gate, w1, w2, k).shape == (0, H)
    # k = E: every expert
    _check(x, gate, w1, w2, E, dev, lambda: fr.fused_moe_decode(x, gate, w1, w2, E, return_routing=True))


def test_refusals(dev):
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(17, 64, 32, 4, seed=1, dtype=torch.bfloat16))
    q = fr.quantize_experts_fp4(w1, w2)
    m = fr.quantize_experts_fp4(w1, w2, 32)
    x1 = x[:2].contiguous()
    call4 = lambda xx, p, **kw: fr.fused_moe_decode_fp4(xx, gate, p[0], p[1], p[3], p[4], 2, **kw)  # noqa: E731
    bad = [lambda: fr.fused_moe_decode(x, gate, w1, w2, 2), lambda: fr.fused_moe_decode(x1, gate, w1, w2, 5),
           lambda: fr.fused_moe_decode(x1, gate, w1, w2, 0), lambda: fr.fused_moe_decode(x1.float(), gate, w1, w2, 2),
           lambda: fr.fused_moe_decode(x1, gate.half(), w1, w2, 2), lambda: fr.fused_moe_decode(x1[:, ::2], gate, w1, w2, 2),
           lambda: fr.fused_moe_decode(x1, gate, w1[:, :, :32], w2, 2), lambda: fr.fused_moe_decode(x1, gate[:32], w1, w2, 2),
           lambda: fr.fused_moe_decode(x1, gate, w1, w2[:, :, :16].contiguous(), 2),
           lambda: call4(x, q), lambda: call4(x1.half(), m), lambda: call4(x1, (q[0], m[1], q[2], q[3], q[4])),
           lambda: call4(x1, (q[0], q[1], q[2], m[3], m[4])), lambda: call4(x1, m, w1_global=torch.ones(4, device=dev)),
           lambda: call4(x1, q, w1_global=torch.ones(3, device=dev))]
    for f in bad:
        with pytest.raises(AssertionError):
            f()
    with pytest.raises(RuntimeError):
        fr.fused_moe_decode(x1, gate.cpu(), w1, w2, 2)
    # sizes whose rows are no multiple of 16 bytes
    for H, I in ((60, 32), (64, 28)):
        xx, gg, a, b = (t.to(dev) for t in synth.moe_inputs(1, H, I, 4, seed=1, dtype=torch.bfloat16))
        with pytest.raises(RuntimeError):
            fr.fused_moe_decode(xx, gg, a, b, 2)


def test_graphs_and_streams(dev):
    """Two captured layers replayed side by side on two streams while eager calls run on a third: no shared scratch."""
    M, H, I, E, k = 3, 512, 384, 16, 4
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=11, dtype=torch.bfloat16, weight_std=0.05))
    xs = [x, x.flip(0).contiguous() * 1.5, x.roll(1, 0).contiguous() * 0.5]
    want = [fr.fused_moe_decode(v, gate, w1, w2, k) for v in xs]
    graphs, outs = [], []
    for v in xs[:2]:
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            outs.append(fr.fused_moe_decode(v, gate, w1, w2, k))
        graphs.append(graph)
    streams = [torch.cuda.Stream() for _ in range(3)]
    torch.cuda.synchronize()
    for rep in range(5):
        for o_ in outs:
            o_.zero_()
        torch.cuda.synchronize()
        # one after the other on the GPU (cooperative launches fill it), in any order the streams give
        for i, graph in enumerate(graphs):
            with torch.cuda.stream(streams[i]):
                graph.replay()
        with torch.cuda.stream(streams[2]):
            eager = fr.fused_moe_decode(xs[2], gate, w1, w2, k)
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[0]) and torch.equal(outs[1], want[1]) and torch.equal(eager, want[2])


@pytest.mark.reads_status
def test_a_wait_that_runs_out_is_reported(dev):
    """The wait for the other CTAs' activations is bounded: with the barrier's base moved up by one it can never be
    satisfied, so it ends after the poll budget written into the control words, and the status block says so.  A zeroed
    workspace serves the next call."""
    from fast_route_b200 import _lib
    M, H, I, E, k = 2, 256, 128, 4, 2
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=2, dtype=torch.bfloat16))
    lib = _lib.load()
    nbytes = lib.fr_moe_decode_workspace_bytes(M, H, I, E, k)
    ws = torch.zeros(nbytes + 1024, dtype=torch.uint8, device=dev)
    ws = ws[(-ws.data_ptr()) % 1024:][:nbytes]
    out = torch.empty_like(x)

    def call():
        return lib.fr_moe_decode(_lib.ptr(x), _lib.ptr(gate), gate.stride(0), gate.stride(1), _lib.ptr(w1), None, None,
                                 _lib.ptr(w2), None, None, 1, 0, M, H, I, E, k, 1, _lib.ptr(out), None, None, _lib.ptr(ws),
                                 nbytes, _lib.stream_ptr(dev))
    assert call() == 0
    torch.cuda.synchronize()
    assert _lib.device_status()[0] == 0
    want = out.clone()
    words = ws[:32].view(torch.int32)
    assert int(words[0]) == int(words[1]) > 0 and int(words[2]) == 0 and int(words[4]) == 1
    words[1] += 1                              # base
    words[3] = 2000                            # polls
    assert call() == 0
    torch.cuda.synchronize()
    code, detail, _, count = _lib.device_status()
    assert code == 1 and detail == 0x802 and count > 0
    ws.zero_()
    assert call() == 0
    torch.cuda.synchronize()
    assert _lib.device_status()[0] == 0 and torch.equal(out, want)


@pytest.mark.parametrize("polls", [1, 3, 10, 30, 100])
def test_a_wait_that_runs_out_in_some_blocks_leaves_the_workspace_usable(dev, polls):
    """With few polls some thread blocks give up and others do not.  Whatever the mixture, the same workspace serves the
    next call: H = 256 has several blocks per row range of the second product, whose counters end at zero."""
    from fast_route_b200 import _lib
    M, H, I, E, k = 3, 256, 512, 8, 2
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=5, dtype=torch.bfloat16))
    lib = _lib.load()
    nbytes = lib.fr_moe_decode_workspace_bytes(M, H, I, E, k)
    ws = torch.zeros(nbytes + 1024, dtype=torch.uint8, device=dev)
    ws = ws[(-ws.data_ptr()) % 1024:][:nbytes]
    out = torch.empty_like(x)

    def call():
        assert lib.fr_moe_decode(_lib.ptr(x), _lib.ptr(gate), gate.stride(0), gate.stride(1), _lib.ptr(w1), None, None,
                                 _lib.ptr(w2), None, None, 1, 0, M, H, I, E, k, 1, _lib.ptr(out), None, None,
                                 _lib.ptr(ws), nbytes, _lib.stream_ptr(dev)) == 0
        torch.cuda.synchronize()
        return _lib.device_status()[0]
    assert call() == 0
    want = out.clone()
    words, counters = ws[:32].view(torch.int32), ws[256:256 + 4 * 128].view(torch.int32)
    for _ in range(20):
        words[3] = polls
        assert call() in (0, 1)
        assert int(words[0]) == int(words[1]) and int(words[2]) == 0
        assert int(counters.abs().sum()) == 0
        words[3] = 0
        out.zero_()
        assert call() == 0
        assert torch.equal(out, want)


@pytest.mark.parametrize("block,dt", [(16, torch.bfloat16), (32, torch.bfloat16)])
@pytest.mark.parametrize("H,I", [(32, 32), (96, 160), (544, 224), (64, 2080)])
def test_scales_that_start_anywhere(dev, H, I, block, dt):
    """Row lengths and tensor offsets that leave the scale rows without any alignment, equal to the aligned result."""
    M, E, k = 5, 3, 2
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=H + I, dtype=dt, weight_std=0.05))
    q1, s1, g1, q2, s2, g2 = fr.quantize_experts_fp4(w1, w2, block)
    want = fr.fused_moe_decode_fp4(x, gate, q1, s1, q2, s2, k, w1_global=g1, w2_global=g2)
    for off in (1, 2, 3, 4, 8):
        moved = []
        for s in (s1, s2):
            buf = torch.zeros(s.numel() + 16, dtype=torch.uint8, device=dev)
            buf[off:off + s.numel()] = s.view(torch.uint8).flatten()
            moved.append(buf[off:off + s.numel()].view(s.dtype).view(s.shape))
        assert torch.equal(fr.fused_moe_decode_fp4(x, gate, q1, moved[0], q2, moved[1], k, w1_global=g1, w2_global=g2), want)


def test_many_calls_of_changing_size_share_one_workspace(dev):
    """Sizes, formats and numbers of tokens in turn on one stream: what one call leaves behind never reaches the next."""
    cases = []
    for i, (M, H, I, E, k) in enumerate([(1, 256, 512, 4, 2), (16, 512, 96, 32, 6), (3, 2048, 64, 8, 1), (9, 64, 1024, 200, 4),
                                         (16, 1024, 256, 8, 8), (2, 4096, 32, 3, 2)]):
        x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=i, dtype=torch.bfloat16, weight_std=0.05))
        cases.append((x, gate, w1, w2, k, fr.quantize_experts_fp4(w1, w2)))

    def go(c):
        x, gate, w1, w2, k, q = c
        return (fr.fused_moe_decode(x, gate, w1, w2, k),
                fr.fused_moe_decode_fp4(x, gate, q[0], q[1], q[3], q[4], k, w1_global=q[2], w2_global=q[5]))
    want = [go(c) for c in cases]
    order = np.random.default_rng(0).integers(0, len(cases), 60)
    got = [(i, go(cases[i])) for i in order]
    for i, (a, b) in got:
        assert torch.equal(a, want[i][0]) and torch.equal(b, want[i][1])


def test_decode_and_prompt_through_the_same_quantised_experts(dev):
    """As a server uses them together: experts quantised once, the prompt through fused_moe on the expanded weights (exact
    in bf16 but for the rounding of the global scale), the following tokens through the few-token layer."""
    H, I, E, k = 512, 320, 16, 4
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(200, H, I, E, seed=13, dtype=torch.bfloat16, weight_std=0.05))
    for block in (16, 32):
        q1, s1, g1, q2, s2, g2 = fr.quantize_experts_fp4(w1, w2, block)
        e1, e2 = fr.dequantize_fp4(q1, s1, g1), fr.dequantize_fp4(q2, s2, g2)
        prompt = fr.fused_moe(x, gate, e1, e2, k)
        for lo in range(0, 200, 16):
            part = fr.fused_moe_decode_fp4(x[lo:lo + 16], gate, q1, s1, q2, s2, k, w1_global=g1, w2_global=g2)
            d = (part.float() - prompt[lo:lo + 16].float()).abs()
            # a few bf16 half-steps of the outputs' size: the expanded weights' rounding and both layers' own
            assert d.max() <= 2.0 ** -8 * 8 * prompt.float().abs().max()
