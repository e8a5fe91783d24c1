"""The product of two 4-bit block-scaled matrices against the product in 64 bits of the numbers the codes stand for.

Bound per element: half a step of the output type, and what adding k terms in fp32 (one step, 2^-23, of the running sum's
magnitude per addition, whether the hardware rounds or truncates) can lose: k * 2^-23 * sum |a| |b|.  The products of
codes and of scales are exact in fp32."""

import numpy as np
import pytest
import torch

import fast_route_b200 as fr
from oracle import fp4 as o

pytestmark = pytest.mark.gpu


def _matrix(g, block, rows, k, wide=False):
    q = torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8)
    if block == 16:
        s = torch.randint(0 if wide else 0x30, 0x7F if wide else 0x48, (rows, k // 16), generator=g, dtype=torch.uint8)
        return q, s, torch.rand(1, generator=g) + 0.5
    s = torch.randint(97 if wide else 122, 157 if wide else 132, (rows, k // 32), generator=g, dtype=torch.uint8)
    return q, s, None


def _dev(t, dev):
    q, s, g = t
    return q.to(dev), s.to(dev).view(torch.float8_e4m3fn if g is not None else torch.float8_e8m0fnu), None if g is None else g.to(dev)


def _ref(a, b, block, k):
    ga, gb = (None if t[2] is None else float(t[2]) for t in (a, b))
    va, vb = (o.values(t[0].numpy(), t[1].numpy(), None, block) for t in (a, b))
    f = (ga or 1.0) * (gb or 1.0)
    return f * (va @ vb.T), f * k * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T)


def _check(c, ref, err):
    eps = torch.finfo(c.dtype).eps
    # alpha is one fp32 product and one multiplication more
    bound = err + (eps / 2 + 2.0 ** -22) * (np.abs(ref) + err) + float(torch.finfo(c.dtype).smallest_normal) * eps
    big = np.abs(ref) > float(torch.finfo(c.dtype).max)
    got = c.detach().cpu().double().numpy()
    assert (np.abs(got - ref)[~big] <= bound[~big]).all(), float((np.abs(got - ref) / bound)[~big].max())


SHAPES = [(1, 128, 32), (1, 4096, 4096), (5, 1, 64), (32, 100, 96), (33, 257, 2080), (1, 20000, 512), (128, 512, 256),
          (129, 300, 320), (333, 1399, 2080), (300, 512, 4096), (1000, 264, 160), (2049, 1000, 288), (64, 3000, 1056),
          (1300, 4100, 32), (16, 16, 8192)]


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m,n,k", SHAPES)
def test_product(dev, block, m, n, k):
    g = torch.Generator().manual_seed(m * 7 + n + k)
    a, b = _matrix(g, block, m, k), _matrix(g, block, n, k)
    (aq, asc, ag), (bq, bsc, bg) = _dev(a, dev), _dev(b, dev)
    ref, err = _ref(a, b, block, k)
    dt = torch.bfloat16 if (m + n) % 2 else torch.float16
    c = fr.matmul_fp4(aq, asc, bq, bsc, ag, bg, dtype=dt)
    _check(c, ref, err)
    assert torch.equal(c, fr.matmul_fp4(aq, asc, bq, bsc, ag, bg, dtype=dt))


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m", [3, 100, 200])
def test_every_scale_is_placed_right(dev, block, m):
    """One non-zero code per row of b in every K block in turn, scales over their whole range: a scale that belongs to
    another row, block or step shows."""
    k, n = 1056, 300
    g = torch.Generator().manual_seed(m + block)
    a, b = _matrix(g, block, m, k, wide=True), _matrix(g, block, n, k, wide=True)
    q = torch.zeros_like(b[0])
    rows = torch.arange(n)
    at = (rows * 37 + 11) % k
    q[rows, at // 2] = torch.where(at % 2 == 0, 2, 32).to(torch.uint8)       # 1.0 at one position per row
    b = (q, b[1], b[2])
    (aq, asc, ag), (bq, bsc, bg) = _dev(a, dev), _dev(b, dev)
    ref, err = _ref(a, b, block, k)
    _check(fr.matmul_fp4(aq, asc, bq, bsc, ag, bg), ref, err)


@pytest.mark.parametrize("ea,eb", [(-70, -72), (-30, -100), (-110, -60), (100, 60), (90, -110), (110, -149)])
@pytest.mark.parametrize("m,k", [(3, 256), (3, 2048), (100, 2048), (260, 256), (260, 2048)])
def test_global_scales_whose_product_leaves_fp32(dev, m, k, ea, eb):
    """Results inside the output's range are as exact as ever, results past it are infinite, and rows of zeros stay zero."""
    g = torch.Generator().manual_seed(m + k)
    n = 150
    (aq, asc, _), (bq, bsc, _) = _matrix(g, 16, m, k, wide=True), _matrix(g, 16, n, k, wide=True)
    aq[1] = 0
    a, b = (aq, asc, torch.tensor([1.3 * 2.0 ** ea])), (bq, bsc, torch.tensor([1.0 * 2.0 ** eb]))
    ref, err = _ref(a, b, 16, k)
    (aq, asc, ag), (bq, bsc, bg) = _dev(a, dev), _dev(b, dev)
    c = fr.matmul_fp4(aq, asc, bq, bsc, ag, bg)
    assert (c[1] == 0).all()
    _check(c, ref, err)
    top = float(torch.finfo(c.dtype).max)
    sure = torch.from_numpy(np.abs(ref) - err > 1.01 * top)
    assert torch.isinf(c.cpu()[sure]).all()


@pytest.mark.parametrize("m,n,k,pitch,lo", [(1111, 5001, 544, 5001, 0), (1111, 5000, 544, 5007, 3), (200, 263, 96, 264, 1),
                                            (2500, 2049, 1024, 2050, 0)])
def test_large_outputs_whose_rows_start_anywhere(dev, m, n, k, pitch, lo):
    g = torch.Generator().manual_seed(n)
    a, b = _matrix(g, 32, m, k), _matrix(g, 32, n, k)
    (aq, asc, _), (bq, bsc, _) = _dev(a, dev), _dev(b, dev)
    buf = torch.full((m + 2, pitch), 7.0, dtype=torch.bfloat16, device=dev)
    out = buf[1:m + 1, lo:lo + n]
    fr.matmul_fp4(aq, asc, bq, bsc, out=out)
    _check(out, *_ref(a, b, 32, k))
    out.fill_(7.0)
    assert (buf == 7.0).all()


@pytest.mark.parametrize("m", [7, 90, 260])
def test_out_with_a_pitch_and_what_lies_around_it(dev, m):
    g = torch.Generator().manual_seed(5)
    n, k = 200, 256
    a, b = _matrix(g, 16, m, k), _matrix(g, 16, n, k)
    (aq, asc, ag), (bq, bsc, bg) = _dev(a, dev), _dev(b, dev)
    want = fr.matmul_fp4(aq, asc, bq, bsc, ag, bg)
    for lo, pitch in ((0, 208), (3, 211), (8, 216)):
        buf = torch.full((m + 2, pitch), 7.0, dtype=torch.bfloat16, device=dev)
        out = buf[1:m + 1, lo:lo + n]
        got = fr.matmul_fp4(aq, asc, bq, bsc, ag, bg, out=out)
        assert got.data_ptr() == out.data_ptr() and torch.equal(out, want)
        out.fill_(7.0)
        assert (buf == 7.0).all()


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m", [4, 300])
def test_nan_scales_stay_in_their_row(dev, block, m):
    g = torch.Generator().manual_seed(6)
    n, k = 150, 512
    a, b = _matrix(g, block, m, k), _matrix(g, block, n, k)
    nan = 0x7F if block == 16 else 0xFF
    clean = fr.matmul_fp4(*_dev(a, dev)[:2], *_dev(b, dev)[:2])
    a[1][1, 3] = nan
    b[1][70, 5] = nan
    c = fr.matmul_fp4(*_dev(a, dev)[:2], *_dev(b, dev)[:2])
    bad = torch.zeros(m, n, dtype=torch.bool, device=dev)
    bad[1], bad[:, 70] = True, True
    assert torch.isnan(c[bad]).all() and torch.equal(c[~bad], clean[~bad])


def test_quantise_then_multiply(dev):
    """The two operators as a user runs them: the result is the product of what the quantised matrices stand for, and near
    the product of the originals (each element off by at most a quarter of itself or of its block's smallest step)."""
    g = torch.Generator().manual_seed(7)
    x, w = torch.randn(70, 1024, generator=g).to(dev), torch.randn(600, 1024, generator=g).to(dev) * 0.02
    for block in (16, 32):
        a, b = fr.quantize_fp4(x, block), fr.quantize_fp4(w, block)
        c = fr.matmul_fp4(a[0], a[1], b[0], b[1], a[2], b[2])
        va, vb = (fr.dequantize_fp4(*t, dtype=torch.float32).double() for t in (a, b))
        ref = va @ vb.t()
        _check(c, ref.cpu().numpy(), (1024 * 2.0 ** -23 * (va.abs() @ vb.abs().t())).cpu().numpy() * 1.01)
        rel = (c.double() - x.double() @ w.double().t()).norm() / (x.double() @ w.double().t()).norm()
        assert rel < 0.25


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("m", [9, 70, 200])
def test_scales_that_start_anywhere(dev, block, m):
    g = torch.Generator().manual_seed(10)
    n, k = 140, 608                                     # scale rows of 38 or 19 bytes
    a, b = _matrix(g, block, m, k), _matrix(g, block, n, k)
    (aq, asc, _), (bq, bsc, _) = _dev(a, dev), _dev(b, dev)
    want = fr.matmul_fp4(aq, asc, bq, bsc)
    for off in (1, 2, 4):
        moved = []
        for s in (asc, bsc):
            buf = torch.zeros(s.numel() + 16, dtype=torch.uint8, device=dev)
            buf[off:off + s.numel()] = s.view(torch.uint8).flatten()
            moved.append(buf[off:off + s.numel()].view(s.dtype).view(s.shape))
        assert torch.equal(fr.matmul_fp4(aq, moved[0], bq, moved[1]), want)


def test_empty_and_refusals(dev):
    g = torch.Generator().manual_seed(8)
    aq, asc, ag = _dev(_matrix(g, 16, 6, 64), dev)
    bq, bsc, bg = _dev(_matrix(g, 16, 10, 64), dev)
    mq, msc, _ = _dev(_matrix(g, 32, 10, 64), dev)
    assert fr.matmul_fp4(aq[:0], asc[:0], bq, bsc).shape == (0, 10)
    assert fr.matmul_fp4(aq, asc, bq[:0], bsc[:0]).shape == (6, 0)
    hq, hsc, _ = _dev(_matrix(g, 16, 10, 48), dev)
    out = torch.empty(6, 10, dtype=torch.bfloat16, device=dev)
    bad = [lambda: fr.matmul_fp4(aq, asc, mq, msc), lambda: fr.matmul_fp4(aq, asc, bq[:, :16].contiguous(), bsc[:, :2].contiguous()),
           lambda: fr.matmul_fp4(hq, hsc, hq, hsc), lambda: fr.matmul_fp4(aq, asc, bq, bsc, dtype=torch.float32),
           lambda: fr.matmul_fp4(aq, asc, bq, bsc, out=out.float()), lambda: fr.matmul_fp4(aq, asc, bq, bsc, out=out.t()),
           lambda: fr.matmul_fp4(aq, asc, bq, bsc, out=out[:5]), lambda: fr.matmul_fp4(aq, asc, bq, bsc, out=out[:1].expand(6, 10)),
           lambda: fr.matmul_fp4(aq, asc, bq, bsc, torch.ones(2, device=dev)), lambda: fr.matmul_fp4(mq, msc, mq, msc, torch.ones(1, device=dev)),
           lambda: fr.matmul_fp4(aq.view(2, 3, 32), asc.view(2, 3, 4), bq, bsc)]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(RuntimeError):
        fr.matmul_fp4(aq, asc, bq.cpu(), bsc)


@pytest.mark.parametrize("m", [2, 150, 700])
def test_captured(dev, m):
    g = torch.Generator().manual_seed(9)
    (aq, asc, ag), (bq, bsc, bg) = _dev(_matrix(g, 16, m, 512), dev), _dev(_matrix(g, 16, 384, 512), dev)
    want = fr.matmul_fp4(aq, asc, bq, bsc, ag, bg)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c = fr.matmul_fp4(aq, asc, bq, bsc, ag, bg)
        d = fr.matmul_fp4(aq, asc, bq, bsc, ag, bg)
    for _ in range(3):
        c.zero_()
        d.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c, want) and torch.equal(d, want)
