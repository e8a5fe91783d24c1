"""Quantisation to and from microscaled 4-bit floating point, bit for bit against the 64-bit oracle."""

import numpy as np
import pytest
import torch

import fast_route_b200 as fr
from oracle import fp4 as o

pytestmark = pytest.mark.gpu


def _np(t):
    return t.view(torch.uint8).cpu().numpy()


def _check(x, block, glob=None):
    """Codes, scales and global scale of every matrix, then the numbers they stand for in each type."""
    q, s, g = fr.quantize_fp4(x, block, None if glob is None else glob.to(x.device))
    xs = x.detach().cpu().double().numpy()
    mats = [xs] if x.dim() == 2 else list(xs)
    qs, ss = _np(q).reshape(len(mats), -1, q.shape[-1]), _np(s).reshape(len(mats), -1, s.shape[-1])
    for i, m in enumerate(mats):
        code, sb, gl = o.quantize(m, block, None if glob is None else float(glob[i]))
        assert np.array_equal(ss[i], sb)
        assert np.array_equal(o.unpack(qs[i]), code)
        if block == 16:
            assert float(g[i]) == gl
    assert (g is None) == (block == 32)
    for dt in (torch.float32, torch.bfloat16, torch.float16):
        back = fr.dequantize_fp4(q, s, g, dtype=dt)
        unit = o.e4m3(ss) if block == 16 else o.e8m0(ss)
        if block == 16:
            unit = (unit * g.cpu().double().numpy().reshape(-1, 1, 1)).astype(np.float32).astype(np.float64)
        with np.errstate(over="ignore"):
            v = (o.E2M1[o.unpack(qs)] * np.repeat(unit, block, -1)).astype(np.float32)
        want = torch.from_numpy(v).to(dt).reshape(x.shape)
        assert back.dtype == dt and back.shape == x.shape
        assert torch.equal(back.cpu().nan_to_num(nan=777.0), want.nan_to_num(nan=777.0))
    return q, s, g


@pytest.mark.parametrize("block", [16, 32])
@pytest.mark.parametrize("dt", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(1, 32), (1, 4096), (7, 96), (33, 2080), (1111, 352), (8, 4096), (9, 4096)])
def test_quantize_2d(dev, block, dt, rows, cols):
    g = torch.Generator().manual_seed(rows * 31 + cols)
    x = torch.randn(rows, cols, generator=g)
    x[:, ::13] *= 20.0
    _check(x.to(dt).to(dev), block)


@pytest.mark.parametrize("block", [16, 32])
def test_quantize_3d_strided_and_unaligned(dev, block):
    g = torch.Generator().manual_seed(2)
    base = (torch.randn(3, 10, 200, generator=g) * torch.tensor([1.0, 1e-3, 50.0]).view(3, 1, 1)).to(torch.bfloat16).to(dev)
    _check(base[:, :, :192], block)                       # row pitch larger than the row
    _check(base[:, ::2, 8:104], block)                    # every other row, 16-byte aligned start
    _check(base[:, 1:, 3:99], block)                      # rows start off a 16-byte boundary
    _check(base.transpose(0, 1)[:, :, :64], block)        # matrices interleaved
    _check(base[0, :1].expand(5, 200)[:, :96], block)     # one row read five times
    _check(base.float()[:, :, 1:97], block)


def test_global_scale_given_by_the_caller(dev):
    g = torch.Generator().manual_seed(4)
    x = torch.randn(2, 40, 64, generator=g).to(dev)
    for glob in (torch.tensor([0.01, 3.0]), torch.tensor([1e-30, 1e30]), torch.tensor([2.0 ** -120, 1e-38])):
        got = _check(x, 16, glob)
        assert torch.equal(got[2].cpu(), glob)


@pytest.mark.parametrize("block", [16, 32])
def test_special_values(dev, block):
    x = torch.zeros(6, 64)
    x[1, 5] = float("inf")
    x[1, 40] = -3.0
    x[2, 0] = float("nan")
    x[3, :] = 1e-40                                        # fp32 subnormal
    x[3, 7] = -1e-38
    x[4, ::2] = 6.0
    x[4, 1::2] = torch.tensor([-0.25, 0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0] * 4)      # every tie
    x[5, 0] = 3.0e38
    _check(x.to(dev), block)
    _check(x[:5].contiguous().to(dev), block)
    _check(x[:1].contiguous().to(dev), block)              # zeros: global scale 1, zero codes
    _check(x[3:4].contiguous().to(dev), block)             # nothing but tiny values
    _check(x[2:3, :32].contiguous().to(dev), block)        # no finite block of 32 at all, or one of 16
    big = torch.randn(600, 64)                             # the same through the two-launch path
    big[:6] = x
    big[5] = 0
    _check(big.to(dev), block)


def test_requantising_is_idempotent(dev):
    x = torch.randn(64, 512, generator=torch.Generator().manual_seed(8)).to(dev)
    for block in (16, 32):
        q, s, g = fr.quantize_fp4(x, block)
        back = fr.dequantize_fp4(q, s, g, dtype=torch.float32)
        q2, s2, g2 = fr.quantize_fp4(back, block)
        assert torch.equal(fr.dequantize_fp4(q2, s2, g2, dtype=torch.float32), back)


def test_empty_and_refusals(dev):
    q, s, g = fr.quantize_fp4(torch.empty(0, 64, device=dev))
    assert q.shape == (0, 32) and s.shape == (0, 4) and g.shape == (1,)
    assert fr.dequantize_fp4(q, s, g).shape == (0, 64)
    q, s, g = fr.quantize_fp4(torch.empty(0, 4, 64, device=dev))
    assert q.shape == (0, 4, 32) and g.shape == (0,)
    x = torch.randn(4, 64, device=dev)
    bad = [lambda: fr.quantize_fp4(x[:, :40]), lambda: fr.quantize_fp4(x[:, :48], 32), lambda: fr.quantize_fp4(x, 8),
           lambda: fr.quantize_fp4(x.t()), lambda: fr.quantize_fp4(x.double()), lambda: fr.quantize_fp4(x[0]),
           lambda: fr.quantize_fp4(x, 32, torch.ones(1, device=dev)), lambda: fr.quantize_fp4(x, 16, torch.ones(2, device=dev)),
           lambda: fr.quantize_fp4(x, 16, torch.ones(1, device=dev, dtype=torch.float64)), lambda: fr.quantize_fp4(x[:, :0])]
    q, s, g = fr.quantize_fp4(x)
    bad += [lambda: fr.dequantize_fp4(q, s[:, :2].contiguous(), g), lambda: fr.dequantize_fp4(q, s.float(), g),
            lambda: fr.dequantize_fp4(q.to(torch.int8), s, g), lambda: fr.dequantize_fp4(q[:, ::2], s[:, ::2], g),
            lambda: fr.dequantize_fp4(q, s, g, dtype=torch.float64), lambda: fr.dequantize_fp4(q, s, torch.ones(4, device=dev))]
    for call in bad:
        with pytest.raises(AssertionError):
            call()
    with pytest.raises(RuntimeError):
        fr.quantize_fp4(x, 16, torch.ones(1))


def test_captured_and_on_another_stream(dev):
    x = torch.randn(300, 256, generator=torch.Generator().manual_seed(1)).to(dev)
    want = fr.quantize_fp4(x)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = fr.quantize_fp4(x)
        back = fr.dequantize_fp4(*got)
    y = torch.randn(300, 256, generator=torch.Generator().manual_seed(2)).to(dev) * 7
    x.copy_(y)
    graph.replay()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = fr.quantize_fp4(y)
    torch.cuda.synchronize()
    assert all(torch.equal(a.view(torch.uint8), b.view(torch.uint8)) for a, b in zip(got, again))
    assert torch.equal(back, fr.dequantize_fp4(*again))
    assert not torch.equal(want[0], got[0])
