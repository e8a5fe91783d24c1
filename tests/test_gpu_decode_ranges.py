"""The 4-bit few-token layer at the ends of its scales' ranges, against the layer in 64 bits with the bound that follows from
the kernel's rounding points (``oracle.fp4.layer_with_bound``)."""

import numpy as np
import pytest
import torch

import fast_route_b200 as fr
from fast_route_b200 import synth
from oracle import fp4 as o

pytestmark = pytest.mark.gpu

E4M3, E8M0 = torch.float8_e4m3fn, torch.float8_e8m0fnu


def _layer(M, H, I, E, block, scale1, scale2, size, seed, dt=torch.bfloat16):
    """Random codes; block scales drawn from the byte ranges; rows of zeros in both matrices; tokens of magnitude ``size``.
    The first element of a token meets zero codes only and decides the routing: expert weights from 1 to e^-30."""
    g = torch.Generator().manual_seed(seed)

    def matrix(rows, cols, scale):
        q = torch.randint(0, 256, (E, rows, cols // 2), generator=g, dtype=torch.uint8)
        s = torch.randint(scale[0], scale[1] + 1, (E, rows, cols // block), generator=g, dtype=torch.uint8)
        return q, s
    q1, s1 = matrix(2 * I, H, scale1)
    q2, s2 = matrix(H, I, scale2)
    q1[:, :, 0] &= 0xF0
    q1[:, 3], q1[:, I + 8], q2[:, 5] = 0, 0, 0
    x = (torch.randn(M, H, generator=g).to(torch.float64) * size).to(dt)
    x[:, 0] = 1.0
    gate = torch.zeros(H, E, dtype=dt)
    gate[0] = torch.linspace(0, -30, E).to(dt)
    return x, gate, q1, s1, q2, s2


def _check(dev, x, gate, q1, s1, q2, s2, block, k, g1=None, g2=None):
    sdt = E4M3 if block == 16 else E8M0
    out, tw, ti = fr.fused_moe_decode_fp4(x.to(dev), gate.to(dev), q1.to(dev), s1.view(sdt).to(dev), q2.to(dev),
                                          s2.view(sdt).to(dev), k, w1_global=None if g1 is None else g1.to(dev),
                                          w2_global=None if g2 is None else g2.to(dev), return_routing=True)
    w1, w2 = (o.values(q.numpy(), s.numpy(), None if g is None else g.double().numpy(), block)
              for q, s, g in ((q1, s1, g1), (q2, s2, g2)))
    ref, err = o.layer_with_bound(x.double().numpy(), w1, w2, ti.cpu().numpy(), tw.cpu().double().numpy(), torch.finfo(x.dtype).eps)
    got = out.cpu().double().numpy()
    top, tiny = float(torch.finfo(x.dtype).max), float(torch.finfo(x.dtype).smallest_normal)
    # The bound is for sums that stay inside fp32 in any order.  That is certain where the sum of the magnitudes of an
    # expert's terms is: no partial sum is larger.  Above it an order exists that overflows, whatever the result: with scales
    # of 2^108 and more in the second matrix magnitudes of 1.0e39 stand behind results of 2.9e38.
    mag = np.zeros_like(ref)
    for t, ids in enumerate(ti.cpu().numpy()):
        for e in ids:
            h = w1[e] @ x[t].double().numpy()
            gate_half, linear = np.split(h, 2)
            mag[t] = np.maximum(mag[t], np.abs(w2[e]) @ np.abs(gate_half / (1 + np.exp(-gate_half)) * linear))
    sure = 1.01 * mag + err < top
    assert sure.any() and np.abs(ref[sure]).max() > 0
    # below the type's normal numbers a rounding is off by at most half of `tiny * eps`: of the output, and of the
    # activations, which the second matrix multiplies
    slack = tiny * torch.finfo(x.dtype).eps * (1 + np.abs(w2).sum(-1).max(0))
    assert (np.abs(got - ref) <= err + slack)[sure].all(), float((np.abs(got - ref) / (err + slack))[sure].max())
    assert (got[:, 5] == 0).all()                    # a row of zeros gives zero, whatever the scales
    return got


@pytest.mark.parametrize("M", [2, 11])
@pytest.mark.parametrize("H,I", [(256, 512), (288, 160)])
@pytest.mark.parametrize("e1,size,e2", [(112, -118, 0), (116, -122, 112), (116, -126, 116), (-110, 104, 116), (-110, 100, -110),
                                        (0, -6, 116), (122, -126, -100), (96, -102, 111)])
def test_global_scales_at_the_ends_of_their_range(dev, M, H, I, e1, size, e2):
    E, k = 4, 3
    x, gate, q1, s1, q2, s2 = _layer(M, H, I, E, 16, (0x20, 0x48), (0x20, 0x38), 2.0 ** size, e1 + M)
    g = torch.Generator().manual_seed(3)
    g1, g2 = ((torch.rand(E, generator=g) * 0.9 + 1).double() * 2.0 ** e for e in (e1, e2))
    _check(dev, x, gate, q1, s1, q2, s2, 16, k, g1.float(), g2.float())


@pytest.mark.parametrize("M", [2, 11])
@pytest.mark.parametrize("H,I", [(256, 512), (288, 160)])
@pytest.mark.parametrize("b1,b2", [(0, 0), (0, 127), (30, 60), (60, 200), (122, 122), (126, 126), (158, 158), (200, 40), (245, 127),
                                   (245, 0), (127, 230), (0, 235)])
def test_power_of_two_scales_of_any_size(dev, M, H, I, b1, b2):
    """Block scales from 2^-127 to 2^125, the tokens such that the first product is of ordinary size."""
    x, gate, q1, s1, q2, s2 = _layer(M, H, I, 4, 32, (b1, b1 + 7), (b2, b2 + 7), 2.0 ** (127 - b1 - 8), b1 + 3 * b2 + M)
    _check(dev, x, gate, q1, s1, q2, s2, 32, 3)


def test_every_code_with_every_power_of_two_scale(dev):
    """One-hot tokens pick single weights of the linear half of w1, and w2 passes silu(1/2) * weight / 2 on.  Rows of w1 have
    every scale up to 2^125, beyond which the largest codes are infinite, columns every code."""
    H, I, n = 128, 256, 253
    code = torch.arange(16, dtype=torch.uint8).repeat(H // 16)
    q1 = torch.full((1, 2 * I, H // 2), 0x22, dtype=torch.uint8)             # 1.0
    q1[0, I:] = code[0::2] | (code[1::2] << 4)
    s1 = torch.full((1, 2 * I, H // 32), 127, dtype=torch.uint8)
    s1[0, I:I + n] = torch.arange(n, dtype=torch.uint8).unsqueeze(1)
    q2 = torch.zeros(1, I, I // 2, dtype=torch.uint8)
    rows = torch.arange(I)
    q2[0, rows, rows // 2] = (2 << (4 * (rows & 1))).to(torch.uint8)
    q2 = torch.cat((q2[:, :H], q2[:, H:]), 0)                                # two experts: the halves of the activations
    q1, s1 = q1.repeat(2, 1, 1), s1.repeat(2, 1, 1)
    s2 = torch.full((2, H, I // 32), 127, dtype=torch.uint8)
    w = o.values(q1.numpy(), s1.numpy(), None, 32)[0]
    silu = 0.5 / (1 + np.exp(-0.5))
    eps, tiny = float(torch.finfo(torch.bfloat16).eps), float(torch.finfo(torch.bfloat16).smallest_normal)
    for col0 in (0, 16, 112):
        x = torch.zeros(16, H, dtype=torch.bfloat16)
        for t in range(16):
            x[t, col0 + t] = 0.5
        for half in (0, 1):
            gate = torch.zeros(H, 2, dtype=torch.bfloat16)
            gate[:, half] = 1
            out = fr.fused_moe_decode_fp4(x.to(dev), gate.to(dev), q1.to(dev), s1.view(E8M0).to(dev), q2.to(dev),
                                          s2.view(E8M0).to(dev), 1)
            want = silu * 0.5 * w[I:, col0:col0 + 16].T[:, H * half:H * half + H]
            # half a step for the activation and for the output, SiLU as in the layer's bound; below normal numbers half
            # of tiny * eps for each
            bound = (eps + 8 * 2.0 ** -23) * np.abs(want) + tiny * eps
            assert (np.abs(out.cpu().double().numpy() - want) <= bound).all()


@pytest.mark.parametrize("M", [6, 13])
@pytest.mark.parametrize("H,I", [(512, 1408), (320, 2080), (1088, 512)])
@pytest.mark.parametrize("value", [0xFF, 170, 254])
def test_scales_beyond_stay_with_their_expert(dev, M, H, I, value):
    """NaN and large scales in one expert: the tokens that go elsewhere keep every bit, also where row tiles are shared."""
    E, k = 8, 2
    x, gate, w1, w2 = (t.to(dev) for t in synth.moe_inputs(M, H, I, E, seed=M + H, dtype=torch.bfloat16, weight_std=0.05))
    q1, s1, _, q2, s2, _ = fr.quantize_experts_fp4(w1, w2, 32)
    run = lambda a, b: fr.fused_moe_decode_fp4(x, gate, q1, a, q2, b, k, return_routing=True)  # noqa: E731
    clean, _, ti = run(s1, s2)
    victim = int(ti[0, 0])
    hit = (ti == victim).any(1)
    assert 0 < int(hit.sum()) < M
    for which in (0, 1):
        for rows in (slice(None), slice(3, None, 7)):
            s = [s1.clone(), s2.clone()]
            s[which].view(torch.uint8)[victim, rows] = value
            out = run(*s)[0]
            assert torch.equal(out[~hit], clean[~hit])
            assert not torch.equal(out[hit], clean[hit])
            if which == 1 and rows.step:          # rows of w2 are rows of the output
                other = [r for r in range(H) if r % 7 != 3]
                assert torch.equal(out[:, other], clean[:, other])
