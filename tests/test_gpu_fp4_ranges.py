"""The product of two 4-bit matrices whose global scales are as large or as small as fp32 allows."""

import numpy as np
import pytest
import torch

import fast_route_b200 as fr
from oracle import fp4 as o

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("ea,eb", [(127, 127), (127, 126), (126, 126), (127, 100), (127, -127), (127, -149), (-126, -126), (-149, -149)])
@pytest.mark.parametrize("m,k", [(3, 256), (3, 2048), (260, 256), (1300, 320)])
def test_global_scales_of_any_size(dev, m, k, ea, eb):
    """Rows of zeros stay zero, results past the output's range are infinite with their sign, the others as exact as ever: half
    a step of the output, k additions in fp32 of 2^-23 of the magnitudes each, two more fp32 roundings for the factor."""
    g = torch.Generator().manual_seed(m + k)
    n = 150

    def matrix(rows):
        q = torch.randint(0, 256, (rows, k // 2), generator=g, dtype=torch.uint8)
        return q, torch.randint(0, 0x7F, (rows, k // 16), generator=g, dtype=torch.uint8)
    (aq, asc), (bq, bsc) = matrix(m), matrix(n)
    aq[1], bq[7] = 0, 0
    ga, gb = torch.tensor([1.3 * 2.0 ** ea]), torch.tensor([2.0 ** eb])
    c = fr.matmul_fp4(aq.to(dev), asc.view(torch.float8_e4m3fn).to(dev), bq.to(dev), bsc.view(torch.float8_e4m3fn).to(dev),
                      ga.to(dev), gb.to(dev)).cpu().double().numpy()
    assert (c[1] == 0).all() and (c[:, 7] == 0).all()
    f = float(ga) * float(gb)
    va, vb = (o.values(q.numpy(), s.numpy(), None, 16) for q, s in ((aq, asc), (bq, bsc)))
    ref, err = f * (va @ vb.T), f * k * 2.0 ** -23 * (np.abs(va) @ np.abs(vb).T)
    top, tiny = float(torch.finfo(torch.bfloat16).max), float(torch.finfo(torch.bfloat16).smallest_normal)
    bound = err + (2.0 ** -8 + 2.0 ** -22) * (np.abs(ref) + err) + tiny * 2.0 ** -8
    past, inside = np.abs(ref) - err > 1.01 * top, np.abs(ref) + bound < top
    assert (c[past] == np.copysign(np.inf, ref[past])).all()
    assert (np.abs(c - ref)[inside] <= bound[inside]).all()
