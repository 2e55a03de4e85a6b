"""The int8 quantiser on FP32 rows, to the bound that its header gives.

q rounds x * c exactly (one fused step into the whole numbers), c = 127 / m rounded once: x c
is within 2^-24 of the quotient t = 127 x / m, relative, so at most 127 * 2^-24 from it, and q
is the rounded quotient unless that is so close to a half.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("rows,k", [(64, 5120), (500, 333), (3, 20003)])
def test_fp32_rounding(cuda_ready, rows, k):
    from qmesh_b200.int8 import quant_int8
    g = torch.Generator().manual_seed(rows + k)
    x = torch.randn(rows, k, generator=g) * torch.exp(4 * torch.randn(rows, 1, generator=g))
    m = x.abs().amax(1, keepdim=True)
    # a fifth of the values next to a half: (n + 1/2) m / 127, moved by up to some 2^-20 of it
    near = (torch.randint(-127, 127, (rows, k), generator=g) + 0.5).double() * m.double() / 127
    near = near * (1 + torch.randn(rows, k, generator=g).double() * 2.0 ** -21)
    pick = (torch.rand(rows, k, generator=g) < 0.2) & (x.abs() < m)
    x = torch.where(pick, near.float(), x)
    q, s = quant_int8(x.cuda())
    m = x.double().abs().amax(1, keepdim=True)
    t = 127.0 * x.double() / m
    off = q.cpu().double() != torch.round(t)
    assert (off & ((t - torch.floor(t) - 0.5).abs() > 127 * 2.0 ** -24 * (1 + 2.0 ** -20))).sum() == 0
    assert (q.cpu().double() - t).abs().max() <= 0.5 + 127 * 2.0 ** -24 * (1 + 2.0 ** -20)
    assert ((s.cpu().double() - m[:, 0] / 127).abs() <= 2.0 ** -24 * m[:, 0] / 127).all()
