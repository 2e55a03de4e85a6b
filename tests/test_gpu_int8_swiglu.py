"""The SwiGLU of the int8 products to the last places of FP32, against 64 bits.

Bound. g and u are within D = 3 * 2^-24 (1 + 2^-22) of the 64-bit products (an exact sum,
one conversion, two multiplications). silu(g) = g / (1 + exp(-g)) moves by at most
(1 + |g|) D with g; expf and the quotient are documented within 2 units of their last places
(4 * 2^-24 each), and the sum and the product with u round once each: with u's own D that
is ((1 + |g|) + 1) D + 10 * 2^-24, plus half a step of the output's type.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
D = 3 * U * (1 + 2.0 ** -22)


def check(out, g, u, dtype):
    want = g / (1 + torch.exp(-g)) * u
    eps = torch.finfo(dtype).eps / 2
    rel = (2 + g.abs()) * D + 10 * U
    tol = (rel + eps * (1 + rel)) * want.abs() + torch.finfo(dtype).smallest_normal * eps
    err = (out.double().cpu() - want).abs()
    assert (err <= tol).all(), f"worst {float((err / tol.clamp_min(1e-300)).max()):.3f} x tolerance"


@pytest.mark.parametrize("m,n,k", [(1, 700, 512), (6, 333, 1000), (32, 64, 5120), (40, 333, 512), (300, 700, 1000),
                                   (7, 65, 333)])
@pytest.mark.parametrize("pad", [16, 1])
def test_fp32_outputs(cuda_ready, m, n, k, pad):
    """Aligned rows and others, gates of every size the clamp lets through."""
    from qmesh_b200.int8 import int8_swiglu
    g = torch.Generator().manual_seed(m + n + k)
    width = (k + pad - 1) // pad * pad + (pad == 1)
    q, w = (torch.randint(-127, 128, (r, width), generator=g, dtype=torch.int8)[:, :k] for r in (m, 2 * n))
    s, ws = torch.rand(m, generator=g) + 0.5, (torch.rand(2 * n, generator=g) + 0.5) * 6e-4 / k ** 0.5
    h = (q.double() @ w.double().T) * s.double()[:, None] * ws.double()
    out = int8_swiglu(q.cuda(), s.cuda(), w.cuda(), ws.cuda(), swiglu_limit=0.0, out_dtype=torch.float32)
    check(out, h[:, :n], h[:, n:], torch.float32)


@pytest.mark.parametrize("m", [1, 20, 50, 300])
@pytest.mark.parametrize("pad", [0, 1])
def test_gates_whose_sigmoid_is_small(cuda_ready, m, pad):
    """Gates down to -88.5: the sigmoid is below 2^-126 there, the product with the gate is
    still a normal number of FP32 and BF16."""
    from qmesh_b200.int8 import int8_swiglu
    n, k = 128, 32
    q = torch.zeros(m, k + pad, dtype=torch.int8)[:, :k]
    w = torch.zeros(2 * n, k + pad, dtype=torch.int8)[:, :k]
    q[:, 0], q[:, 1] = 100, torch.arange(m) % 100 + 1
    w[:n, 0], w[n:, 1] = -100, (torch.arange(n) % 127 + 1).to(torch.int8)
    gate = torch.linspace(-88.5, -60.0, n)
    s, ws = torch.ones(m), torch.cat([gate / -10000.0, torch.full((n,), 0.01)])
    h = (q.double() @ w.double().T) * ws.double()
    assert h[:, :n].min() < -88.4
    for dtype in (torch.float32, torch.bfloat16):
        out = int8_swiglu(q.cuda(), s.cuda(), w.cuda(), ws.cuda(), swiglu_limit=10.0, out_dtype=dtype)
        check(out, h[:, :n], h[:, n:].clamp(-10, 10), dtype)
        assert (out != 0).all()


@pytest.mark.parametrize("m", [1, 40])
def test_zero_and_far_gates(cuda_ready, m):
    """Zero gates give zero, gates past FP32's exp give zero, large ones pass through."""
    from qmesh_b200.int8 import int8_swiglu
    n, k = 96, 16
    q, w = torch.zeros(m, k, dtype=torch.int8), torch.zeros(2 * n, k, dtype=torch.int8)
    q[:, 0], w[:n, 0], w[n:, 0] = 1, (torch.arange(n) % 3 - 1).to(torch.int8), 2
    out = int8_swiglu(q.cuda(), torch.full((m,), 100.0).cuda(), w.cuda(), torch.ones(2 * n).cuda(), swiglu_limit=0.0,
                      out_dtype=torch.float32).cpu()
    assert torch.equal(out, torch.tensor([0.0, 0.0, 20000.0]).repeat(n // 3).expand(m, n))
