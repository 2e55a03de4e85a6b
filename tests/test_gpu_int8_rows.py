"""The int8 products at more rows than a grid's second dimension counts: rows off 16-byte
boundaries take as many as aligned ones."""

import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("pad", [1, 16])
def test_many_rows(cuda_ready, pad):
    """Whole-number results below 2^24, so FP32 holds them exactly."""
    from qmesh_b200.int8 import int8_matmul, int8_swiglu
    m, n, k = 65536 * 64 + 77, 4, 1
    g = torch.Generator(device="cuda").manual_seed(1)
    q = torch.randint(-127, 128, (m, pad), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    w = torch.randint(-127, 128, (n, pad), generator=g, device="cuda", dtype=torch.int8)[:, :k]
    s = torch.randint(1, 4, (m,), generator=g, device="cuda").float()
    one = torch.ones(n, device="cuda")
    want = q.float() * w.float().t() * s[:, None]
    out = torch.full((m + 1, n), 7.0, device="cuda")
    int8_matmul(q, s, w, one, out=out[:m])
    assert torch.equal(out[:m], want) and (out[m] == 7.0).all()
    # the SwiGLU form: the last rows against the same rows alone
    whole = int8_swiglu(q, s, w, one, out_dtype=torch.float32)
    assert torch.equal(whole[-200:], int8_swiglu(q[-200:], s[-200:], w, one, out_dtype=torch.float32))
    assert torch.equal(whole[:200], int8_swiglu(q[:200], s[:200], w, one, out_dtype=torch.float32))
