"""Bounded waits of the int8 products that run out: the call returns, QX_DEV_TIMEOUT is
recorded, and the calls behind it are right. The wait is made to run out by the library's
test hook (a barrier that expects an arrival which never comes), never by a fault."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def operands(m, n, k):
    g = torch.Generator().manual_seed(m + n + k)
    q, w = (torch.randint(-127, 128, (r, (k + 15) // 16 * 16), generator=g, dtype=torch.int8).cuda()[:, :k]
            for r in (m, n))
    s, ws = (torch.rand(r, generator=g).cuda() + 0.5 for r in (m, n))
    return q, s, w, ws


def check(monkeypatch, hold, m, n, k):
    from qmesh_b200 import _lib
    from qmesh_b200.int8 import device_status, int8_matmul, int8_swiglu
    args = operands(m, n, k)
    want = [fn(*args, out_dtype=torch.float32) for fn in (int8_matmul, int8_swiglu)]
    assert device_status() == 0
    monkeypatch.setenv("QX_TEST_INT8_HOLD", str(hold))
    monkeypatch.setenv("QX_TIMEOUT_MS", "20")
    for fn in (int8_matmul, int8_swiglu):
        fn(*args)
        assert device_status() == _lib.QX_DEV_TIMEOUT
    monkeypatch.delenv("QX_TEST_INT8_HOLD")
    monkeypatch.delenv("QX_TIMEOUT_MS")
    for fn, w in zip((int8_matmul, int8_swiglu), want):
        assert torch.equal(fn(*args, out_dtype=torch.float32), w)
    assert device_status() == 0


@pytest.mark.parametrize("m,n,k", [(1, 4608, 5120), (16, 130, 96), (32, 2304, 640)])
def test_few_token_kernel_sums_never_come(cuda_ready, monkeypatch, m, n, k):
    check(monkeypatch, 1, m, n, k)


@pytest.mark.parametrize("m,n,k", [(40, 300, 2000), (100, 64, 96), (2048, 5120, 2304)])
def test_pair_kernel_sums_never_come(cuda_ready, monkeypatch, m, n, k):
    """With three tiles per pair of CTAs the MMAs come to a stop too, in the middle of a
    ring of copies."""
    check(monkeypatch, 1, m, n, k)


@pytest.mark.parametrize("m,n,k", [(1, 4608, 5120), (16, 130, 96), (32, 2304, 640), (3, 64, 20000),
                                   (40, 300, 2000), (100, 64, 96), (2048, 5120, 2304)])
def test_copies_in_flight_when_the_mmas_give_up(cuda_ready, monkeypatch, m, n, k):
    """Short rings and full ones: what was sent for lands before the CTA leaves, so the next
    call finds its shared memory to itself."""
    check(monkeypatch, 2, m, n, k)
