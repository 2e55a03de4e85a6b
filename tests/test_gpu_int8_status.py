"""The int8 calls' status word against reads that come while it is being written."""

import random
import threading

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_no_report_is_lost_to_a_read_beside_it(cuda_ready):
    """A refused row is reported by a read that ran beside the call, or by the one after it,
    whatever moment the first read fell on."""
    from qmesh_b200 import _lib
    from qmesh_b200.int8 import device_status, quant_int8
    x = torch.full((1, 64), float("nan"), device="cuda")
    q, s = quant_int8(x)
    side = torch.cuda.Stream()
    rng, lost = random.Random(1), 0
    torch.cuda.synchronize()
    device_status()
    for _ in range(1500):
        with torch.cuda.stream(side):
            torch.cuda._sleep(rng.randint(1, 120000))       # up to about 60 us
            quant_int8(x, q=q, scale=s)
        beside = device_status()
        side.synchronize()
        lost += (beside | device_status()) != _lib.QX_DEV_NONFINITE
    assert lost == 0


def test_reads_on_every_stream_clear_once(cuda_ready):
    """One word per device: the first read after a report takes it, on whichever stream."""
    from qmesh_b200 import _lib
    from qmesh_b200.int8 import device_status, quant_int8
    x = torch.full((3, 64), float("inf"), device="cuda")
    device_status()
    quant_int8(x)
    torch.cuda.synchronize()
    with torch.cuda.stream(torch.cuda.Stream()):
        assert device_status() == _lib.QX_DEV_NONFINITE
    assert device_status() == 0


def test_reads_from_many_threads(cuda_ready):
    """More readers at once than the library has words for them: a report goes to exactly one."""
    from qmesh_b200 import _lib
    from qmesh_b200.int8 import device_status, quant_int8
    x = torch.full((1, 64), float("nan"), device="cuda")
    device_status()
    for _ in range(5):
        quant_int8(x)
        torch.cuda.synchronize()
        got = []

        def read():
            with torch.cuda.stream(torch.cuda.Stream()):
                got.append(device_status())

        threads = [threading.Thread(target=read) for _ in range(80)]
        for t in threads:
            t.start()
        for t in threads:
            t.join()
        assert sorted(got) == [0] * 79 + [_lib.QX_DEV_NONFINITE]
