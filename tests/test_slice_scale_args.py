"""The FP8 dequant scales of a slice call, without a GPU: the kernels read them one behind
the other, so scales that lie apart are refused."""

import pytest
import torch


def test_scales_that_lie_apart_are_refused():
    from qmesh_b200.expert_slice import _slice_args
    rows = 4
    x = torch.zeros(rows, 5120, dtype=torch.float8_e4m3fn)
    out, ws = torch.zeros(rows, 5120, dtype=torch.bfloat16), torch.zeros(16, dtype=torch.uint8)
    ids, tw = torch.zeros(rows, 6, dtype=torch.int32), torch.zeros(rows, 6)
    wide = torch.rand(rows, 3)

    def call(scale, topk=None):
        a = (None, None) if topk else (ids, tw)
        return _slice_args(x, *a, out, 0, 64, ws, scale, 10.0, True, topk=topk)

    for topk in (None, 6):                                  # given ids; the whole MoE layer
        for bad in (wide[:, 0], wide[:, 1:2], wide[:1, 0].expand(rows)):
            with pytest.raises(ValueError):
                call(bad, topk)
        for good in (wide[:, 0].contiguous(), wide[:, 0].contiguous()[:, None], wide[:1, 0], wide[2, 1:2]):
            assert call(good, topk).x_scale == good.data_ptr()
