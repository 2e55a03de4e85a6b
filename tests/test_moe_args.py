"""Refusals of the whole MoE layer, without a GPU."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from qmesh_b200 import _lib, build
    build.build()
    return _lib.load()


def _call(lib, router=None, arena=None, **kw):
    from qmesh_b200 import _lib
    base = dict(x=16, x_scale=16, x_stride=10240, x_fmt=_lib.QX_X_BF16, ids=0, ids_int64=0, tw=0, rows=2, topk=6,
                c0=0, c1=256, swiglu_limit=10.0, has_limit=1, out=16, out_stride=5120, workspace=256,
                workspace_bytes=1 << 30)
    base.update(kw)
    args = _lib.QxSliceArgs(*[base[f[0]] for f in _lib.QxSliceArgs._fields_])
    a = dict(w13=16, w2=16, g13=16, g2=16, n_experts=8, a0=0, a1=256, layout=_lib.QX_LAYOUT_TC)
    a.update(arena or {})
    ar = _lib.QxArena(*[a[f[0]] for f in _lib.QxArena._fields_])
    r = dict(gate=16, gate_type=0, gate_stride=5120, bias=0, ids=0, tw=0, addend=0, addend_stride=0)
    r.update(router or {})
    rt = _lib.QxRouterArgs(*[r[f[0]] for f in _lib.QxRouterArgs._fields_])
    return lib.qx_moe_decode_tc(ctypes.byref(ar), ctypes.byref(args), ctypes.byref(rt), None, None)


def test_refusals(lib):
    from qmesh_b200 import _lib
    assert lib.qx_moe_decode_tc(None, None, None, None, None) == _lib.QX_ERR_ARG
    assert _call(lib, {"gate": 0}) == _call(lib, {"gate_type": 1}) == _lib.QX_ERR_ARG
    assert _call(lib, {"gate_stride": 5119}) == _lib.QX_ERR_SHAPE
    assert _call(lib, {"gate": 24}) == _call(lib, {"gate_stride": 5124}) == _lib.QX_ERR_ALIGN
    assert _call(lib, {"bias": 18}) == _call(lib, {"ids": 17}) == _call(lib, {"tw": 18}) == _lib.QX_ERR_ALIGN
    assert _call(lib, {"addend": 16, "addend_stride": 5000}) == _lib.QX_ERR_SHAPE
    assert _call(lib, {"addend": 20, "addend_stride": 5120}) == _lib.QX_ERR_ALIGN
    assert _call(lib, arena={"n_experts": 5}) == _lib.QX_ERR_SHAPE          # fewer experts than slots
    assert _call(lib, arena={"n_experts": 4097}) == _call(lib, rows=65) == _call(lib, topk=9) == _lib.QX_ERR_SHAPE
    assert _call(lib, rows=0) == _call(lib, topk=0) == _lib.QX_ERR_SHAPE
    assert _call(lib, arena={"layout": _lib.QX_LAYOUT_FRAG}) == _lib.QX_ERR_ARG
    assert _call(lib, x_fmt=_lib.QX_X_E4M3, x_scale=0) == _lib.QX_ERR_ARG
    assert _call(lib, workspace_bytes=lib.qx_slice_workspace_tc_bytes(2, 6, 0, 256)) == _lib.QX_ERR_WORKSPACE
    need = lib.qx_moe_workspace_bytes(2, 8, 6, 0, 256)
    assert need == lib.qx_slice_workspace_tc_bytes(2, 6, 0, 256) + 4 * 2 * 8 * 4 + 2 * 6 * 8
    assert lib.qx_moe_workspace_bytes(2, 5, 6, 0, 256) == lib.qx_moe_workspace_bytes(65, 8, 6, 0, 256) == 0


def test_python_refusals(lib):
    from qmesh_b200.arena import Arena
    from qmesh_b200.moe import moe_layer, workspace_bytes
    from oracle import moe
    x = torch.zeros(2, 5120, dtype=torch.bfloat16)
    gate = torch.zeros(8, 5120, dtype=torch.bfloat16)
    ar = Arena("cpu", 1, 8, 0, 64)
    with pytest.raises(RuntimeError):
        moe_layer(ar, 0, x, gate)                       # layer not loaded
    ar.load_layer(0, moe.random_code_layer(8, torch.Generator().manual_seed(0), inter=64))
    for bad, err in ((dict(gate=gate.half()), TypeError), (dict(gate=gate[:7]), ValueError),
                     (dict(bias=torch.zeros(7)), TypeError), (dict(bias=torch.zeros(8).double()), TypeError),
                     (dict(ids=torch.zeros(2, 6, dtype=torch.int64)), TypeError),
                     (dict(tw=torch.zeros(2, 5)), TypeError), (dict(), ValueError)):   # not on a GPU
        with pytest.raises(err):
            moe_layer(ar, 0, x, **{"gate": gate, **bad})
    with pytest.raises(ValueError):
        moe_layer(Arena("cpu", 1, 8, 0, 64, layout="frag"), 0, x, gate)
    with pytest.raises(ValueError):
        workspace_bytes(0, 8, 6, 0, 64)
