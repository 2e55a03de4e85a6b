"""Refusals of the W8A8 calls, without a GPU: the C entries' argument checks come
before any device work, and the Python calls check types and shapes first."""

import ctypes

import pytest
import torch


@pytest.fixture(scope="module")
def lib():
    from qmesh_b200 import _lib, build
    build.build()
    return _lib.load()


def _mm(lib, **kw):
    from qmesh_b200 import _lib
    base = dict(a=64, a_stride=128, a_scale=64, w=64, w_stride=128, w_scale=64, out=64, out_stride=32, out_type=0,
                m=4, n=32, k=128, swiglu=0, has_limit=0, limit=0.0)
    base.update(kw)
    args = _lib.QxInt8Args(*[base[f[0]] for f in _lib.QxInt8Args._fields_])
    return lib.qx_int8_matmul(ctypes.byref(args), None)


def test_matmul_refusals(lib):
    from qmesh_b200 import _lib
    assert lib.qx_int8_matmul(None, None) == _lib.QX_ERR_ARG
    for name in ("a", "w", "a_scale", "w_scale", "out"):
        assert _mm(lib, **{name: 0}) == _lib.QX_ERR_ARG
    assert _mm(lib, m=-1) == _mm(lib, n=0) == _mm(lib, k=0) == _lib.QX_ERR_SHAPE
    assert _mm(lib, k=_lib.INT8_MAX_K + 1, a_stride=1 << 20, w_stride=1 << 20) == _lib.QX_ERR_SHAPE
    assert _mm(lib, a_stride=127) == _mm(lib, w_stride=127) == _mm(lib, out_stride=31) == _lib.QX_ERR_SHAPE
    assert _mm(lib, out_type=3) == _mm(lib, out_type=-1) == _lib.QX_ERR_ARG
    assert _mm(lib, out=65) == _mm(lib, out=66, out_type=2) == _mm(lib, a_scale=66) == _lib.QX_ERR_ALIGN
    assert _mm(lib, m=0, a=0, out=0) == _lib.QX_OK


def _quant(lib, **kw):
    base = dict(x=64, x_stride=128, x_type=0, x_scale=0, n_scale=0, rows=4, k=128, q=64, q_stride=128, scale=64)
    base.update(kw)
    return lib.qx_quant_int8(*[base[k] for k in ("x", "x_stride", "x_type", "x_scale", "n_scale", "rows", "k", "q",
                                                 "q_stride", "scale")], None)


def test_quantiser_refusals(lib):
    from qmesh_b200 import _lib
    assert _quant(lib, x=0) == _quant(lib, q=0) == _quant(lib, scale=0) == _lib.QX_ERR_ARG
    assert _quant(lib, x_type=4) == _quant(lib, x_type=3) == _lib.QX_ERR_ARG
    assert _quant(lib, x_type=3, x_scale=64, n_scale=2) == _lib.QX_ERR_ARG
    assert _quant(lib, k=0) == _quant(lib, rows=-1) == _quant(lib, x_stride=127) == _lib.QX_ERR_SHAPE
    assert _quant(lib, q_stride=127) == _quant(lib, k=_lib.INT8_MAX_K + 1) == _lib.QX_ERR_SHAPE
    assert _quant(lib, x=65) == _quant(lib, x=66, x_type=2) == _quant(lib, scale=66) == _lib.QX_ERR_ALIGN
    assert _quant(lib, rows=0, x=0) == _lib.QX_OK


def test_python_refusals():
    from qmesh_b200 import int8
    q, w = torch.zeros(2, 32, dtype=torch.int8), torch.zeros(6, 32, dtype=torch.int8)
    s, ws = torch.ones(2), torch.ones(6)
    with pytest.raises(TypeError):
        int8.quant_int8(torch.zeros(2, 32, dtype=torch.float64))
    with pytest.raises(ValueError):
        int8.quant_int8(torch.zeros(2, 32))                       # not on a GPU
    with pytest.raises(ValueError):
        int8.quant_int8(torch.zeros(32))
    with pytest.raises(TypeError):
        int8.int8_matmul(q.float(), s, w, ws)
    with pytest.raises(ValueError):
        int8.int8_matmul(q, s, w, ws)                             # not on a GPU
    with pytest.raises(ValueError):
        int8.Int8Expert(w, ws, torch.zeros(32, 4, dtype=torch.int8), torch.ones(32))   # inter 3, not 4
    with pytest.raises(TypeError):
        int8.Int8Expert(w, ws.double(), torch.zeros(32, 3, dtype=torch.int8), torch.ones(32))
    ex = int8.Int8Expert(w, ws, torch.zeros(32, 3, dtype=torch.int8), torch.ones(32))
    with pytest.raises(ValueError):
        ex(torch.zeros(2, 31))
    with pytest.raises(ValueError):
        ex(torch.zeros(2, 32), workspace=torch.zeros(8, dtype=torch.uint8))
