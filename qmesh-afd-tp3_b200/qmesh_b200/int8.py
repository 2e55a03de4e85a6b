"""W8A8 dense products (qx_quant_int8, qx_int8_matmul): int8 weights with one FP32
scale per output channel, int8 activations with one FP32 scale per token.

* ``quant_int8(x)``: rows of BF16 / FP16 / FP32 values, or the slice's FP8 rows with
  their dequant scale, -> (int8 rows, scale per row). Weights [n, k] are quantised
  with the same call (one scale per row is one per output channel).
* ``int8_matmul(q, scale, w, w_scale)``: [m, n] = (q . w^T) * scale[m] * w_scale[n].
* ``int8_swiglu(q, scale, w13, w13_scale)``: the gate/up product with the clamped
  SwiGLU in its epilogue; w13 holds the gate rows, then the up rows.
* ``Int8Expert``: a dense SwiGLU expert of these parts, the W8A8 form of a shared
  expert (``prefill_slice(shared=)``, ``moe.moe_layer(shared=)``).

The calls launch on the current stream of the tensors' device, never
synchronise the host, and allocate only outputs and workspaces that are not given;
with both given they can be captured in a CUDA graph.
"""

from __future__ import annotations

import ctypes
from contextlib import nullcontext

import torch

from . import _lib
from .trace import rng

SWIGLU_LIMIT = 10.0
OUT_TYPES = {torch.bfloat16: _lib.QX_T_BF16, torch.float16: _lib.QX_T_F16, torch.float32: _lib.QX_T_F32}
X_TYPES = {**OUT_TYPES, torch.float8_e4m3fn: _lib.QX_T_E4M3, torch.uint8: _lib.QX_T_E4M3}


def _p(t: torch.Tensor | None) -> ctypes.c_void_p:
    return ctypes.c_void_p(t.data_ptr() if t is not None else 0)


def _on(dev: torch.device):
    """The tensors' device as the current one (launches go to the current device)."""
    return nullcontext() if dev.index == torch.cuda.current_device() else torch.cuda.device(dev)


def _stream(dev: torch.device) -> ctypes.c_void_p:
    return ctypes.c_void_p(torch.cuda.current_stream(dev).cuda_stream)


def _same_device(dev: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, not on {dev}")


def _rows(t: torch.Tensor, name: str) -> None:
    if t.dim() != 2 or t.shape[1] < 1 or (t.stride(1) != 1 and t.shape[1] > 1):
        raise ValueError(f"{name} must be [rows, columns] with unit column stride, got {tuple(t.shape)}")
    if t.shape[1] > _lib.INT8_MAX_K:
        raise ValueError(f"{name} has {t.shape[1]} columns, at most {_lib.INT8_MAX_K} sum exactly in 32 bits")


def _row_stride(t: torch.Tensor) -> int:
    """Elements between rows (a tensor of one row may carry any stride)."""
    return t.stride(0) if t.shape[0] > 1 else max(t.stride(0), t.shape[1])


def _scales(t: torch.Tensor, n: int, name: str) -> None:
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if t.shape != (n,) or (n > 1 and t.stride(0) != 1):
        raise ValueError(f"{name} must be a contiguous [{n}] tensor, got {tuple(t.shape)}")


def padded(k: int) -> int:
    """Row stride of int8 rows of k values: the next multiple of 16 bytes, which the
    copy engine needs to feed the tensor cores."""
    return (k + 15) // 16 * 16


def _empty_rows(rows: int, k: int, dev) -> torch.Tensor:
    return torch.empty(rows, padded(k), dtype=torch.int8, device=dev)[:, :k]


def quant_int8(x: torch.Tensor, x_scale: torch.Tensor | None = None, q: torch.Tensor | None = None,
               scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(q int8 [rows, k], scale float32 [rows]): x[r] ~ q[r] * scale[r], the largest
    |x| of a row at +-127. A fresh `q` has its rows 16-byte aligned. A row with a NaN
    or an infinity gets q = 0 and scale = NaN, and is reported by `device_status`."""
    if x.dtype not in X_TYPES:
        raise TypeError(f"x must be bf16, fp16, fp32 or e4m3, got {x.dtype}")
    _rows(x, "x")
    if not x.is_cuda:
        raise ValueError("x must be on a CUDA device")
    rows, k, dev = x.shape[0], x.shape[1], x.device
    fp8 = X_TYPES[x.dtype] == _lib.QX_T_E4M3
    if fp8 and x_scale is None:
        raise TypeError("FP8 activations need x_scale (per row [rows] or per post [1])")
    if x_scale is not None and not fp8:
        raise TypeError("x_scale goes with FP8 activations only")
    if fp8:
        if x_scale.dtype != torch.float32:
            raise TypeError(f"x_scale must be float32, got {x_scale.dtype}")
        if x_scale.numel() not in (1, rows) or not x_scale.is_contiguous():
            raise ValueError(f"x_scale has {x_scale.numel()} values for {rows} rows")
    if q is None:
        q = _empty_rows(rows, k, dev)
    if scale is None:
        scale = torch.empty(rows, dtype=torch.float32, device=dev)
    if q.dtype != torch.int8:
        raise TypeError(f"q must be int8, got {q.dtype}")
    _rows(q, "q")
    if q.shape != x.shape:
        raise ValueError(f"q is {tuple(q.shape)}, x {tuple(x.shape)}")
    _scales(scale, rows, "scale")
    _same_device(dev, x_scale=x_scale, q=q, scale=scale)
    with _on(dev), rng("qx.quant_int8"):
        rc = _lib.load().qx_quant_int8(_p(x), _row_stride(x), X_TYPES[x.dtype], _p(x_scale),
                                       x_scale.numel() if fp8 else 0, rows, k, _p(q), _row_stride(q), _p(scale),
                                       _stream(dev))
    _lib.check(rc, "qx_quant_int8")
    return q, scale


def _product(q, scale, w, w_scale, out, out_dtype, swiglu, limit) -> torch.Tensor:
    if q.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError(f"q and w must be int8, got {q.dtype}/{w.dtype}")
    _rows(q, "q")
    _rows(w, "w")
    if not q.is_cuda:
        raise ValueError("q must be on a CUDA device")
    m, k, dev = q.shape[0], q.shape[1], q.device
    if w.shape[0] < 1 or w.shape[1] != k or (swiglu and w.shape[0] % 2):
        raise ValueError(f"shape mismatch: q {tuple(q.shape)} w {tuple(w.shape)}")
    n = w.shape[0] // 2 if swiglu else w.shape[0]
    _scales(scale, m, "scale")
    _scales(w_scale, w.shape[0], "w_scale")
    if out is None:
        if out_dtype not in OUT_TYPES:
            raise TypeError(f"out_dtype must be bf16, fp16 or fp32, got {out_dtype}")
        out = torch.empty(m, n, dtype=out_dtype, device=dev)
    if out.dtype not in OUT_TYPES:
        raise TypeError(f"out must be bf16, fp16 or fp32, got {out.dtype}")
    if out.shape != (m, n) or (out.stride(1) != 1 and n > 1):
        raise ValueError(f"out must be [{m}, {n}] with unit column stride, got {tuple(out.shape)}")
    _same_device(dev, scale=scale, w=w, w_scale=w_scale, out=out)
    args = _lib.QxInt8Args(_p(q), _row_stride(q), _p(scale), _p(w), _row_stride(w), _p(w_scale), _p(out),
                           _row_stride(out), OUT_TYPES[out.dtype], m, n, k, 1 if swiglu else 0,
                           1 if swiglu and limit > 0 else 0, float(max(limit, 0.0)))
    with _on(dev), rng("qx.int8_matmul"):
        rc = _lib.load().qx_int8_matmul(ctypes.byref(args), _stream(dev))
    _lib.check(rc, "qx_int8_matmul")
    return out


def int8_matmul(q: torch.Tensor, scale: torch.Tensor, w: torch.Tensor, w_scale: torch.Tensor,
                out: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """[m, n] of `out`'s type (or out_dtype): ((q . w^T) * scale[:, None]) * w_scale,
    q int8 [m, k], w int8 [n, k]; the whole-number sums are exact. `out` must not
    overlap the inputs."""
    return _product(q, scale, w, w_scale, out, out_dtype, False, 0.0)


def int8_swiglu(q: torch.Tensor, scale: torch.Tensor, w13: torch.Tensor, w13_scale: torch.Tensor,
                swiglu_limit: float = SWIGLU_LIMIT, out: torch.Tensor | None = None,
                out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """[m, n] = silu(min(g, L)) * clamp(u, -L, L) of the products g, u with w13's first
    n rows (gate) and last n rows (up); L = swiglu_limit, no clamp for L <= 0."""
    return _product(q, scale, w13, w13_scale, out, out_dtype, True, swiglu_limit)


def device_status(device=None) -> int:
    """QX_DEV_* bits (NONFINITE, TIMEOUT) that this module's calls recorded on `device`
    since the last read (synchronises and clears)."""
    dev = torch.device("cuda", torch.cuda.current_device()) if device is None else torch.device(device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    st = ctypes.c_uint32(0)
    with _on(dev):
        _lib.check(_lib.load().qx_int8_status(ctypes.byref(st), _stream(dev)), "qx_int8_status")
    return int(st.value)


class Int8Expert:
    """A dense SwiGLU expert in 8 bits: q = quant(x); h = swiglu(q . w13^T) in FP32;
    q2 = quant(h); y = q2 . w2^T. w13 int8 [2 inter, k] (gate rows, then up rows), w2
    int8 [k, inter], one FP32 scale per row of each."""

    def __init__(self, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor,
                 swiglu_limit: float = SWIGLU_LIMIT):
        if w13.dtype != torch.int8 or w2.dtype != torch.int8:
            raise TypeError(f"w13 and w2 must be int8, got {w13.dtype}/{w2.dtype}")
        _rows(w13, "w13")
        _rows(w2, "w2")
        if w13.shape[0] % 2 or w13.shape[0] < 2 or w2.shape != (w13.shape[1], w13.shape[0] // 2):
            raise ValueError(f"shape mismatch: w13 {tuple(w13.shape)} w2 {tuple(w2.shape)}")
        _scales(w13_scale, w13.shape[0], "w13_scale")
        _scales(w2_scale, w2.shape[0], "w2_scale")
        self.dev = w13.device
        _same_device(self.dev, w13_scale=w13_scale, w2=w2, w2_scale=w2_scale)
        self.w13, self.w13_scale, self.w2, self.w2_scale = w13, w13_scale, w2, w2_scale
        self.k, self.inter = w13.shape[1], w13.shape[0] // 2
        self.limit = float(swiglu_limit)

    @classmethod
    def from_weights(cls, w13: torch.Tensor, w2: torch.Tensor, swiglu_limit: float = SWIGLU_LIMIT) -> "Int8Expert":
        """Quantise BF16 / FP16 / FP32 weights, one scale per output channel."""
        return cls(*quant_int8(w13), *quant_int8(w2), swiglu_limit=swiglu_limit)

    def _layout(self, rows: int) -> tuple[list[int], int]:
        """Byte offsets of q, scale, h, q2, scale2 for `rows` rows, and the total."""
        offs, o = [], 0
        for n in (rows * padded(self.k), rows * 4, rows * self.inter * 4, rows * padded(self.inter), rows * 4):
            offs.append(o)
            o += (n + 255) // 256 * 256
        return offs, o

    def workspace_bytes(self, rows: int) -> int:
        return self._layout(rows)[1]

    def alloc_workspace(self, rows: int) -> torch.Tensor:
        """Workspace for calls of up to `rows` rows. Calls that may overlap on the GPU
        (two streams, two graphs in flight at once) need one each."""
        return torch.empty(self.workspace_bytes(rows), dtype=torch.uint8, device=self.dev)

    def __call__(self, x: torch.Tensor, x_scale: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """[rows, k] of `out`'s type (or out_dtype) for x [rows, k] (bf16, fp16, fp32, or
        e4m3 with x_scale)."""
        if x.dim() != 2 or x.shape[1] != self.k:
            raise ValueError(f"x must be [rows, {self.k}], got {tuple(x.shape)}")
        _same_device(self.dev, x=x, out=out, workspace=workspace)
        rows = x.shape[0]
        (o_q, o_s, o_h, o_q2, o_s2), need = self._layout(rows)
        if workspace is None:
            workspace = torch.empty(need, dtype=torch.uint8, device=self.dev)
        if workspace.dtype != torch.uint8 or workspace.dim() != 1 or not workspace.is_contiguous():
            raise TypeError("workspace must be a contiguous uint8 tensor (alloc_workspace)")
        if workspace.numel() < need:
            raise ValueError(f"workspace has {workspace.numel()} bytes, {rows} rows need {need}")
        if workspace.data_ptr() % 16:
            raise ValueError("workspace must be 16-byte aligned")

        def part(off: int, r: int, c: int, dtype: torch.dtype) -> torch.Tensor:
            n = r * c * dtype.itemsize
            return workspace[off:off + n].view(dtype).view(r, c)

        q = part(o_q, rows, padded(self.k), torch.int8)[:, :self.k]
        s = part(o_s, rows, 1, torch.float32)[:, 0]
        h = part(o_h, rows, self.inter, torch.float32)
        q2 = part(o_q2, rows, padded(self.inter), torch.int8)[:, :self.inter]
        s2 = part(o_s2, rows, 1, torch.float32)[:, 0]
        quant_int8(x, x_scale, q=q, scale=s)
        int8_swiglu(q, s, self.w13, self.w13_scale, self.limit, out=h)
        quant_int8(h, q=q2, scale=s2)
        return int8_matmul(q2, s2, self.w2, self.w2_scale, out=out, out_dtype=out_dtype)
