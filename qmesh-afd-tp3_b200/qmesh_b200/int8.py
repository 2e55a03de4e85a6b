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

import torch

from . import _lib, trace
from .trace import rng

SWIGLU_LIMIT = 10.0
OUT_TYPES = {torch.bfloat16: _lib.QX_T_BF16, torch.float16: _lib.QX_T_F16, torch.float32: _lib.QX_T_F32}
X_TYPES = {**OUT_TYPES, torch.float8_e4m3fn: _lib.QX_T_E4M3, torch.uint8: _lib.QX_T_E4M3}

# The current stream's handle without building a Stream object (2 us of a call that
# can take 8 on the device); the public route where this torch has no such function.
_raw_stream = getattr(torch._C, "_cuda_getCurrentRawStream", None) or (
    lambda index: torch.cuda.current_stream(index).cuda_stream)


def launch_on(dev: torch.device, fn, what: str, *args) -> None:
    """Call the C entry `fn(*args, stream)` on the current stream of `dev`, with `dev` as
    the current device, and raise on its status."""
    if dev.index == torch.cuda.current_device():
        if trace.ENABLED:
            with rng(what):
                rc = fn(*args, _raw_stream(dev.index))
        else:
            rc = fn(*args, _raw_stream(dev.index))
    else:
        with torch.cuda.device(dev), rng(what):
            rc = fn(*args, _raw_stream(dev.index))
    if rc:
        _lib.check(rc, what)


def same_device(dev: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.device != dev:
            raise ValueError(f"{name} is on {t.device}, not on {dev}")
    if dev.type != "cuda":
        raise ValueError(f"the tensors must be on a CUDA device, not on {dev}")


def _rows(t: torch.Tensor, name: str) -> tuple[int, int, int]:
    """(rows, columns, elements between rows) of a [rows, columns] tensor with unit
    column stride (a tensor of one row may carry any row stride)."""
    shape, stride = t.shape, t.stride()
    if len(shape) != 2 or shape[1] < 1 or (stride[1] != 1 and shape[1] > 1):
        raise ValueError(f"{name} must be [rows, columns] with unit column stride, got {tuple(shape)}")
    rows, cols = shape
    if cols > _lib.INT8_MAX_K:
        raise ValueError(f"{name} has {cols} columns, at most {_lib.INT8_MAX_K} sum exactly in 32 bits")
    return rows, cols, stride[0] if rows > 1 or stride[0] > cols else cols


def _scales(t: torch.Tensor, n: int, name: str) -> None:
    if t.dtype != torch.float32:
        raise TypeError(f"{name} must be float32, got {t.dtype}")
    if t.dim() != 1 or t.numel() != n or (n > 1 and t.stride()[0] != 1):
        raise ValueError(f"{name} must be a contiguous [{n}] tensor, got {tuple(t.shape)}")


def padded(k: int) -> int:
    """Row stride of int8 rows of k values: the next multiple of 16 bytes, which the
    copy engine needs to feed the tensor cores."""
    return (k + 15) // 16 * 16


def _check_x(x: torch.Tensor, x_scale: torch.Tensor | None) -> tuple[int, int, int, int, int, int]:
    """(rows, columns, row stride, QX_T_*, scale pointer, scale count) of activations x
    with their scale (FP8 only)."""
    kind = X_TYPES.get(x.dtype)
    if kind is None:
        raise TypeError(f"x must be bf16, fp16, fp32 or e4m3, got {x.dtype}")
    rows, k, stride = _rows(x, "x")
    if kind != _lib.QX_T_E4M3:
        if x_scale is not None:
            raise TypeError("x_scale goes with FP8 activations only")
        return rows, k, stride, kind, 0, 0
    if x_scale is None:
        raise TypeError("FP8 activations need x_scale (per row [rows] or per post [1])")
    if x_scale.dtype != torch.float32:
        raise TypeError(f"x_scale must be float32, got {x_scale.dtype}")
    if x_scale.numel() not in (1, rows) or not x_scale.is_contiguous():
        raise ValueError(f"x_scale has {x_scale.numel()} values for {rows} rows")
    return rows, k, stride, kind, x_scale.data_ptr(), x_scale.numel()


def _check_out(out: torch.Tensor, m: int, n: int) -> tuple[int, int]:
    """(row stride, QX_T_*) of an output tensor."""
    kind = OUT_TYPES.get(out.dtype)
    if kind is None:
        raise TypeError(f"out must be bf16, fp16 or fp32, got {out.dtype}")
    shape, stride = out.shape, out.stride()
    if len(shape) != 2 or shape[0] != m or shape[1] != n or (n > 1 and stride[1] != 1):
        raise ValueError(f"out must be [{m}, {n}] with unit column stride, got {tuple(shape)}")
    return stride[0] if m > 1 or stride[0] > n else n, kind


def _new_out(m: int, n: int, dtype: torch.dtype, dev) -> torch.Tensor:
    if dtype not in OUT_TYPES:
        raise TypeError(f"out_dtype must be bf16, fp16 or fp32, got {dtype}")
    return torch.empty(m, n, dtype=dtype, device=dev)


def quant_int8(x: torch.Tensor, x_scale: torch.Tensor | None = None, q: torch.Tensor | None = None,
               scale: torch.Tensor | None = None) -> tuple[torch.Tensor, torch.Tensor]:
    """(q int8 [rows, k], scale float32 [rows]): x[r] ~ q[r] * scale[r], the largest
    |x| of a row at +-127. A fresh `q` has its rows 16-byte aligned. A row with a NaN
    or an infinity gets q = 0 and scale = NaN, and is reported by `device_status`."""
    rows, k, stride, kind, scale_ptr, n_scale = _check_x(x, x_scale)
    dev = x.device
    same_device(dev, x_scale=x_scale, q=q, scale=scale)
    if q is None:
        q = torch.empty(rows, padded(k), dtype=torch.int8, device=dev)[:, :k]
    if scale is None:
        scale = torch.empty(rows, dtype=torch.float32, device=dev)
    if q.dtype != torch.int8:
        raise TypeError(f"q must be int8, got {q.dtype}")
    q_rows, q_k, q_stride = _rows(q, "q")
    if q_rows != rows or q_k != k:
        raise ValueError(f"q is {tuple(q.shape)}, x {tuple(x.shape)}")
    _scales(scale, rows, "scale")
    launch_on(dev, _lib.load().qx_quant_int8, "qx_quant_int8", x.data_ptr(), stride, kind, scale_ptr, n_scale, rows, k,
              q.data_ptr(), q_stride, scale.data_ptr())
    return q, scale


def _product(q, scale, w, w_scale, out, out_dtype, swiglu, limit) -> torch.Tensor:
    if q.dtype != torch.int8 or w.dtype != torch.int8:
        raise TypeError(f"q and w must be int8, got {q.dtype}/{w.dtype}")
    m, k, q_stride = _rows(q, "q")
    wn, wk, w_stride = _rows(w, "w")
    if wn < 1 or wk != k or (swiglu and wn % 2):
        raise ValueError(f"shape mismatch: q {tuple(q.shape)} w {tuple(w.shape)}")
    n = wn // 2 if swiglu else wn
    _scales(scale, m, "scale")
    _scales(w_scale, wn, "w_scale")
    dev = q.device
    same_device(dev, scale=scale, w=w, w_scale=w_scale, out=out)
    if out is None:
        out = _new_out(m, n, out_dtype, dev)
    out_stride, kind = _check_out(out, m, n)
    args = _lib.QxInt8Args(q.data_ptr(), q_stride, scale.data_ptr(), w.data_ptr(), w_stride, w_scale.data_ptr(),
                           out.data_ptr(), out_stride, kind, m, n, k, swiglu, swiglu and limit > 0, max(limit, 0.0))
    launch_on(dev, _lib.load().qx_int8_matmul, "qx_int8_matmul", ctypes.byref(args))
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
    (default: the current one) since the last read: one word for all streams and callers of
    the device, read and cleared in one step (synchronises the current stream)."""
    dev = torch.device("cuda" if device is None else device)
    if dev.index is None:
        dev = torch.device("cuda", torch.cuda.current_device())
    st = ctypes.c_uint32(0)
    launch_on(dev, _lib.load().qx_int8_status, "qx_int8_status", ctypes.byref(st))
    return int(st.value)


class Int8Expert:
    """A dense SwiGLU expert in 8 bits: q = quant(x); h = swiglu(q . w13^T) in FP32;
    q2 = quant(h); y = q2 . w2^T. w13 int8 [2 inter, k] (gate rows, then up rows), w2
    int8 [k, inter], one FP32 scale per row of each. One C call (qx_int8_expert).

    The weights are the tensors given, best in rows on 16-byte boundaries as `quant_int8`
    lays them out (others take a path 6 to 40 times slower): they are not copied, what is written into them in
    place counts from the next call on, and they cannot be exchanged for others (make
    another expert)."""

    def __init__(self, w13: torch.Tensor, w13_scale: torch.Tensor, w2: torch.Tensor, w2_scale: torch.Tensor,
                 swiglu_limit: float = SWIGLU_LIMIT):
        if w13.dtype != torch.int8 or w2.dtype != torch.int8:
            raise TypeError(f"w13 and w2 must be int8, got {w13.dtype}/{w2.dtype}")
        w13_stride, w2_stride = _rows(w13, "w13")[2], _rows(w2, "w2")[2]
        if w13.shape[0] % 2 or w13.shape[0] < 2 or w2.shape != (w13.shape[1], w13.shape[0] // 2):
            raise ValueError(f"shape mismatch: w13 {tuple(w13.shape)} w2 {tuple(w2.shape)}")
        _scales(w13_scale, w13.shape[0], "w13_scale")
        _scales(w2_scale, w2.shape[0], "w2_scale")
        self.dev = w13.device
        for name, t in (("w13_scale", w13_scale), ("w2", w2), ("w2_scale", w2_scale)):
            if t.device != self.dev:
                raise ValueError(f"{name} is on {t.device}, not on {self.dev}")
        # Views of its own: the addresses below stay those of memory that this object holds,
        # whatever becomes of the caller's tensor objects.
        self._held = tuple(t.detach() for t in (w13, w13_scale, w2, w2_scale))
        self.weights = (w13.data_ptr(), w13_stride, w13_scale.data_ptr(), w2.data_ptr(), w2_stride, w2_scale.data_ptr())
        self.k, self.inter = w13.shape[1], w13.shape[0] // 2
        self.limit = float(max(swiglu_limit, 0.0))

    w13 = property(lambda self: self._held[0].detach())
    w13_scale = property(lambda self: self._held[1].detach())
    w2 = property(lambda self: self._held[2].detach())
    w2_scale = property(lambda self: self._held[3].detach())

    @classmethod
    def from_weights(cls, w13: torch.Tensor, w2: torch.Tensor, swiglu_limit: float = SWIGLU_LIMIT) -> "Int8Expert":
        """Quantise BF16 / FP16 / FP32 weights, one scale per output channel."""
        return cls(*quant_int8(w13), *quant_int8(w2), swiglu_limit=swiglu_limit)

    def workspace_bytes(self, rows: int) -> int:
        return _lib.load().qx_int8_expert_workspace_bytes(rows, self.k, self.inter)

    def alloc_workspace(self, rows: int) -> torch.Tensor:
        """Workspace for calls of up to `rows` rows. Calls that may overlap on the GPU
        (two streams, two graphs in flight at once) need one each."""
        return torch.empty(self.workspace_bytes(rows), dtype=torch.uint8, device=self.dev)

    def __call__(self, x: torch.Tensor, x_scale: torch.Tensor | None = None, out: torch.Tensor | None = None,
                 workspace: torch.Tensor | None = None, out_dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """[rows, k] of `out`'s type (or out_dtype) for x [rows, k] (bf16, fp16, fp32, or
        e4m3 with x_scale)."""
        rows, k, stride, kind, scale_ptr, n_scale = _check_x(x, x_scale)
        if k != self.k:
            raise ValueError(f"x must be [rows, {self.k}], got {tuple(x.shape)}")
        same_device(self.dev, x=x, x_scale=x_scale, out=out, workspace=workspace)
        if out is None:
            out = _new_out(rows, k, out_dtype, self.dev)
        out_stride, out_kind = _check_out(out, rows, k)
        if workspace is None:
            workspace = self.alloc_workspace(rows)
        if workspace.dtype != torch.uint8 or not workspace.is_contiguous():
            raise TypeError("workspace must be a contiguous uint8 tensor (alloc_workspace)")
        args = _lib.QxInt8ExpertArgs(
            x.data_ptr(), stride, kind, n_scale, scale_ptr, *self.weights, out.data_ptr(), out_stride, out_kind, rows,
            k, self.inter, self.limit > 0, self.limit, workspace.data_ptr(), workspace.numel())
        launch_on(self.dev, _lib.load().qx_int8_expert, "qx_int8_expert", ctypes.byref(args))
        return out
