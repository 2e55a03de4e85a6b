"""Fixed-order combine of per-rank BF16 partials (the reference's seam combine,
native/qmesh_afd_seam.cu:310-484): out = bf16(p0 + p1 + ... ) summed in FP32 in
list order with one rounding, or kept in FP32 (out_f32)."""

from __future__ import annotations

import ctypes

import torch

from . import _lib


def check_out(out: torch.Tensor, rows: int, dev: torch.device, dtype: torch.dtype = torch.bfloat16) -> None:
    """An output of at least `rows` rows of 5120 on `dev`: the C entries see its address
    and its row stride only."""
    if out.dtype != dtype:
        raise TypeError(f"out must be {dtype}, got {out.dtype}")
    if out.dim() != 2 or out.shape[0] < rows or out.shape[1] != _lib.HIDDEN or out.stride(1) != 1 \
            or (rows > 1 and out.stride(0) < _lib.HIDDEN):
        raise ValueError(f"out must be [{rows}, {_lib.HIDDEN}] with unit column stride, got {tuple(out.shape)} "
                         f"with strides {out.stride()}")
    if out.device != dev:
        raise ValueError(f"out is on {out.device}, not on {dev}")


def combine_ordered(parts: list[torch.Tensor], out: torch.Tensor | None = None, out_f32: bool = False,
                    stream=None) -> torch.Tensor:
    if not parts:
        raise ValueError("no partials to combine")
    rows, dev = parts[0].shape[0], parts[0].device
    for p in parts:
        if p.dtype != torch.bfloat16 or p.shape != (rows, _lib.HIDDEN) or p.stride(1) != 1:
            raise TypeError("partials must be bf16 [rows, 5120] with unit column stride, all the same shape")
        if p.stride(0) != parts[0].stride(0):
            raise ValueError("partials must share one row stride")
        if p.device != dev:
            raise ValueError(f"partials are on {dev} and {p.device}")
    dtype = torch.float32 if out_f32 else torch.bfloat16
    if out is None:
        out = torch.empty(rows, _lib.HIDDEN, dtype=dtype, device=dev)
    else:
        check_out(out, rows, dev, dtype)
    arr = (ctypes.c_void_p * len(parts))(*[p.data_ptr() for p in parts])
    if stream is None:
        stream = torch.cuda.current_stream(dev).cuda_stream
    rc = _lib.load().qx_combine_ordered(arr, len(parts), parts[0].stride(0), ctypes.c_void_p(out.data_ptr()),
                                        out.stride(0), 1 if out_f32 else 0, rows, ctypes.c_void_p(stream))
    _lib.check(rc, "qx_combine_ordered")
    return out
