"""A whole MoE layer for a few tokens (qx_moe_decode_tc): the router's product, the
top-k selection, the NVFP4 routed experts over a column range and a shared expert in
one call.

    out = moe_layer(arena, li, x, gate, topk=6, shared=shared_arena.view(0))

``x`` is the layer's activation as the slice takes it (BF16, or FP8 with x_scale),
``gate`` the router weights [n_experts, 5120] in BF16 or FP32. `expert_slice` is the
same layer from ids and weights that were selected elsewhere.
"""

from __future__ import annotations

import ctypes

import torch

from . import _lib
from .arena import Arena
from .expert_slice import SWIGLU_LIMIT, _slice_args
from .int8 import Int8Expert, launch_on, same_device


def workspace_bytes(rows: int, n_experts: int, topk: int, c0: int, c1: int) -> int:
    n = _lib.load().qx_moe_workspace_bytes(rows, n_experts, topk, c0, c1)
    if n == 0:
        raise ValueError(f"no workspace for rows={rows} experts={n_experts} topk={topk} columns [{c0}, {c1})")
    return n


def alloc_workspace(rows: int, n_experts: int, topk: int, c0: int, c1: int, device) -> torch.Tensor:
    """Workspace for calls of up to `rows` rows over columns [c0, c1). Calls that may
    overlap on the GPU need one each; read the last call's status with
    `expert_slice.device_status(workspace)`."""
    return torch.empty(workspace_bytes(rows, n_experts, topk, c0, c1), dtype=torch.uint8, device=device)


def moe_layer(arena: Arena, li: int, x: torch.Tensor, gate: torch.Tensor, bias: torch.Tensor | None = None,
              topk: int = 6, shared: _lib.QxArena | Int8Expert | None = None, x_scale: torch.Tensor | None = None,
              c0: int | None = None, c1: int | None = None, out: torch.Tensor | None = None,
              ids: torch.Tensor | None = None, tw: torch.Tensor | None = None,
              workspace: torch.Tensor | None = None, swiglu_limit: float = SWIGLU_LIMIT) -> torch.Tensor:
    """BF16 [rows, 5120] = sum over the topk experts of x . gate^T (+ bias) of their
    softmax weight (over the selected) times the expert over columns [c0, c1), plus
    the shared expert: the view of a one-expert tensor-core arena, which `swiglu_limit`
    clamps too, or an `Int8Expert`, which has its own limit from its construction (its
    FP32 output and its workspace are allocated per call, its reports go to
    `int8.device_status`).
    All parts are summed in FP32 and rounded once. `ids` (int32 [rows, topk]) and `tw`
    (float32) receive the selection when given. 1 to 64 rows."""
    if arena.layout != "tc":
        raise ValueError("the MoE layer runs on the tensor-core slice (layout 'tc')")
    if x.dim() != 2:
        raise ValueError(f"x must be [rows, {_lib.HIDDEN}], got {tuple(x.shape)}")
    rows, dev = x.shape[0], x.device
    if gate.dtype not in (torch.bfloat16, torch.float32):
        raise TypeError(f"gate must be bf16 or fp32, got {gate.dtype}")
    if gate.shape != (arena.n_experts, _lib.HIDDEN) or gate.stride(1) != 1:
        raise ValueError(f"gate must be [{arena.n_experts}, {_lib.HIDDEN}] with unit column stride, "
                         f"got {tuple(gate.shape)}")
    if bias is not None and (bias.dtype != torch.float32 or bias.shape != (arena.n_experts,)
                             or not bias.is_contiguous()):
        raise TypeError(f"bias must be a contiguous float32 [{arena.n_experts}] tensor")
    for name, t, dtype in (("ids", ids, torch.int32), ("tw", tw, torch.float32)):
        if t is not None and (t.dtype != dtype or t.shape != (rows, topk) or not t.is_contiguous()):
            raise TypeError(f"{name} must be a contiguous {dtype} [{rows}, {topk}] tensor")
    c0 = arena.a0 if c0 is None else c0
    c1 = arena.a1 if c1 is None else c1
    view = arena.view(li)
    if dev != arena.w13[li].device:
        raise ValueError(f"x is on {dev}, the arena on {arena.w13[li].device}")
    same_device(dev, gate=gate, bias=bias, ids=ids, tw=tw, x_scale=x_scale, out=out, workspace=workspace)
    if out is None:
        out = torch.empty(rows, _lib.HIDDEN, dtype=torch.bfloat16, device=dev)
    if workspace is None:
        workspace = alloc_workspace(rows, arena.n_experts, topk, c0, c1, dev)
    addend = None
    if isinstance(shared, Int8Expert):
        if shared.k != _lib.HIDDEN:
            raise ValueError(f"the shared expert's width is {shared.k}, the layer's {_lib.HIDDEN}")
        addend = shared(x, x_scale, out_dtype=torch.float32)
        shared = None
    args = _slice_args(x, None, None, out, c0, c1, workspace, x_scale, max(swiglu_limit, 0.0), swiglu_limit > 0,
                       topk=topk)
    router = _lib.QxRouterArgs(
        gate.data_ptr(), _lib.QX_T_BF16 if gate.dtype == torch.bfloat16 else _lib.QX_T_F32, gate.stride(0),
        bias.data_ptr() if bias is not None else 0, ids.data_ptr() if ids is not None else 0,
        tw.data_ptr() if tw is not None else 0, addend.data_ptr() if addend is not None else 0, _lib.HIDDEN)
    launch_on(dev, _lib.load().qx_moe_decode_tc, "qx_moe_decode_tc", ctypes.byref(view), ctypes.byref(args),
              ctypes.byref(router), ctypes.byref(shared) if shared is not None else None)
    return out
