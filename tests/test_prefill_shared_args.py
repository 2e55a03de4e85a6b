"""Refusals of a prefill chunk with a W8A8 shared expert and of the ordered combine
behind it, without a GPU: an output that the call would write outside of is refused
before anything is launched."""

import pytest
import torch

ROWS, HID = 8, 5120


def outs(dtype=torch.bfloat16):
    """(output that must be refused, error) pairs for ROWS rows."""
    other = torch.float32 if dtype == torch.bfloat16 else torch.bfloat16
    return [(torch.zeros(ROWS // 2, HID, dtype=dtype), ValueError),                # too few rows
            (torch.zeros(ROWS, HID - 8, dtype=dtype), ValueError),                 # too narrow
            (torch.zeros(ROWS * HID, dtype=dtype), ValueError),                    # no rows at all
            (torch.zeros(ROWS, HID, dtype=other), TypeError),
            (torch.zeros(ROWS, 2 * HID, dtype=dtype)[:, ::2], ValueError),         # column stride 2
            (torch.zeros(HID, ROWS, dtype=dtype).t(), ValueError),
            (torch.zeros(1, HID, dtype=dtype).expand(ROWS, HID), ValueError),      # rows on top of one another
            (torch.empty(ROWS, HID, dtype=dtype, device="meta"), ValueError)]      # elsewhere


@pytest.fixture
def chunk(monkeypatch):
    """A call's arguments, with every launch recorded instead of made."""
    from oracle import moe
    from qmesh_b200 import expert_slice
    from qmesh_b200.arena import Arena
    from qmesh_b200.int8 import Int8Expert
    calls = []
    ar = Arena("cpu", 1, 8, 0, 64)
    ar.load_layer(0, moe.random_code_layer(8, torch.Generator().manual_seed(0), inter=64))
    ex = Int8Expert(torch.zeros(64, HID, dtype=torch.int8), torch.ones(64), torch.zeros(HID, 32, dtype=torch.int8),
                    torch.ones(HID))
    monkeypatch.setattr(expert_slice, "launch_prefill", lambda *a, **k: calls.append("prefill"))
    monkeypatch.setattr(expert_slice, "combine_ordered", lambda parts, out: calls.append(tuple(out.shape)))
    monkeypatch.setattr(Int8Expert, "__call__", lambda self, x, xs=None: torch.zeros(ROWS, HID, dtype=torch.bfloat16))
    args = (ar, 0, torch.zeros(ROWS, HID, dtype=torch.bfloat16), torch.zeros(ROWS, 6, dtype=torch.int32),
            torch.zeros(ROWS, 6), torch.ones(8))
    return expert_slice.prefill_slice, args, ex, calls


def test_prefill_with_shared_expert_refuses_outputs(chunk):
    call, args, ex, calls = chunk
    for out, err in outs():
        with pytest.raises(err):
            call(*args, shared=ex, out=out)
        assert not calls, f"launched with out {tuple(out.shape)} {out.dtype}"


def test_prefill_with_shared_expert_takes_outputs(chunk):
    """More rows than the call's and rows further apart are fine, as without `shared`."""
    call, args, ex, calls = chunk
    for out in (None, torch.zeros(ROWS + 3, HID, dtype=torch.bfloat16),
                torch.zeros(ROWS, HID + 64, dtype=torch.bfloat16)[:, 32:32 + HID]):
        calls.clear()
        got = call(*args, shared=ex, out=out)
        assert calls == ["prefill", (ROWS, HID)] and (out is None or got is out)


def test_prefill_refuses_other_shared_experts(chunk):
    """Only a W8A8 expert of the chunk's width and device can be the shared expert."""
    from qmesh_b200.int8 import Int8Expert
    call, args, ex, calls = chunk
    for bad in (args[0].view(0), args[0], torch.nn.Identity()):
        with pytest.raises(TypeError):
            call(*args, shared=bad)
    narrow = Int8Expert(torch.zeros(64, 128, dtype=torch.int8), torch.ones(64), torch.zeros(128, 32, dtype=torch.int8),
                        torch.ones(128))
    away = Int8Expert(*(t.to("meta") for t in (ex.w13, ex.w13_scale, ex.w2, ex.w2_scale)))
    for bad in (narrow, away):
        with pytest.raises(ValueError):
            call(*args, shared=bad)
    assert not calls


@pytest.mark.parametrize("out_f32", [False, True])
def test_combine_refuses_outputs(monkeypatch, out_f32):
    """The ordered combine itself: its C entry sees a pointer and a stride only."""
    from qmesh_b200 import combine

    class Lib:
        def qx_combine_ordered(self, *args):
            raise AssertionError("launched")

    monkeypatch.setattr(combine._lib, "load", lambda: Lib())
    parts = [torch.zeros(ROWS, HID, dtype=torch.bfloat16) for _ in range(2)]
    for out, err in outs(torch.float32 if out_f32 else torch.bfloat16):
        with pytest.raises(err):
            combine.combine_ordered(parts, out=out, out_f32=out_f32, stream=0)
    with pytest.raises((TypeError, ValueError)):                   # parts that are no rows of 5120
        combine.combine_ordered([p[:, :HID - 8] for p in parts], stream=0)
    with pytest.raises(ValueError):                                # a part on another device
        combine.combine_ordered([parts[0], parts[1].to("meta")], stream=0)
