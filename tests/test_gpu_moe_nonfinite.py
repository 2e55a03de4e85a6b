"""Rows of a whole MoE layer that hold a NaN or an infinity: NaN weights and a NaN output,
whatever the router's weights make of them, and the other rows as without them."""

import pytest
import torch

import helpers as H
from oracle import moe

pytestmark = pytest.mark.gpu

ROWS, E = 5, 12


@pytest.fixture(scope="module")
def arenas(cuda_ready):
    from qmesh_b200.arena import Arena

    def make(n):
        ar = Arena(cuda_ready, 1, n, 0, 64)
        ar.load_layer(0, moe.random_code_layer(n, torch.Generator().manual_seed(n), inter=64))
        return ar
    return {n: make(n) for n in (1, E)}


def call(ar, x, gate, topk, **kw):
    from qmesh_b200.moe import moe_layer
    ids = torch.empty(x.shape[0], topk, dtype=torch.int32, device="cuda")
    tw = torch.empty(x.shape[0], topk, device="cuda")
    out = moe_layer(ar, 0, x.cuda(), gate.cuda(), topk=topk, ids=ids, tw=tw, **kw)
    return out, ids, tw


@pytest.mark.parametrize("n_exp,topk", [(E, 4), (1, 1)])
@pytest.mark.parametrize("gate_dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("sign", [-1.0, 1.0, 0.0])
def test_one_element(arenas, n_exp, topk, gate_dtype, sign):
    """sign: of every router weight at the row's bad element (0: as they come). With -1 and an
    infinity all logits are -infinity, as if every expert were masked."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn(ROWS, 5120, generator=g).to(torch.bfloat16)
    gate = torch.randn(n_exp, 5120, generator=g) * 0.02
    keep = [0, 1, 3, 4]
    for at in (0, 1290, 5119):                              # in the first and in other quarters of K
        w = gate.clone()
        if sign:
            w[:, at] = sign * (w[:, at].abs() + 1e-3)
        w = w.to(gate_dtype)
        clean = call(arenas[n_exp], x, w, topk)
        for bad in (float("inf"), float("-inf"), float("nan")):
            y = x.clone()
            y[2, at] = bad
            out, ids, tw = call(arenas[n_exp], y, w, topk)
            assert out[2].isnan().all() and tw[2].isnan().all(), (at, bad)
            assert sorted(set(ids[2].tolist())) == sorted(ids[2].tolist()) and 0 <= ids[2].min() and ids[2].max() < n_exp
            for a, b in zip((out, ids, tw), clean):
                assert torch.equal(a[keep], b[keep])


def test_infinite_scale(arenas):
    """FP8 rows whose dequant scale is infinite."""
    _, q, inv = H.activations(ROWS, 4)
    w = -torch.rand(E, 5120, generator=torch.Generator().manual_seed(5)).to(torch.bfloat16) - 0.1
    q = q.view(torch.uint8) & 0x7f                           # no negative values, none of them 0 or NaN
    q = q.clamp(8, 0x70).view(torch.float8_e4m3fn)
    clean = call(arenas[E], q, w, 3, x_scale=inv.cuda())
    bad = inv.clone()
    bad[1] = float("inf")
    out, ids, tw = call(arenas[E], q, w, 3, x_scale=bad.cuda())
    assert out[1].isnan().all() and tw[1].isnan().all()
    keep = [0, 2, 3, 4]
    for a, b in zip((out, ids, tw), clean):
        assert torch.equal(a[keep], b[keep])


def test_masked_rows_that_are_finite(arenas):
    """Every expert masked: nothing is selected and the output is 0, as before."""
    g = torch.Generator().manual_seed(6)
    x = torch.randn(ROWS, 5120, generator=g).to(torch.bfloat16)
    x[1], x[2, 7] = 0.0, torch.finfo(torch.bfloat16).max / 4
    gate = (torch.randn(E, 5120, generator=g) * 0.02).to(torch.bfloat16)
    out, ids, tw = call(arenas[E], x, gate, 4, bias=torch.full((E,), float("-inf"), device="cuda"))
    assert (ids == -1).all() and (tw == 0).all() and (out == 0).all()
