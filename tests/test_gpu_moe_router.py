"""The router's product of a whole MoE layer on inputs whose logits are known exactly.

Where x has few non-zero elements and every partial sum is a number of FP32, the logits
are exact whatever the order and rounding of the sums: FP32 router weights are three
BF16 parts whose sum they are (24 bits are three times 8). So the order of experts that
differ in their last bit is checked, and the weights exp(l_j - l_0) / sum against 64 bits:
with |l_j - l_0| <= 8, the difference moves a term by 8 * 2^-24, expf by 4 * 2^-24 (2 units of
its last place), the sum of up to 8 terms by 7 * 2^-24 and the quotient by 2^-24, numerator
and sum together (8 + 4) * 2 + 7 + 1 = 32 times 2^-24. (A missing third part moves a logit
near 1 by up to 2^-17, 128 times 2^-24.)
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
E = 48


@pytest.fixture(scope="module")
def arena(cuda_ready):
    from qmesh_b200.arena import Arena
    ar = Arena(cuda_ready, 1, E, 0, 32)
    ar.fill_synthetic(0, seed=3)
    return ar


def select(ar, x, gate, topk=8, bias=None, x_scale=None):
    from qmesh_b200.moe import moe_layer
    rows = x.shape[0]
    ids = torch.empty(rows, topk, dtype=torch.int32, device="cuda")
    tw = torch.empty(rows, topk, device="cuda")
    moe_layer(ar, 0, x.cuda(), gate.cuda(), topk=topk, ids=ids, tw=tw, bias=None if bias is None else bias.cuda(),
              x_scale=None if x_scale is None else x_scale.cuda())
    return ids.cpu().long(), tw.cpu().double()


def check(ids, tw, logits, topk=8):
    """Against exact logits: the order of torch's stable sort (lower id of equals first)."""
    want = torch.sort(logits, dim=1, descending=True, stable=True)
    assert torch.equal(ids, want.indices[:, :topk])
    w = torch.softmax(want.values[:, :topk], 1)
    assert ((tw - w).abs() <= 32 * U * w).all(), float(((tw - w).abs() / w).max() / U)


# one position in every quarter of K, several warps, lanes and places of a lane's eight
PLACES = [0, 7, 33, 170, 1279, 1280, 1999, 2562, 3839, 3844, 5000, 5119]


@pytest.mark.parametrize("gate_dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("fp8", [False, True])
def test_one_element(arena, gate_dtype, fp8):
    """Row r reads the router's column PLACES[r]: logits are that column."""
    g = torch.Generator().manual_seed(1)
    gate = torch.rand(E, 5120, generator=g) * 4 - 2
    # the last column: experts that differ in the last bit of FP32 only
    gate[:, PLACES[-1]] = 1.0 + torch.randperm(E, generator=g) * 2.0 ** -23
    gate = gate.to(gate_dtype)
    x = torch.zeros(len(PLACES), 5120)
    for r, k in enumerate(PLACES):
        x[r, k] = 1.0
    x = x.to(torch.float8_e4m3fn) if fp8 else x.to(torch.bfloat16)
    ids, tw = select(arena, x, gate, x_scale=torch.ones(len(PLACES)) if fp8 else None)
    check(ids, tw, gate[:, PLACES].double().t())


@pytest.mark.parametrize("rows", [1, 9, 20])
def test_exact_sums_over_all_quarters(arena, rows):
    """Weights in multiples of 2^-14 up to 1/8, x in {-2, -1, 1, 2} at 32 places per row: every
    partial sum is a multiple of 2^-14 up to 8, and so is the bias."""
    g = torch.Generator().manual_seed(rows)
    gate = torch.randint(-2 ** 14 + 1, 2 ** 14, (E, 5120), generator=g).float() / 2 ** 14 / 8
    gate = torch.round(gate * 2 ** 14) / 2 ** 14
    x = torch.zeros(rows, 5120)
    for r in range(rows):
        k = torch.randperm(5120, generator=g)[:32]
        x[r, k] = torch.tensor([-2.0, -1.0, 1.0, 2.0])[torch.randint(0, 4, (32,), generator=g)]
    bias = torch.randint(-2 ** 13, 2 ** 13, (E,), generator=g).float() / 2 ** 14
    ids, tw = select(arena, x.to(torch.bfloat16), gate, bias=bias)
    check(ids, tw, x.double() @ gate.double().t() + bias.double())


def test_close_logits_of_the_third_part(arena):
    """Two places: a common 0.5, and weights that only the third part tells apart; reversed
    signs reverse the order."""
    g = torch.Generator().manual_seed(8)
    gate = torch.zeros(E, 5120)
    order = torch.randperm(E, generator=g)
    gate[:, 100] = 0.5
    gate[:, 4000] = 1.0 + 2.0 ** -9 + order * 2.0 ** -23
    x = torch.zeros(2, 5120)
    x[0, [100, 4000]] = 1.0
    x[1, 100], x[1, 4000] = 1.0, -1.0
    ids, tw = select(arena, x.to(torch.bfloat16), gate)
    check(ids, tw, x.double() @ gate.double().t())
    assert torch.equal(order[ids[0]], torch.arange(E - 1, E - 9, -1)) and torch.equal(order[ids[1]], torch.arange(8))
