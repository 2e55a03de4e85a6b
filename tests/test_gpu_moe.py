"""A whole MoE layer for a few tokens (qx_moe_decode_tc) against its formula in 64 bits.

Tolerances. A logit is a sum of 5120 products in FP32: each product enters one FMA
chain of at most 24 terms, then 5 tree steps over lanes, 7 over warps and the bias,
so |l - l64| <= B = 38 * 2^-24 * (sum |x w| + |bias|) to first order. Selection: the
j-th selected expert's 64-bit logit is within 2 B of the j-th largest. A weight
exp(l_j - l_0) / sum changes by at most a factor exp(4 B); CUDA documents expf within
2 ulp (4 * 2^-24), and the differences, the sum of up to 8 and the quotient add
2^-24 each of the values involved. The output is one BF16 rounding (half an ulp) of
an FP32 sum: at most 1 BF16 ulp at max(|value|, 2^-10 rms of the row).
"""

import pytest
import torch

import helpers as H
from oracle import moe

pytestmark = pytest.mark.gpu

U = 2.0 ** -24


def layer_of(seed, n_experts, inter):
    return moe.random_code_layer(n_experts, torch.Generator().manual_seed(seed), inter=inter)


def arena_of(dev, layer, n_experts, inter):
    from qmesh_b200.arena import Arena
    ar = Arena(dev, 1, n_experts, 0, inter)
    ar.load_layer(0, layer)
    return ar


def inputs(seed, rows, n_experts, gate_dtype, bias):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, 5120, generator=g).to(torch.bfloat16)
    gate = (torch.randn(n_experts, 5120, generator=g) * 0.02).to(gate_dtype)
    b = torch.randn(n_experts, generator=g) if bias else None
    return x, gate, b


def logits64(x, gate, bias):
    l = x.double() @ gate.double().T
    mag = x.double().abs() @ gate.double().abs().T
    if bias is not None:
        l, mag = l + bias.double(), mag + bias.double().abs()
    return l, 38 * U * mag


def check_selection(ids, tw, l, b, topk):
    """The selection follows the 64-bit logits within their bound, and the weights the
    softmax over the selected."""
    ids, tw = ids.cpu().long(), tw.cpu().double()
    want = l.sort(dim=1, descending=True).values[:, :topk]
    got = torch.gather(l, 1, ids)
    bound = b.amax(1, keepdim=True)
    assert ((got - want).abs() <= 2 * bound).all()
    assert all(len(set(r)) == topk for r in ids.tolist())
    w = torch.softmax(got, 1)
    rel = torch.expm1(4 * bound) + (4 + 4 + 8 + 1 + 2) * U
    assert ((tw - w).abs() <= rel * w + 1e-40).all()


def want_out(x, ids, tw, layer, c0, c1, limit=10.0):
    return moe.slice_w4a16(x.float(), ids.cpu().int(), tw.cpu(), layer, c0, c1, limit=limit, has_limit=limit > 0,
                           dtype=torch.float64, round_out=False)


def assert_one_rounding(out, want, what):
    p = H.parity(out, want.float())
    assert p["max_ulp"] <= 1.0 and p["rel_l2"] <= 2.0 ** -8, f"{what} {p}"


CASES = [  # rows, experts, topk, inter, gate, bias
    (1, 8, 6, 128, torch.bfloat16, False),
    (1, 1, 1, 64, torch.float32, True),
    (6, 384, 6, 64, torch.bfloat16, False),
    (6, 16, 6, 288, torch.float32, False),
    (7, 130, 3, 96, torch.bfloat16, True),
    (13, 100, 8, 64, torch.float32, True),
    (64, 24, 8, 96, torch.bfloat16, True),
    (9, 515, 4, 32, torch.bfloat16, True),
    (17, 3, 3, 320, torch.float32, False),
]


@pytest.mark.parametrize("rows,n_exp,topk,inter,gate_dtype,bias", CASES)
def test_layer(cuda_ready, rows, n_exp, topk, inter, gate_dtype, bias):
    """Selection, weights and output; and the same bytes as the slice given that selection."""
    from qmesh_b200.expert_slice import device_status, expert_slice
    from qmesh_b200.moe import alloc_workspace, moe_layer
    dev = cuda_ready
    layer = layer_of(rows + n_exp, n_exp, inter)
    ar = arena_of(dev, layer, n_exp, inter)
    x, gate, b = inputs(rows * 3 + n_exp, rows, n_exp, gate_dtype, bias)
    ids = torch.full((rows, topk), -7, dtype=torch.int32, device=dev)
    tw = torch.full((rows, topk), -7.0, device=dev)
    ws = alloc_workspace(rows, n_exp, topk, 0, inter, dev)
    dx, dg, db = x.to(dev), gate.to(dev), None if b is None else b.to(dev)
    out = moe_layer(ar, 0, dx, dg, bias=db, topk=topk, ids=ids, tw=tw, workspace=ws)
    assert device_status(ws) == 0
    l, bound = logits64(x, gate, b)
    check_selection(ids, tw, l, bound, topk)
    assert torch.equal(out, expert_slice(ar, 0, dx, ids, tw))
    assert_one_rounding(out, want_out(x, ids, tw, layer, 0, inter), f"rows={rows} E={n_exp}")
    # the same call again, without the optional outputs and with its own workspace
    assert torch.equal(out, moe_layer(ar, 0, dx, dg, bias=db, topk=topk))


@pytest.mark.parametrize("rows,c0,c1,limit", [(2, 64, 192, 10.0), (5, 128, 288, 0.0), (10, 0, 32, 1.5)])
def test_layer_with_shared_expert_and_column_range(cuda_ready, rows, c0, c1, limit):
    """The shared expert's FP32 output joins before the one rounding; a column range and
    other clamps."""
    from qmesh_b200.moe import moe_layer
    dev = cuda_ready
    layer, sh = layer_of(1, 12, 288), layer_of(2, 1, 160)
    ar, sar = arena_of(dev, layer, 12, 288), arena_of(dev, sh, 1, 160)
    x, gate, _ = inputs(rows, rows, 12, torch.bfloat16, False)
    ids = torch.empty(rows, 6, dtype=torch.int32, device=dev)
    tw = torch.empty(rows, 6, device=dev)
    out = moe_layer(ar, 0, x.to(dev), gate.to(dev), shared=sar.view(0), c0=c0, c1=c1, ids=ids, tw=tw,
                    swiglu_limit=limit)
    one = torch.zeros(rows, 1, dtype=torch.int32)
    want = want_out(x, ids, tw, layer, c0, c1, limit) + want_out(x, one, torch.ones(rows, 1), sh, 0, 160, limit)
    assert_one_rounding(out, want, f"shared rows={rows}")


@pytest.mark.parametrize("rows", [1, 9])
def test_layer_with_int8_shared_expert(cuda_ready, rows):
    """A W8A8 shared expert: its FP32 output is the addend, and all parts round once."""
    from qmesh_b200.int8 import Int8Expert
    from qmesh_b200.moe import moe_layer
    dev = cuda_ready
    layer = layer_of(4, 10, 96)
    ar = arena_of(dev, layer, 10, 96)
    x, gate, _ = inputs(rows, rows, 10, torch.float32, False)
    g = torch.Generator().manual_seed(6)
    ex = Int8Expert.from_weights((torch.randn(256, 5120, generator=g) * 0.02).to(dev),
                                 (torch.randn(5120, 128, generator=g) * 0.05).to(dev))
    ids = torch.empty(rows, 6, dtype=torch.int32, device=dev)
    tw = torch.empty(rows, 6, device=dev)
    out = moe_layer(ar, 0, x.to(dev), gate.to(dev), shared=ex, ids=ids, tw=tw)
    add = ex(x.to(dev), out_dtype=torch.float32).cpu().double()
    assert_one_rounding(out, want_out(x, ids, tw, layer, 0, 96) + add, "int8 shared")


def test_fp8_activations(cuda_ready):
    """FP8 rows with a scale per row or one for all: the router and the experts read
    bf16(float(e4m3) scale)."""
    from qmesh_b200.moe import moe_layer
    dev = cuda_ready
    layer = layer_of(5, 14, 64)
    ar = arena_of(dev, layer, 14, 64)
    _, gate, b = inputs(5, 1, 14, torch.bfloat16, True)
    for rows, one in ((6, False), (10, True)):
        _, q, inv = H.activations(rows, rows)
        inv = inv[:1].clone() if one else inv
        x = H.ingest(q, inv.expand(rows) if one else inv).to(torch.bfloat16)
        ids = torch.empty(rows, 5, dtype=torch.int32, device=dev)
        tw = torch.empty(rows, 5, device=dev)
        out = moe_layer(ar, 0, q.to(dev), gate.to(dev), bias=b.to(dev), topk=5, x_scale=inv.to(dev), ids=ids, tw=tw)
        l, bound = logits64(x, gate, b)
        check_selection(ids, tw, l, bound, 5)
        assert_one_rounding(out, want_out(x, ids, tw, layer, 0, 64), "fp8")


def test_ties_masks_and_nan_rows(cuda_ready):
    """Equal logits go to the lower id; an expert at -infinity is not selected (id -1,
    weight 0, no contribution), not even when nothing else is left; a bias at the type's
    lowest value only weighs nothing; a row with a NaN or an infinity is NaN and leaves
    the other rows as they are."""
    from qmesh_b200.expert_slice import expert_slice
    from qmesh_b200.moe import moe_layer
    dev = cuda_ready
    layer = layer_of(7, 40, 64)
    ar = arena_of(dev, layer, 40, 64)
    x, gate, _ = inputs(8, 4, 40, torch.float32, False)
    gate[5:] = gate[5]                                  # experts 5..39 always tie
    ids = torch.empty(4, 6, dtype=torch.int32, device=dev)
    tw = torch.empty(4, 6, device=dev)

    def call(xx, bias=None, topk=6):
        i, t = ids[:, :topk].contiguous(), tw[:, :topk].contiguous()
        o = moe_layer(ar, 0, xx.to(dev), gate.to(dev), bias=None if bias is None else bias.to(dev), topk=topk, ids=i,
                      tw=t)
        return o, i.cpu(), t.cpu()

    out, i, t = call(x)
    for r in range(4):
        tied = [e for e in i[r].tolist() if e >= 5]
        assert tied == list(range(5, 5 + len(tied)))
    # all but two experts masked
    b = torch.full((40,), float("-inf"))
    b[[3, 17]] = 0.0
    out, i, t = call(x, b)
    assert (i[:, 2:] == -1).all() and (t[:, 2:] == 0).all()
    assert all(sorted(r) == [3, 17] for r in i[:, :2].tolist())
    assert torch.allclose(t.sum(1), torch.ones(4), rtol=1e-6)
    assert torch.equal(out, expert_slice(ar, 0, x.to(dev), i.to(dev), t.to(dev)))
    # all masked: nothing is selected
    out, i, t = call(x, torch.full((40,), float("-inf")))
    assert (i == -1).all() and (t == 0).all() and (out == 0).all()
    # masked with the lowest finite value: selected last, at weight 0
    b = torch.full((40,), torch.finfo(torch.float32).min)
    b[[3, 17]] = 0.0
    out, i, t = call(x, b, 4)
    assert all(sorted(r) == [3, 17] for r in i[:, :2].tolist()) and (t[:, 2:] == 0).all()
    assert i[:, 2:].tolist() == [[0, 1]] * 4 and torch.isfinite(out.float()).all()
    # non-finite rows
    clean, ci, ct = call(x)
    for bad in (float("nan"), float("inf"), float("-inf")):
        y = x.clone()
        y[2, 77] = bad
        out, i, t = call(y)
        assert out[2].isnan().all()
        keep = [0, 1, 3]
        assert torch.equal(out[keep], clean[keep]) and torch.equal(i[keep], ci[keep]) and torch.equal(t[keep], ct[keep])


def test_views_graphs_and_streams(cuda_ready):
    """Strided x, gate and out; a captured call replayed on new inputs, two graphs on one
    workspace one after the other, and a side stream; rows past the call's stay as they were."""
    from qmesh_b200.moe import alloc_workspace, moe_layer
    dev = cuda_ready
    layer, sh = layer_of(9, 20, 160), layer_of(10, 1, 96)
    ar, sar = arena_of(dev, layer, 20, 160), arena_of(dev, sh, 1, 96)
    _, gate, b = inputs(11, 1, 20, torch.bfloat16, True)
    wide = torch.zeros(20, 5120 + 64, dtype=torch.bfloat16, device=dev)
    wide[:, 32:32 + 5120] = gate.to(dev)
    dg, db = wide[:, 32:32 + 5120], b.to(dev)
    xs = [inputs(20 + i, 6, 20, torch.bfloat16, False)[0].to(dev) for i in range(3)]
    want = [moe_layer(ar, 0, x, gate.to(dev), bias=db, shared=sar.view(0)) for x in xs]
    ws = alloc_workspace(6, 20, 6, 0, 160, dev)
    xb = torch.zeros(8, 5120 + 16, dtype=torch.bfloat16, device=dev)
    ob = torch.full((8, 5120 + 8), 5.0, dtype=torch.bfloat16, device=dev)
    x, out = xb[1:7, 8:8 + 5120], ob[1:7, 4:4 + 5120]
    view = sar.view(0)

    def call():
        moe_layer(ar, 0, x, dg, bias=db, shared=view, out=out, workspace=ws)

    x.copy_(xs[0])
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        call()
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want[0])
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for g in graphs:
        with torch.cuda.graph(g):
            call()
    for i in (1, 2, 0, 1):
        x.copy_(xs[i])
        graphs[i % 2].replay()
        torch.cuda.synchronize()
        assert torch.equal(out, want[i])
    ob[1:7, 4:4 + 5120] = 5.0
    assert (ob == 5.0).all()


def test_full_width_layer(cuda_ready):
    """The layer at its full width (2304 columns, shared expert) against the slice and
    the separate shared call."""
    from qmesh_b200.arena import Arena
    from qmesh_b200.expert_slice import expert_slice
    from qmesh_b200.moe import moe_layer
    dev = cuda_ready
    ar, sar = Arena(dev, 1, 40, 0, 2304), Arena(dev, 1, 1, 0, 2304)
    ar.fill_synthetic(0, seed=5)
    sar.fill_synthetic(0, seed=6)
    for rows in (1, 6, 30):
        x, gate, _ = inputs(rows, rows, 40, torch.bfloat16, False)
        ids = torch.empty(rows, 6, dtype=torch.int32, device=dev)
        tw = torch.empty(rows, 6, device=dev)
        dx = x.to(dev)
        out = moe_layer(ar, 0, dx, gate.to(dev), shared=sar.view(0), ids=ids, tw=tw)
        l, bound = logits64(x, gate, None)
        check_selection(ids, tw, l, bound, 6)
        routed = expert_slice(ar, 0, dx, ids, tw).float()
        one = torch.zeros(rows, 1, dtype=torch.int32, device=dev)
        shared = expert_slice(sar, 0, dx, one, torch.ones(rows, 1, device=dev)).float()
        # each part within half an ulp of its FP32 value, the output half an ulp of the sum
        err = (out.float() - (routed + shared)).abs().cpu()
        tol = 0.5 * (H.bf16_ulp(routed.cpu()) + H.bf16_ulp(shared.cpu()) + H.bf16_ulp(out.float().cpu())) * 1.001
        assert (err <= tol).all()


def test_prefill_with_int8_shared_expert(cuda_ready):
    """A prefill chunk with a W8A8 shared expert: the ordered combine of the routed
    partial and the expert's BF16 output, bit for bit, for FP8 and BF16 activations."""
    from qmesh_b200.combine import combine_ordered
    from qmesh_b200.expert_slice import prefill_slice
    from qmesh_b200.int8 import Int8Expert
    dev = cuda_ready
    rows = 150
    layer = layer_of(12, 6, 128)
    ar = arena_of(dev, layer, 6, 128)
    ids, tw = H.random_routing(rows, 6, 3, topk=4)
    _, q, inv = H.activations(rows, 3)
    a2 = torch.full((6,), 50.0, device=dev)
    g = torch.Generator().manual_seed(6)
    ex = Int8Expert.from_weights((torch.randn(320, 5120, generator=g) * 0.02).to(dev),
                                 (torch.randn(5120, 160, generator=g) * 0.05).to(dev))
    for x, xs in ((q.to(dev), inv.to(dev)), (H.ingest(q, inv).to(torch.bfloat16).to(dev), None)):
        kw = dict(x_scale=xs)
        got = prefill_slice(ar, 0, x, ids.to(dev), tw.to(dev), a2, shared=ex, **kw)
        routed = prefill_slice(ar, 0, x, ids.to(dev), tw.to(dev), a2, **kw)
        assert torch.equal(got, combine_ordered([routed, ex(x, xs)]))
        assert not torch.equal(got, routed)


@pytest.mark.parametrize("rows,n_exp,topk", [(64, 4096, 8), (33, 1501, 8), (1, 4096, 1)])
def test_many_experts(cuda_ready, rows, n_exp, topk):
    """The most rows, experts and slots that a call takes: up to 4096 keys per row in
    shared memory, 512 pairs in the routing tables. The last expert ties with the first."""
    from qmesh_b200.arena import Arena
    from qmesh_b200.expert_slice import device_status, expert_slice
    from qmesh_b200.moe import alloc_workspace, moe_layer
    dev = cuda_ready
    ar = Arena(dev, 1, n_exp, 0, 32)
    ar.fill_synthetic(0, seed=3)
    x, gate, b = inputs(n_exp, rows, n_exp, torch.bfloat16, True)
    gate[-1], b[-1] = gate[0], b[0]
    ids = torch.empty(rows, topk, dtype=torch.int32, device=dev)
    tw = torch.empty(rows, topk, device=dev)
    ws = alloc_workspace(rows, n_exp, topk, 0, 32, dev)
    dx = x.to(dev)
    out = torch.full((rows + 1, 5120), 3.0, dtype=torch.bfloat16, device=dev)
    moe_layer(ar, 0, dx, gate.to(dev), bias=b.to(dev), topk=topk, ids=ids, tw=tw, workspace=ws, out=out)
    assert device_status(ws) == 0
    l, bound = logits64(x, gate, b)
    check_selection(ids, tw, l, bound, topk)
    for r in ids.tolist():
        assert n_exp - 1 not in r or (0 in r and r.index(0) < r.index(n_exp - 1))
    assert torch.equal(out[:rows], expert_slice(ar, 0, dx, ids, tw)) and (out[rows] == 3.0).all()


def test_two_layers_on_two_streams(cuda_ready):
    """Two calls at once, each with its own workspace and its own INT8 shared expert
    workspaces, give the bytes of the calls one after the other."""
    from qmesh_b200.int8 import Int8Expert
    from qmesh_b200.moe import alloc_workspace, moe_layer
    dev = cuda_ready
    layer = layer_of(14, 16, 96)
    ar = arena_of(dev, layer, 16, 96)
    g = torch.Generator().manual_seed(2)
    ex = Int8Expert.from_weights((torch.randn(192, 5120, generator=g) * 0.02).to(dev),
                                 (torch.randn(5120, 96, generator=g) * 0.05).to(dev))
    data = [[t if t is None else t.to(dev) for t in inputs(30 + i, 5 + i, 16, torch.float32, True)] for i in range(2)]
    want = [moe_layer(ar, 0, x, gate, bias=b, shared=ex) for x, gate, b in data]
    ws = [alloc_workspace(6, 16, 6, 0, 96, dev) for _ in range(2)]
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (x, gate, b) in enumerate(data):
            with torch.cuda.stream(streams[i]):
                got[i].append(moe_layer(ar, 0, x, gate, bias=b, shared=ex, workspace=ws[i]))
    torch.cuda.synchronize()
    for i in range(2):
        assert all(torch.equal(o, want[i]) for o in got[i])
