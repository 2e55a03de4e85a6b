"""W8A8 products (quantiser, matmul, SwiGLU product, dense expert) against 64-bit
restatements of their formulas on the CPU.

Tolerances. A product's value is ((float)sum * scale) * w_scale: the sum is exact,
and the conversion and the two products round once each, at most 2^-24 relative
apiece, so the FP32 value is within D = 3 * 2^-24 (1 + 2^-22), and the output
rounding adds eps / 2 of its type. SwiGLU: silu(g) = g / (1 + exp(-g)) changes by
at most (1 + |g|) times g's relative change; CUDA documents expf and __fdividef within
2 ulp each (4 * 2^-24 relative; the divisor is below 2^126 for |g| < 87), and the sum
and the product add 2^-24 each, so act is within ((1 + |g|) + 1) D + 10 * 2^-24 before
the output rounding.
"""

import pytest
import torch

pytestmark = pytest.mark.gpu

U = 2.0 ** -24
D = 3 * U * (1 + 2.0 ** -22)
TINY = 1e-30


def ref_quant(x):
    x = x.double()
    m = x.abs().amax(1, keepdim=True).clamp(min=TINY)
    return torch.round(127.0 * x / m).to(torch.int8), (m / 127.0)[:, 0]


def ref_product(q, s, w, ws):
    return (q.double() @ w.double().T) * s.double()[:, None] * ws.double()[None, :]


def ref_swiglu(h, limit):
    n = h.shape[1] // 2
    g, u = h[:, :n], h[:, n:]
    if limit > 0:
        g, u = g.clamp(max=limit), u.clamp(-limit, limit)
    return g, u, g / (1 + torch.exp(-g)) * u


def rows_of(seed, n, k, std=1.0, pad=True, lead=0):
    """Random int8 rows and scales; pad: rows 16-byte aligned, else odd strides."""
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    q[0, : min(k, 3)] = torch.tensor([-128, 127, -127], dtype=torch.int8)[: min(k, 3)]
    stride = (k + 15) // 16 * 16 if pad else k + 3
    buf = torch.zeros(n * stride + 64, dtype=torch.int8, device="cuda")
    d = torch.as_strided(buf, (n, k), (stride, 1), lead)
    d.copy_(q)
    s = (torch.rand(n, generator=g) + 0.5) * std / 127
    return q, s, d, s.cuda()


def close(out, want, rel, dtype):
    """|out - want| <= (rel + eps/2) |want|, with the type's smallest step as the floor."""
    eps = torch.finfo(dtype).eps / 2
    err = (out.double().cpu() - want).abs()
    tol = (rel + eps * (1 + rel)) * want.abs() + torch.finfo(dtype).smallest_normal * eps
    bad = ~(err <= tol)
    assert not bad.any(), f"{int(bad.sum())} of {bad.numel()}: worst {float((err / tol.clamp_min(1e-300)).max()):.3f} x tolerance"


QUANT = [(1, 1), (1, 5120), (6, 5120), (3, 17), (5, 255), (2, 4100), (300, 64), (7, 2304), (2, 20003)]


@pytest.mark.parametrize("rows,k", QUANT)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantiser(cuda_ready, rows, k, dtype):
    """BF16 and FP16: q is the exactly rounded quotient, halves to even. FP32: 127 x is
    rounded first, so q may differ where the quotient is within 127 * 2^-23 of a half."""
    from qmesh_b200.int8 import quant_int8
    g = torch.Generator().manual_seed(rows * 31 + k)
    x = (torch.randn(rows, k, generator=g) * torch.exp(2 * torch.randn(rows, 1, generator=g))).to(dtype)
    x[0, 0] = 0.0
    if k > 4:
        m = x.abs().amax(1)
        x[:, 1] = m                                  # x = m / 2 -> 63.5 exactly: rounds to 64
        x[:, 2] = -m / 2
    q, s = quant_int8(x.cuda())
    wq, ws = ref_quant(x)
    if dtype == torch.float32:
        t = 127.0 * x.double() / x.double().abs().amax(1, keepdim=True).clamp(min=TINY)
        off = (q.cpu() != wq) & ((t - torch.floor(t) - 0.5).abs() > 127 * 2.0 ** -23)
        assert not off.any() and (q.cpu().int() - wq.int()).abs().max() <= 1
    else:
        assert torch.equal(q.cpu(), wq)
    assert ((s.cpu().double() - ws).abs() <= U * ws).all()
    assert q.stride(0) % 16 == 0 or rows == 1


def test_quantiser_special_rows(cuda_ready):
    """Zero rows, denormals, the largest values, and rows that hold a NaN or an infinity
    (q = 0, scale = NaN, reported once); the other rows are as without them."""
    from qmesh_b200 import _lib
    from qmesh_b200.int8 import device_status, quant_int8
    device_status()
    x = torch.randn(8, 700, generator=torch.Generator().manual_seed(3))
    x[0] = 0.0
    x[1] = x[1] * 1e-38
    x[2] = x[2].clamp(-1, 1) * 3e38
    x[2, 5] = torch.finfo(torch.float32).max
    x[3, 699] = float("nan")
    x[5, 0] = float("-inf")
    good = [0, 1, 2, 4, 6, 7]
    q, s = quant_int8(x.cuda())
    assert device_status() == _lib.QX_DEV_NONFINITE and device_status() == 0
    wq, ws = ref_quant(x[good])
    assert (q.cpu()[good].int() - wq.int()).abs().max() <= 1
    assert (q.cpu()[good] != wq).float().mean() < 1e-3
    assert torch.allclose(s.cpu()[good].double(), ws, rtol=2 * U, atol=0)
    assert q.cpu()[[3, 5]].abs().max() == 0 and s.cpu()[[3, 5]].isnan().all()
    assert q.cpu()[0].abs().max() == 0 and float(s[0]) > 0


def test_quantiser_fp8_rows_and_strides(cuda_ready):
    """The slice's FP8 rows (one scale per row, one for all) and rows at odd offsets and
    strides; bytes between q's rows stay as they were."""
    from qmesh_b200.int8 import quant_int8
    g = torch.Generator().manual_seed(9)
    x8 = (torch.randn(5, 333, generator=g) * 30).to(torch.float8_e4m3fn)
    for inv in (torch.rand(5, generator=g) + 0.1, torch.rand(1, generator=g) + 0.1):
        x = (x8.float() * inv[:, None]).to(torch.bfloat16)
        q, s = quant_int8(x8.cuda(), inv.cuda())
        wq, ws = ref_quant(x)
        assert torch.equal(q.cpu(), wq)
        q, _ = quant_int8(x8.view(torch.uint8).cuda(), inv.cuda())
        assert torch.equal(q.cpu(), wq)
    big = torch.randn(9, 401, generator=g).to(torch.bfloat16)
    view = big.cuda()[1:8, 3:260]
    buf = torch.full((7, 300), 77, dtype=torch.int8, device="cuda")
    quant_int8(view, q=buf[:, 5:262])
    wq, _ = ref_quant(big[1:8, 3:260])
    assert torch.equal(buf[:, 5:262].cpu(), wq)
    assert (buf[:, :5] == 77).all() and (buf[:, 262:] == 77).all()


SIZES = [(1, 1, 1), (1, 8, 16), (1, 4608, 512), (2, 131, 130), (16, 128, 128), (17, 129, 257), (37, 1003, 2311),
         (64, 64, 5120), (65, 320, 96), (128, 256, 384), (129, 257, 129), (200, 640, 1000), (300, 72, 2304),
         (513, 515, 300), (1025, 384, 160),
         (1024, 5120, 272), (2100, 640, 208), (700, 9000, 64), (3000, 301, 130), (4500, 2304, 96)]


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("pad", [True, False])
def test_matmul(cuda_ready, m, n, k, pad):
    from qmesh_b200.int8 import device_status, int8_matmul
    qa, sa, da, dsa = rows_of(m + n, m, k, 1.0, pad)
    qw, sw, dw, dsw = rows_of(m * 7 + k, n, k, 0.02, pad)
    want = ref_product(qa, sa, qw, sw)
    outs = {}
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        out = int8_matmul(da, dsa, dw, dsw, out_dtype=dtype)
        close(out, want, D, dtype)
        outs[dtype] = out
    assert device_status() == 0
    # the same bytes whatever the alignment, and again for the same call
    assert torch.equal(int8_matmul(da, dsa, dw, dsw, out_dtype=torch.float32), outs[torch.float32])
    alt = rows_of(m * 7 + k, n, k, 0.02, not pad)[2]
    assert torch.equal(int8_matmul(da, dsa, alt, dsw, out_dtype=torch.float32), outs[torch.float32])


def test_matmul_largest_sums(cuda_ready):
    """Every product at -128 * -128 over the longest K allowed: the sum 128^2 (2^17 - 1)
    still fits 32 bits."""
    from qmesh_b200 import _lib
    from qmesh_b200.int8 import int8_matmul
    k = _lib.INT8_MAX_K
    for m in (1, 130):
        a = torch.full((m, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
        w = torch.full((3, k + 1), -128, dtype=torch.int8, device="cuda")[:, :k]
        one = torch.ones(m, device="cuda")
        out = int8_matmul(a, one, w, torch.ones(3, device="cuda"), out_dtype=torch.float32)
        assert (out == float(torch.tensor(128.0 * 128 * k, dtype=torch.float32))).all()


@pytest.mark.parametrize("m,n,k", [(1, 1, 16), (1, 2304, 512), (6, 100, 5120), (33, 65, 300), (130, 128, 128),
                                   (257, 333, 1111), (600, 384, 640), (1500, 2304, 144), (4100, 1111, 96)])
@pytest.mark.parametrize("limit", [10.0, 0.5, 0.0])
@pytest.mark.parametrize("pad", [True, False])
def test_swiglu(cuda_ready, m, n, k, limit, pad):
    from qmesh_b200.int8 import device_status, int8_swiglu
    qa, sa, da, dsa = rows_of(m + n, m, k, 2.0 / k ** 0.5 / 0.02, pad)
    qw, sw, dw, dsw = rows_of(m * 5 + k, 2 * n, k, 0.02, pad)
    g, u, want = ref_swiglu(ref_product(qa, sa, qw, sw), limit)
    rel = (2 + g.abs()) * D + 10 * U
    for dtype in (torch.float32, torch.bfloat16):
        out = int8_swiglu(da, dsa, dw, dsw, swiglu_limit=limit, out_dtype=dtype)
        close(out, want, rel, dtype)
    assert device_status() == 0


def test_outputs_at_odd_strides_and_guards(cuda_ready):
    """Output views whose rows start at odd element offsets: every value lands, and no
    byte around the view changes."""
    from qmesh_b200.int8 import int8_matmul
    for m, n, k in ((5, 77, 96), (140, 301, 256), (300, 500, 256)):
        qa, sa, da, dsa = rows_of(1, m, k)
        qw, sw, dw, dsw = rows_of(2, n, k, 0.02)
        want = ref_product(qa, sa, qw, sw)
        for dtype in (torch.bfloat16, torch.float32):
            buf = torch.full((m + 2, n + 9), 3.0, dtype=dtype, device="cuda")
            view = buf[1:-1, 3:3 + n]
            int8_matmul(da, dsa, dw, dsw, out=view)
            close(view, want, D, dtype)
            buf[1:-1, 3:3 + n] = 3.0
            assert (buf == 3.0).all()


@pytest.mark.parametrize("m", [3, 150, 400])
def test_nan_rows_stay_in_their_rows(cuda_ready, m):
    from qmesh_b200.int8 import int8_matmul, int8_swiglu, quant_int8
    x = torch.randn(m, 256, generator=torch.Generator().manual_seed(m))
    bad = x.clone()
    bad[1, 9] = float("nan")
    _, _, dw, dsw = rows_of(2, 128, 256, 0.02)
    for fn in (int8_matmul, int8_swiglu):
        a = fn(*quant_int8(x.cuda()), dw, dsw)
        b = fn(*quant_int8(bad.cuda()), dw, dsw)
        assert b[1].isnan().all()
        keep = torch.arange(m) != 1
        assert torch.equal(a[keep], b[keep])


def _expert(seed, k, inter):
    g = torch.Generator().manual_seed(seed)
    w13 = torch.randn(2 * inter, k, generator=g) * (1.2 / k ** 0.5)
    w2 = torch.randn(k, inter, generator=g) * (1.2 / inter ** 0.5)
    return w13, w2


@pytest.mark.parametrize("rows,k,inter,dtype", [(1, 5120, 64, torch.bfloat16), (6, 640, 288, torch.bfloat16),
                                                (13, 500, 111, torch.float16), (150, 256, 130, torch.float32),
                                                (333, 320, 192, torch.bfloat16), (16, 1000, 111, torch.float16),
                                                (5, 324, 130, torch.float32), (17, 640, 96, torch.bfloat16)])
def test_expert(cuda_ready, rows, k, inter, dtype):
    """The whole expert equals its four parts called one by one, and is within a bound of
    the 64-bit chain: h differs by at most its relative bound, so h's quantised value can
    differ (by one) only where the exact quotient is that close to a half; the output then
    moves by at most the sum of |w2| over those places times the scales."""
    from qmesh_b200.int8 import Int8Expert, int8_matmul, int8_swiglu, quant_int8
    w13, w2 = _expert(rows, k, inter)
    ex = Int8Expert.from_weights(w13.cuda(), w2.cuda())
    x = torch.randn(rows, k, generator=torch.Generator().manual_seed(rows + 1)).to(dtype)
    out = ex(x.cuda(), out_dtype=torch.float32)
    q, s = quant_int8(x.cuda())
    h = int8_swiglu(q, s, ex.w13, ex.w13_scale, out_dtype=torch.float32)
    q2, s2 = quant_int8(h)
    assert torch.equal(out, int8_matmul(q2, s2, ex.w2, ex.w2_scale, out_dtype=torch.float32))
    ws = ex.alloc_workspace(rows + 2)
    assert torch.equal(out, ex(x.cuda(), out_dtype=torch.float32, workspace=ws))
    # the 64-bit chain from the kernel's own q (exact or checked above) on
    g, u, hw = ref_swiglu(ref_product(q.cpu(), s.cpu(), ex.w13.cpu(), ex.w13_scale.cpu()), 10.0)
    rel = (2 + g.abs()) * D + 10 * U
    assert ((h.cpu().double() - hw).abs() <= (rel + U) * hw.abs() + 1e-42).all()
    m = hw.abs().amax(1, keepdim=True).clamp(min=TINY)
    t = 127.0 * hw / m
    # the quotient moves by its own and the maximum's relative bound, and 127 x rounds once
    close_to_half = ((t - torch.floor(t) - 0.5).abs() <= t.abs() * (rel + rel.amax(1, keepdim=True) + 4 * U)).double()
    w2q, w2s = ex.w2.cpu().double(), ex.w2_scale.cpu().double()
    want = torch.round(t) @ w2q.T * (m / 127.0) * w2s
    slack = close_to_half @ w2q.abs().T * (m / 127.0) * w2s
    err = (out.cpu().double() - want).abs()
    tol = slack + (want.abs() + slack) * (D + rel.amax(1, keepdim=True) + 2 * U)
    assert (err <= tol).all(), float((err / tol).max())


@pytest.mark.parametrize("rows", [1, 7, 16, 40])
def test_expert_fp8_rows_strides_and_nan_rows(cuda_ready, rows):
    """The expert on the slice's FP8 rows, on strided rows, and with a NaN row, against its
    four parts; a row that is not finite is NaN, is reported, and leaves the others alone."""
    from qmesh_b200 import _lib
    from qmesh_b200.int8 import Int8Expert, device_status, int8_matmul, int8_swiglu, quant_int8
    w13, w2 = _expert(2, 336, 80)
    ex = Int8Expert.from_weights(w13.cuda(), w2.cuda(), swiglu_limit=3.0)

    def parts(x, xs=None):
        h = int8_swiglu(*quant_int8(x, xs), ex.w13, ex.w13_scale, swiglu_limit=3.0, out_dtype=torch.float32)
        return int8_matmul(*quant_int8(h), ex.w2, ex.w2_scale, out_dtype=torch.float32)

    g = torch.Generator().manual_seed(rows)
    x = torch.randn(rows, 336, generator=g)
    x8 = (x * 30).to(torch.float8_e4m3fn).cuda()
    device_status()
    for xs in (torch.rand(rows, generator=g).cuda() + 0.1, torch.rand(1, generator=g).cuda() + 0.1):
        assert torch.equal(ex(x8, xs, out_dtype=torch.float32), parts(x8, xs))
    wide = torch.zeros(rows, 400, device="cuda")
    for lead in (0, 4, 3):
        view = wide[:, lead:lead + 336]
        view.copy_(x)
        assert torch.equal(ex(view, out_dtype=torch.float32), parts(view))
    assert device_status() == 0
    clean = ex(x.cuda())
    x[rows // 2, 5] = float("inf")
    out = ex(x.cuda())
    assert device_status() == _lib.QX_DEV_NONFINITE
    keep = torch.arange(rows) != rows // 2
    assert out[rows // 2].isnan().all() and torch.equal(out[keep], clean[keep])


def test_expert_after_its_weights_are_written(cuda_ready):
    """Weights that the work right in front of the call writes: the call's copies must not
    run ahead of it (a captured chain: quantise the weights, then the expert)."""
    from qmesh_b200.int8 import Int8Expert, quant_int8
    for rows in (4, 40, 300):
        w = [_expert(s, 2048, 512) for s in (1, 2)]
        w13, w2 = w[0][0].cuda(), w[0][1].cuda()
        q13, s13 = quant_int8(w13)
        q2, s2 = quant_int8(w2)
        ex = Int8Expert(q13, s13, q2, s2)
        x = torch.randn(rows, 2048, generator=torch.Generator().manual_seed(3)).to(torch.bfloat16).cuda()
        out, ws = torch.empty_like(x), ex.alloc_workspace(rows)
        ex(x, out=out, workspace=ws)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            quant_int8(w2, q=q2, scale=s2)
            quant_int8(w13, q=q13, scale=s13)
            ex(x, out=out, workspace=ws)
        for a, b in (w[1], w[0], w[1]):
            w13.copy_(a)
            w2.copy_(b)
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, Int8Expert.from_weights(a.cuda(), b.cuda())(x))


def test_expert_graph_streams_and_empty_batch(cuda_ready):
    """Captured and replayed on new inputs, on a side stream, and for no rows at all."""
    from qmesh_b200.int8 import Int8Expert
    w13, w2 = _expert(5, 320, 96)
    ex = Int8Expert.from_weights(w13.cuda(), w2.cuda())
    g = torch.Generator().manual_seed(8)
    xs = [torch.randn(9, 320, generator=g).to(torch.bfloat16).cuda() for _ in range(3)]
    want = [ex(x) for x in xs]
    x, out, ws = xs[0].clone(), torch.empty(9, 320, dtype=torch.bfloat16, device="cuda"), ex.alloc_workspace(9)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ex(x, out=out, workspace=ws)
    torch.cuda.synchronize()
    assert torch.equal(out, want[0])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ex(x, out=out, workspace=ws)
    for xi, wi in zip(xs, want):
        x.copy_(xi)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, wi)
    assert ex(xs[0][:0]).shape == (0, 320)


def test_far_offsets(cuda_ready):
    """A row stride that puts rows past 2^31 bytes (and the output past 2^31 elements)."""
    from qmesh_b200.int8 import int8_matmul
    stride = 1 << 30
    buf = torch.zeros(3 * stride, dtype=torch.int8, device="cuda")
    qa, sa, _, dsa = rows_of(4, 3, 160)
    da = torch.as_strided(buf, (3, 160), (stride, 1))
    da.copy_(qa)
    qw, sw, dw, dsw = rows_of(5, 40, 160, 0.02)
    want = ref_product(qa, sa, qw, sw)
    close(int8_matmul(da, dsa, dw, dsw, out_dtype=torch.float32), want, D, torch.float32)
    close(int8_matmul(dw, dsw, da, dsa, out_dtype=torch.float32), want.T, D, torch.float32)
    del buf, da
    out = torch.as_strided(torch.zeros(3 * stride, dtype=torch.bfloat16, device="cuda"), (3, 40), (stride, 1))
    int8_matmul(rows_of(4, 3, 160)[2], dsa, dw, dsw, out=out)
    close(out, want, D, torch.bfloat16)


@pytest.mark.parametrize("m", [3, 50, 300])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_outputs_inside_aligned_rows(cuda_ready, m, dtype):
    """Output rows on 16-byte boundaries whose last column lies inside a 16-byte piece:
    the columns behind it are left as they were."""
    from qmesh_b200.int8 import int8_matmul, int8_swiglu
    k = 160
    for n in (1, 2, 3, 7, 9, 31, 33, 63, 100, 129, 250, 1003):
        width = (n + 63) // 64 * 64 + 64
        _, _, da, dsa = rows_of(n, m, k)
        _, _, dw, dsw = rows_of(n + 1, 2 * n, k, 0.02)
        for call, w, s in ((int8_matmul, dw[:n], dsw[:n]), (int8_swiglu, dw, dsw)):
            buf = torch.full((m + 1, width), 7.0, dtype=dtype, device="cuda")
            call(da, dsa, w, s, out=buf[:m, :n])
            assert torch.equal(buf[:m, :n], call(da, dsa, w, s, out_dtype=dtype))
            buf[:m, :n] = 7.0
            assert (buf == 7.0).all(), f"n={n}"
