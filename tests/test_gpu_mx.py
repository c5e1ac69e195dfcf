"""Quantisation to microscaled floating point, bit for bit against its definition in 64 bits, and the products of such operands: on numbers
whose sums are exact, bit for bit as well."""
import math

import pytest
import torch

from dhellam_amd import _lib
from tests import mx_reference as R
from dhellam_amd.operators.mx import MXTensor, mx_gemm_nt, mx_quantise

pytestmark = pytest.mark.gpu

FORMS = ["e4m3", "e2m1"]


def matrix(rows, cols, dtype, seed, spread=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(spread * torch.randn(rows, 1, generator=g, device="cuda"))
    return (x * torch.exp(0.5 * torch.randn(1, cols, generator=g, device="cuda"))).to(dtype)


def same(q, x, form, rule):
    codes, scales = R.quantise(x, form, rule)
    assert (q.rows, q.cols, q.format) == (*x.shape, form)
    assert q.scales.shape == scales.shape and torch.equal(q.scales, scales), (q.scales != scales).nonzero()[:5]
    assert q.codes.shape == codes.shape and torch.equal(q.codes, codes), (q.codes != codes).nonzero()[:5]


SHAPES = [(1, 1), (1, 32), (3, 33), (4, 128), (5, 129), (31, 8), (127, 250), (128, 128), (129, 257), (300, 1000), (1, 8192), (1999, 1001), (8192, 3),
          (260, 4096)]


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("form", FORMS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
def test_quantise_bits(rows, cols, form, dtype):
    x = matrix(rows, cols, dtype, rows * 7 + cols)
    for rule in ("floor", "cover"):
        q, ms = mx_quantise(x, form, "rows", rule)
        assert ms == 0
        same(q, x, form, rule)
        t, _ = mx_quantise(x, form, "columns", rule)
        same(t, x.t(), form, rule)
        (a, b), _ = mx_quantise(x, form, "both", rule)
        assert torch.equal(a.codes, q.codes) and torch.equal(a.scales, q.scales)
        assert torch.equal(b.codes, t.codes) and torch.equal(b.scales, t.scales)


@pytest.mark.parametrize("form", FORMS)
def test_quantise_special_values(form):
    """Every half-way point and its neighbours, zeros of both signs, the smallest and largest numbers, infinities and NaN."""
    g = R.grid(form)
    half = ((g[1:] + g[:-1]) / 2).float()
    points = torch.cat([g.float(), half, torch.nextafter(half, half + 1), torch.nextafter(half, half - 1)])
    points = torch.cat([points, -points])
    rows = torch.zeros(9, up32 := R.up(len(points), 32))
    rows[0, :len(points)] = points
    rows[0, 0::32] = R.TOP[form]                                    # every block has scale 1
    rows[1] = rows[0] * 2.0 ** -100
    rows[2] = rows[0] * 2.0 ** 110
    rows[3] = rows[0] * 2.0 ** -126                                 # subnormal numbers, scales at their lowest
    rows[4] = torch.full((up32,), -0.0)
    rows[5] = torch.finfo(torch.float32).max
    rows[6] = 1e-45
    rows[7, 5], rows[7, 40] = float("inf"), float("nan")
    rows[8] = rows[0] * 1.1
    rows[8, -1] = -float("inf")
    x = rows.cuda()
    for rule in ("floor", "cover"):
        same(mx_quantise(x, form, "rows", rule)[0], x, form, rule)
        same(mx_quantise(x, form, "columns", rule)[0], x.t(), form, rule)
        for low in (x[:3].bfloat16(), x[7:].bfloat16(), x[:1].half()):
            same(mx_quantise(low, form, "both", rule)[0][0], low, form, rule)


def test_quantise_views_and_leading_dimensions():
    x = matrix(50, 700, torch.bfloat16, 3)
    for view in (x[:, 3:130], x[::2], x[7:8, 1:], x[:, 5:6]):
        (a, b), _ = mx_quantise(view, "e4m3", "both")
        same(a, view, "e4m3", "floor")
        same(b, view.t(), "e4m3", "floor")
    y = matrix(24, 96, torch.float32, 4)
    q, _ = mx_quantise(y.view(2, 3, 4, 96), "e2m1")
    same(q, y, "e2m1", "floor")
    q, _ = mx_quantise(y[0], "e2m1")
    same(q, y[:1], "e2m1", "floor")
    (a, b), _ = mx_quantise(x[:0], "e4m3", "both")
    assert a.codes.shape == (0, 768) and b.codes.shape == (700, 0) and (a.rows, b.cols) == (0, 0)


def exact_operand(rows, cols, form, seed):
    """Small numbers under scales 1 and 2: products are multiples of 1/4 of at most 144, and 2^24 / 576 = 29127 of them add up
    exactly in fp32 in any order."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    small = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
    pick = torch.randint(0, 16, (rows, R.up(cols, 128)), generator=g, device="cuda")
    if form == "e2m1":
        elements = pick.to(torch.uint8)
    else:
        table = torch.tensor(small + [-v for v in small], device="cuda")
        elements = table[pick].to(torch.float8_e4m3fn).view(torch.uint8)
    elements[:, cols:] = 0
    s = torch.randint(127, 129, (rows, R.up(cols, 128) // 32), generator=g, device="cuda")
    return MXTensor(R.pack(elements, form).contiguous(), R.lay_out(s, rows), rows, cols, form)


PRODUCTS = [(1, 1, 1), (1, 1000, 160), (1, 7168, 8192), (3, 17, 128), (16, 16, 384), (17, 65, 130), (24, 8192, 3584), (33, 100, 4096), (64, 64, 64), (65, 129, 257),
            (130, 1000, 512), (256, 256, 256), (257, 512, 640), (777, 1001, 2080), (300, 2048, 8192), (1999, 520, 1000), (2048, 2304, 1152), (520, 8200, 384),
            (32, 1280, 4096), (130, 300, 8192), (2050, 4400, 640), (4100, 2300, 128), (2200, 4111, 1032)]


def test_products_reach_every_kernel():
    path = lambda s, fa, fb, out: _lib.load().dh_mx_gemm_path(*s, FORMS.index(fa), FORMS.index(fb), out)
    seen = {path(s, fa, fb, out) // 100 for s in PRODUCTS for fa in FORMS for fb in FORMS for out in (0, 1)}
    assert seen == {11, 12, 22, 42, 44, 128, 256}
    assert {path(s, "e4m3", "e4m3", out) % 100 > 1 for s in PRODUCTS for out in (0, 1) if path(s, "e4m3", "e4m3", out) // 100 == 128} == {False, True}
    assert {path(s, "e4m3", "e4m3", 1) % 100 > 1 for s in PRODUCTS if path(s, "e4m3", "e4m3", 1) // 100 < 100} == {False, True}


@pytest.mark.parametrize("m,n,k", PRODUCTS)
@pytest.mark.parametrize("fa", FORMS)
@pytest.mark.parametrize("fb", FORMS)
def test_product_bits(m, n, k, fa, fb):
    a, b = exact_operand(m, k, fa, 1), exact_operand(n, k, fb, 2)
    want = R.values(a) @ R.values(b).t()
    assert want.abs().max() < 2 ** 22
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        got = mx_gemm_nt(a, b, out_dtype=dtype)
        assert got.dtype == dtype and got.shape == (m, n)
        wrong = (got != want.to(dtype)).nonzero()
        assert len(wrong) == 0, (dtype, len(wrong), wrong[:5], wrong[-5:])
    old = torch.randint(-64, 64, (m, n), generator=torch.Generator(device="cuda").manual_seed(3), device="cuda")
    for dtype in (torch.float32, torch.bfloat16, torch.float16):
        out = old.to(dtype)
        assert mx_gemm_nt(a, b, out=out, accumulate=True) is out
        assert torch.equal(out, (want + old).to(dtype))


@pytest.mark.parametrize("m,n,k", [(1, 2048, 8192), (100, 520, 1024), (1999, 1001, 520), (2304, 2048, 1024), (2050, 4400, 1024)])
@pytest.mark.parametrize("fa,fb", [("e4m3", "e4m3"), ("e4m3", "e2m1"), ("e2m1", "e2m1")])
def test_product_of_quantised_data(m, n, k, fa, fb):
    """Elements have few bits and scales are powers of two: products are exact.  fp32 results are sums of fp32: should every addition round, each of k
    loses 2^-24 of S = sum |a||b| at most, and where signs differ at random the norm of the error is that of the sums' roundings, far below 2^-20.
    16-bit results come from sums that drop, of 16 products, what is 2^-13 below the largest: 16 2^-13 of a group's largest and with it of the group's
    sum of magnitudes at most; in the norm over random signs sqrt(16) 2^-13 / sqrt(12) of the largest, and less than 2^-12 of the result."""
    a, _ = mx_quantise(matrix(m, k, torch.bfloat16, 5), fa)
    b, _ = mx_quantise(matrix(n, k, torch.bfloat16, 6, 0.1) * 0.02, fb, "rows", "cover")
    va, vb = R.values(a), R.values(b)
    got, want, size = mx_gemm_nt(a, b, out_dtype=torch.float32).double(), va @ vb.t(), va.abs() @ vb.abs().t()
    assert ((got - want).abs() <= k * 2.0 ** -24 * size).all()
    assert (got - want).norm() <= 2.0 ** -20 * want.norm()
    for dtype in (torch.bfloat16, torch.float16):
        half, low = torch.finfo(dtype).eps / 2, mx_gemm_nt(a, b, out_dtype=dtype).double()
        tiny = torch.finfo(dtype).tiny * 2 * half
        assert ((low - want).abs() <= 2.0 ** -9 * size + k * 2.0 ** -24 * size + half * (want.abs() + 2.0 ** -8 * size) + tiny).all()
        assert (low - want).norm() <= (half + 2.0 ** -12) * want.norm()


@pytest.mark.parametrize("m,n", [(1, 40), (40, 100), (300, 300), (2304, 2048), (2050, 4400)])
@pytest.mark.parametrize("fa,fb", [("e4m3", "e2m1"), ("e2m1", "e2m1"), ("e4m3", "e4m3")])
def test_product_not_finite_and_extreme_scales(m, n, fa, fb):
    k = 512
    a, b = exact_operand(m, k, fa, 7), exact_operand(n, k, fb, 8)
    want = R.values(a) @ R.values(b).t()
    row, col = m - 1, n // 2
    a.scales[2, row // 4, 1, row % 4] = 255
    b.scales[0, col // 4, 3, col % 4] = 255
    want[row, :], want[:, col] = float("nan"), float("nan")
    got = mx_gemm_nt(a, b, out_dtype=torch.float32)
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(0), want.nan_to_num(0).float())
    a, b = exact_operand(m, k, fa, 7), exact_operand(n, k, fb, 8)
    want = R.values(a) @ R.values(b).t()
    a.scales += 100
    b.scales -= 120
    assert torch.equal(mx_gemm_nt(a, b, out_dtype=torch.float32), (want * 2.0 ** -20).float())


def test_product_into_views_leaves_the_rest():
    for m, n in ((5, 33), (70, 130), (1000, 520), (2304, 2050), (2050, 4401)):
        a, b = exact_operand(m, 384, "e4m3", 9), exact_operand(n, 384, "e2m1", 10)
        want = R.values(a) @ R.values(b).t()
        for dtype in (torch.float32, torch.bfloat16):
            for left, right in ((0, 0), (1, 6), (8, 8), (4, 3)):
                whole = torch.full((m + 2, left + n + right), 7.0, dtype=dtype, device="cuda")
                view = whole[1:m + 1, left:left + n]
                mx_gemm_nt(a, b, out=view)
                assert torch.equal(view, want.to(dtype))
                view.fill_(7.0)
                assert (whole == 7.0).all()


def test_product_of_nothing():
    a, b = exact_operand(5, 128, "e4m3", 1), exact_operand(7, 128, "e4m3", 2)
    none = lambda rows, cols, form: MXTensor(torch.empty(rows, R.up(cols, 128), dtype=torch.uint8, device="cuda"),
                                             torch.empty(R.up(cols, 128) // 128, R.up(rows, 4) // 4, 4, 4, dtype=torch.uint8, device="cuda"), rows, cols, form)
    assert mx_gemm_nt(none(0, 128, "e4m3"), b).shape == (0, 7)
    assert mx_gemm_nt(a, none(0, 128, "e4m3")).shape == (5, 0)
    assert (mx_gemm_nt(none(5, 0, "e4m3"), none(7, 0, "e4m3")) == 0).all()
    out = torch.ones(5, 7, device="cuda")
    assert (mx_gemm_nt(none(5, 0, "e4m3"), none(7, 0, "e4m3"), out=out, accumulate=True) == 1).all()


@pytest.mark.parametrize("shape", [(5, 0), (0, 5), (0, 0), (2, 0, 3), (3, 2, 0)])
@pytest.mark.parametrize("form", ["e4m3", "e2m1"])
def test_matrices_of_nothing(shape, form):
    """No rows or no columns: operands of those sizes in either direction, whose products are empty or zero."""
    x = torch.empty(shape, device="cuda")
    rows, cols = math.prod(shape[:-1]), shape[-1]
    (q, qt), _ = mx_quantise(x, form, along="both")
    for along, m in (("rows", q), ("columns", qt)):
        alone = mx_quantise(x, form, along=along)[0]
        assert (alone.rows, alone.cols) == (m.rows, m.cols) == ((rows, cols) if along == "rows" else (cols, rows))
        assert not m.codes.any() and not m.scales.any()
        got = mx_gemm_nt(m, mx_quantise(torch.ones(7, m.cols, device="cuda"))[0])
        assert got.shape == (m.rows, 7) and not got.any()


def test_product_twice_the_same_bits_other_streams_and_graphs():
    """Two graphs captured on one stream and calls in between: each product has its own workspace."""
    cases = [(1, 512, 8192), (40, 640, 4096), (300, 512, 8192), (2304, 2048, 1024)]
    ops = [(exact_operand(m, k, "e4m3", i), exact_operand(n, k, "e2m1", 20 + i)) for i, (m, n, k) in enumerate(cases)]
    want = [(R.values(a) @ R.values(b).t()).float() for a, b in ops]
    x = matrix(300, 700, torch.bfloat16, 11)
    qx = R.quantise(x, "e2m1")
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    graphs, outs = [], []
    for a, b in ops:
        mx_gemm_nt(a, b, out_dtype=torch.float32, stream=stream)
        mx_quantise(x, "e2m1", stream=stream)
        stream.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=stream):
            outs.append((mx_gemm_nt(a, b, out_dtype=torch.float32), mx_quantise(x, "e2m1")[0]))
        graphs.append(graph)
    for _ in range(3):
        for o, q in outs:
            o.zero_()
            q.codes.zero_()
        for graph in graphs:
            graph.replay()
        for (a, b), w in zip(ops, want):
            assert torch.equal(mx_gemm_nt(a, b, out_dtype=torch.float32), w)
        for (o, q), w in zip(outs, want):
            assert torch.equal(o, w) and torch.equal(q.codes, qx[0]) and torch.equal(q.scales, qx[1])
