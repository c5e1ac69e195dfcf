"""The RMS norm that writes 8 bits with scales, against 64 bits."""
import pytest
import torch

from tests import mx_reference as R
from dhellam_amd.operators.layernorm import pylayernorm_fwd, pyrmsnorm_mx_fwd

pytestmark = pytest.mark.gpu

EPS = 1e-5
SHAPES = [(1, 1), (1, 8192), (3, 33), (5, 100), (64, 512), (7, 520), (130, 1000), (33, 1024), (9, 1032), (30, 2047), (17, 2048), (6, 2056), (65, 4096), (10, 5120),
          (3, 8192), (4, 8200), (2, 16384), (3, 16392), (5, 40000), (2500, 300)]


def inputs(rows, cols, dtype, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g, device="cuda") * torch.exp(torch.randn(rows, 1, generator=g, device="cuda"))).to(dtype)
    r = (torch.randn(rows, cols, generator=g, device="cuda") * 2).to(dtype)
    return x, r, (1 + 0.1 * torch.randn(cols, generator=g, device="cuda")).to(dtype)


def check(q, rsigma, held, gamma, shift, rule):
    """y = x rsigma gamma in fp32: rsigma of a sum of squares of one sign, added 32 at most behind one another and then in trees, is off by 2^-19,
    a product by 2^-24 each: y by less than 2^-18 |y|.  A scale is the rule's for some such y, and an element the nearest one under it:
    half a step, 2^-4 of itself or 2^-10 of the scale, past the largest the largest."""
    rows, cols = held.shape
    rs = torch.rsqrt(held.double().square().mean(1) + EPS)
    assert ((rsigma.double() - rs).abs() <= 2.0 ** -19 * rs).all()
    y = held.double() * rs[:, None] * (gamma.double() + shift)
    near = 2.0 ** -18
    lo, hi = R.scale_codes(y * (1 - near), "e4m3", rule), R.scale_codes(y * (1 + near), "e4m3", rule)
    s = q.scales.permute(1, 3, 0, 2).reshape(-1, lo.shape[1])
    assert (s[rows:] == 0).all()
    s = s[:rows].long()
    assert ((s == lo) | (s == hi)).all()
    scale = R.power(s - 127).repeat_interleave(32, 1)
    got, y = R.values(q), torch.nn.functional.pad(y, (0, R.up(cols, 128) - cols))
    assert (q.codes[:, cols:] == 0).all()
    y = y.clamp(-448 * scale, 448 * scale)
    assert ((got - y).abs() <= torch.maximum(2.0 ** -4 * y.abs(), 2.0 ** -10 * scale) * (1 + 2.0 ** -10) + 2 * near * y.abs()).all()


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("residual", [False, True])
def test_norm(rows, cols, dtype, residual):
    x, r, gamma = inputs(rows, cols, dtype, rows + cols)
    for rule, centered in (("floor", False), ("cover", True)):
        y = torch.empty_like(x)
        q, rsigma, total, ms = pyrmsnorm_mx_fwd(x, gamma, EPS, centered, residual=r if residual else None, ln_out=y, scale_rule=rule)
        held = (x.float() + r.float()).to(dtype) if residual else x
        assert ms == 0 and (q.rows, q.cols, q.format) == (rows, cols, "e4m3") and (total is None) == (not residual)
        if residual:
            assert torch.equal(total, held)
        check(q, rsigma, held, gamma, 1.0 if centered else 0.0, rule)
        # the norm in the input's type, from the same fp32 values up to their last bits
        ref = pylayernorm_fwd(held, gamma, None, EPS, 0, centered, None)[0]
        half = torch.finfo(dtype).eps / 2
        assert ((y.double() - ref.double()).abs() <= (2 * half + 2.0 ** -17) * ref.double().abs() + 2 * torch.finfo(dtype).tiny).all()
        again = pyrmsnorm_mx_fwd(x, gamma, EPS, centered, residual=r if residual else None, scale_rule=rule)
        assert torch.equal(again[0].codes, q.codes) and torch.equal(again[0].scales, q.scales) and torch.equal(again[1], rsigma)


def test_norm_in_place_not_finite_and_leading_dimensions():
    for cols in (520, 8192, 20000):
        x, r, gamma = inputs(12, cols, torch.bfloat16, 5)
        want = pyrmsnorm_mx_fwd(x, gamma, EPS, False, residual=r)
        for target in (x.clone(), r.clone()):
            a, b = (target, r) if torch.equal(target, x) else (x, target)
            got = pyrmsnorm_mx_fwd(a, gamma, EPS, False, residual=b, sum_out=target)
            assert got[2] is target and torch.equal(target, want[2]) and torch.equal(got[0].codes, want[0].codes)
        got = pyrmsnorm_mx_fwd(x.view(3, 4, cols), gamma, EPS, False, residual=r.view(3, 4, cols))
        assert torch.equal(got[0].codes, want[0].codes) and got[2].shape == (3, 4, cols)
        x[2, 5], x[7, cols - 1] = float("nan"), float("inf")
        bad = pyrmsnorm_mx_fwd(x, gamma, EPS, False, residual=r)
        v = R.values(bad[0])[:, :cols]
        fine = [i for i in range(12) if i not in (2, 7)]
        assert torch.equal(bad[0].codes[fine], want[0].codes[fine]) and v[2].isnan().all() and v[7, cols - 1].isnan()
        assert (bad[0].codes[2] == 0).all()
        zero = pyrmsnorm_mx_fwd(torch.zeros_like(x), gamma, EPS, False)
        assert (zero[0].codes & 127 == 0).all() and (zero[0].scales == 0).all()
    empty = pyrmsnorm_mx_fwd(x[:0], gamma, EPS, False)
    assert empty[0].codes.shape[0] == 0 and empty[1].numel() == 0
    with pytest.raises(AssertionError):
        pyrmsnorm_mx_fwd(x[:, :0].contiguous(), gamma[:0], EPS, False)


@pytest.mark.parametrize("rows,cols,dtype", [(1999, 1000, torch.float32), (512, 8192, torch.bfloat16), (128, 16384, torch.float16), (1024, 4096, torch.bfloat16),
                                             (64, 40000, torch.bfloat16)])
@pytest.mark.parametrize("centered,rule", [(False, "floor"), (True, "cover")])
def test_codes_are_those_of_64_bits(rows, cols, dtype, centered, rule):
    """y is off by 2^-43 of itself, and an element's boundaries lie a 16th of it apart: of 17 million elements in all these cases 3e-5 are expected to differ.
    (In fp32 throughout it would be some 10; with the squares alone added in fp32, 2.)"""
    x, _, gamma = inputs(rows, cols, dtype, 71)
    q = pyrmsnorm_mx_fwd(x, gamma, EPS, centered, scale_rule=rule)[0]
    held = x.double()
    eps = torch.tensor(EPS, dtype=torch.float32).double().item()
    y = held / torch.sqrt(held.square().mean(1, keepdim=True) + eps) * (gamma.double() + (1.0 if centered else 0.0))
    codes, scales = R.quantise(y, "e4m3", rule)
    assert torch.equal(q.scales, scales)
    assert (((q.codes ^ codes) == 0) | (((q.codes | codes) & 127) == 0)).all()      # (zeros of either sign)


def test_norm_of_products_past_the_smallest_number():
    """x rsigma gamma below every fp32 number: zeros, of either sign."""
    x = torch.randn(8, 256, device="cuda")
    gamma = torch.full((256,), 1e-38, device="cuda")
    x[:, ::2] *= 1e-30
    q = pyrmsnorm_mx_fwd(x, gamma, EPS, False)[0]
    assert (q.scales != 255).all() and (q.codes[:, :256:2] & 127 == 0).all() and R.values(q).isfinite().all()


def test_norm_captured():
    x, r, gamma = inputs(33, 1000, torch.bfloat16, 9)
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    pyrmsnorm_mx_fwd(x, gamma, EPS, False, stream, residual=r)
    stream.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=stream):
        q, rsigma, total, _ = pyrmsnorm_mx_fwd(x, gamma, EPS, False, residual=r)
    for i in range(3):
        x.mul_(1.25)
        graph.replay()
        want = pyrmsnorm_mx_fwd(x, gamma, EPS, False, residual=r)
        assert torch.equal(q.codes, want[0].codes) and torch.equal(q.scales, want[0].scales) and torch.equal(rsigma, want[1]) and torch.equal(total, want[2])
