"""The RMS norm that writes 8 bits with scales over the whole range of its types: rows whose mean square or 1/rms lies past fp32's numbers,
results below them, infinities."""
import math

import pytest
import torch

from tests import mx_reference as R
from dhellam_amd.operators.layernorm import pyrmsnorm_mx_fwd

pytestmark = pytest.mark.gpu

# one of every way a row is dealt out: single wavefronts, 256 and 1024 threads, the form of any length; whole groups of 8 columns and ragged
SHAPES = [(6, 264), (7, 1000), (9, 2056), (300, 3333), (300, 5120), (3, 8192), (5, 10001), (3, 16392), (5, 40000)]
BLOCK = 32


def randn(rows, cols, seed):
    return torch.randn(rows, cols, generator=torch.Generator(device="cuda").manual_seed(seed), device="cuda")


def exact(held, gamma, shift, eps):
    """1/rms and the result in 64 bits, with eps as fp32 holds it."""
    rs = 1 / torch.sqrt(held.double().square().mean(1, keepdim=True) + torch.tensor(eps, dtype=torch.float32).double().item())
    return rs[:, 0], held.double() * rs * (gamma.double() + shift)


def same_codes(q, y, rule):
    codes, scales = R.quantise(y, "e4m3", rule)
    assert torch.equal(q.scales, scales)
    assert (((q.codes ^ codes) == 0) | (((q.codes | codes) & 127) == 0)).all()      # (zeros of either sign)


def check(x, gamma, eps, residual=None, centered=False, rule="floor"):
    """Codes and scales: of 64 bits.  rsigma: rounded to fp32 once (half a step, 2^-24 of itself or 2^-150), beside 2^-43 in 64 bits."""
    q, rsigma, total, _ = pyrmsnorm_mx_fwd(x, gamma, eps, centered, residual=residual, scale_rule=rule)
    held = x if residual is None else (x.float() + residual.float()).to(x.dtype)
    assert total is None or torch.equal(total, held)
    rs, y = exact(held, gamma, 1.0 if centered else 0.0, eps)
    same_codes(q, y, rule)
    past = rs > torch.finfo(torch.float32).max
    assert torch.equal(rsigma.isinf(), past)
    assert ((rsigma.double() - rs).abs()[~past] <= 2.0 ** -24 * (1 + 2.0 ** -18) * rs[~past] + 2.0 ** -150).all()
    return q, rsigma, y


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("size,eps", [(1e25, 1e-5), (5e37, 1e-5), (1e-22, 0.0), (1e-30, 0.0), (2e-40, 0.0)])
def test_rows_past_the_squares_of_fp32(rows, cols, dtype, size, eps):
    x = (randn(rows, cols, rows + cols) * size).to(dtype)
    assert x.isfinite().all()
    gamma = (1 + 0.1 * randn(1, cols, 3)[0]).to(dtype)
    for residual in (None, (randn(rows, cols, 5) * size * 0.25).to(dtype)):
        check(x, gamma, eps, residual)
    check(x, (gamma.float() - 1).to(dtype), eps, centered=True, rule="cover")


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_one_row_among_others_and_a_subnormal_rsigma(dtype):
    for cols in (1000, 5120, 20000):
        x, gamma = randn(300, cols, 1).to(dtype), (1 + 0.1 * randn(1, cols, 3)[0]).to(dtype)
        x[7] = torch.sign(x[7]) * 3e38                             # 1/rms is below fp32's normal numbers
        x[9] = (randn(1, cols, 8)[0] * 1e20).to(dtype)
        _, rsigma, _ = check(x, gamma, 1e-5)
        assert 0 < rsigma[7].item() < torch.finfo(torch.float32).tiny


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_infinity_in_a_row(rows, cols, dtype):
    """1/rms of the row is 0: zeros where it is finite, NaN in the block of the infinity alone."""
    x = randn(rows, cols, 7).to(dtype)
    gamma = (1 + 0.1 * randn(1, cols, 3)[0]).to(dtype)
    for at in (0, cols // 2, cols - 1):
        for value in (math.inf, -math.inf):
            bad = x.clone()
            bad[2, at] = value
            y = torch.empty_like(bad)
            q, rsigma, _, _ = pyrmsnorm_mx_fwd(bad, gamma, 1e-5, False, ln_out=y)
            assert rsigma[2].item() == 0 and (rsigma[torch.arange(rows) != 2] > 0).all()
            v = R.values(q)[2, :cols]
            block = torch.arange(cols, device="cuda") // BLOCK == at // BLOCK
            assert v[block].isnan().all() and (v[~block] == 0).all()
            assert y[2, at].isnan() and (y[2, torch.arange(cols) != at] == 0).all()
            same_codes(q, exact(bad, gamma, 0.0, 1e-5)[1], "floor")


@pytest.mark.parametrize("rows,cols", SHAPES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_factors_and_results_below_the_normal_numbers(rows, cols, dtype):
    """Blocks of x whose quotient by rms is subnormal in fp32 while gamma brings it back; results that are subnormal themselves."""
    x, gamma = randn(rows, cols, 11), 1 + 0.1 * randn(1, cols, 3)[0]
    small = torch.where((torch.arange(cols, device="cuda") // BLOCK) % 2 == 1, 3e-39, 1.0)
    mixed = (x * small).to(dtype)
    check(mixed, (gamma * 1e30).to(dtype), 1e-5)
    for size in (1e-38, 1e-39, 1e-41):
        check(x.to(dtype), (gamma * size).to(dtype), 1e-5)
    one = gamma.clone()
    one[cols // 3] = 1e33
    check(mixed, one.to(dtype), 1e-5, rule="cover")
    one[cols // 2] = math.inf
    check(mixed, one.to(dtype), 1e-5)


@pytest.mark.parametrize("rows,cols,dtype", [(1999, 1000, torch.float32), (512, 8192, torch.bfloat16), (128, 16384, torch.float16), (1024, 4096, torch.bfloat16),
                                             (64, 40000, torch.bfloat16)])
@pytest.mark.parametrize("residual", [False, True])
def test_codes_rsigma_and_result_at_ordinary_sizes(rows, cols, dtype, residual):
    """Codes of 64 bits with a residual as well.  y: rsigma and gamma + 1 rounded, two products: 2^-22 of itself, beside its rounding to the type."""
    x = (randn(rows, cols, 71) * torch.exp(randn(rows, 1, 2))).to(dtype)
    r = (randn(rows, cols, 72) * 2).to(dtype) if residual else None
    gamma = (0.1 * randn(1, cols, 73)[0]).to(dtype)
    _, rsigma, want = check(x, gamma, 1e-5, r, centered=True)
    y = torch.empty_like(x)
    pyrmsnorm_mx_fwd(x, gamma, 1e-5, True, residual=r, ln_out=y)
    info = torch.finfo(dtype)
    half = info.eps / 2
    assert ((y.double() - want).abs() <= (half + 2.0 ** -22 * (1 + half)) * want.abs() + info.tiny * half).all()


def test_masked_rows():
    """Rows of zeros (padding) among others: zeros, scales of 2^-127, rsigma 1/sqrt(eps)."""
    for cols in (1000, 8192, 20000):
        x, gamma = randn(301, cols, 21).bfloat16(), (1 + 0.1 * randn(1, cols, 3)[0]).bfloat16()
        x[100:250] = 0
        x[3, : cols // 2] = 0
        q, rsigma, _ = check(x, gamma, 1e-5)
        assert (q.codes[100:250] == 0).all() and (rsigma[100:250] == rsigma[100]).all()
