"""Microscaled operators and the gradients' norm past 32 bits of offset."""
import pytest
import torch

from dhellam_amd.operators.grads import clip_grads, grad_norm
from dhellam_amd.operators.layernorm import pyrmsnorm_mx_fwd
from dhellam_amd.operators.mx import MXTensor, mx_gemm_nt, mx_quantise
from tests import mx_reference as R

pytestmark = pytest.mark.gpu


def halves(rows, cols, seed):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = torch.empty(rows, cols, dtype=torch.bfloat16, device="cuda")
    for part in x.split(8192):
        part.copy_(torch.randn(part.shape, generator=g, device="cuda"))
    return x


def nibbles(rows, cols, seed):
    """Any 4-bit elements under scales of 1: products are multiples of 1/4 of at most 36, sums of 8192 of them exact."""
    g = torch.Generator(device="cuda").manual_seed(seed)
    codes = torch.randint(0, 256, (rows, cols // 2), generator=g, device="cuda", dtype=torch.uint8)
    return MXTensor(codes, torch.full((cols // 128, (rows + 3) // 4, 4, 4), 127, dtype=torch.uint8, device="cuda"), rows, cols, "e2m1")


def rows_of(q, lo, hi):
    """Rows lo..hi (lo a multiple of 4) as a matrix of their own."""
    return MXTensor(q.codes[lo:hi].contiguous(), q.scales[:, lo // 4:(hi + 3) // 4].contiguous(), hi - lo, q.cols, q.format)


def test_quantise():
    x = halves(33001, 70001, 1)
    assert x.numel() > 2 ** 31
    (q, qt), _ = mx_quantise(x, "e4m3", "both")
    last = 32900
    codes, scales = R.quantise(x[last:], "e4m3")
    assert torch.equal(q.codes[last:], codes) and torch.equal(q.scales[:, last // 4:], scales)
    codes, scales = R.quantise(x[:, 69996:].t(), "e4m3")
    assert torch.equal(qt.codes[69996:], codes) and torch.equal(qt.scales[:, 69996 // 4:], scales)


def test_norm():
    x, gamma = halves(140000, 16384, 2), halves(1, 16384, 3)[0]
    assert x.numel() > 2 ** 31
    q, rsigma, total, _ = pyrmsnorm_mx_fwd(x, gamma, 1e-5, False, residual=x, ln_out=None)
    end, r, t, _ = pyrmsnorm_mx_fwd(x[-8:].contiguous(), gamma, 1e-5, False, residual=x[-8:].contiguous())
    assert torch.equal(q.codes[-8:], end.codes) and torch.equal(q.scales[:, -2:], end.scales) and torch.equal(rsigma[-8:], r) and torch.equal(total[-8:], t)


@pytest.mark.parametrize("m,n", [(600000, 40), (600000, 256), (1, 600000), (40, 600000)])
def test_products_of_large_operands(m, n):
    k = 8192
    a, b = nibbles(m, k, 4), nibbles(n, k, 5)
    assert max(a.codes.numel(), b.codes.numel()) > 2 ** 31
    got = mx_gemm_nt(a, b, out_dtype=torch.float32)
    for lo in (0, 299996, 599900):
        ra, rb = (rows_of(a, lo, lo + 100), b) if m > n else (a, rows_of(b, lo, lo + 100))
        part = got[lo:lo + 100] if m > n else got[:, lo:lo + 100]
        assert torch.equal(part.double(), R.values(ra) @ R.values(rb).t())


def test_products_of_large_results():
    a, b = nibbles(70000, 128, 6), nibbles(40000, 128, 7)
    got = mx_gemm_nt(a, b)
    assert got.numel() > 2 ** 31
    for lo in (0, 35000, 69900):
        assert torch.equal(got[lo:lo + 100], (R.values(rows_of(a, lo, lo + 100)) @ R.values(b).t()).bfloat16())


def test_gradients():
    x = halves(33000, 70000, 8).view(-1)
    sum_sq, _ = grad_norm([x, x[:5]])
    want = sum(float(p.double().square().sum()) for p in x.split(1 << 28)) + float(x[:5].double().square().sum())
    assert abs(sum_sq.item() - want) <= 1e-9 * want
    first, end = x[:1000].clone(), x[-1000:].clone()
    found, _ = clip_grads([x], sum_sq, 1.0, scale=2.0 ** 20)
    factor = float(2 ** 20 * min(1.0, 1.0 / (2 ** 20 * want ** 0.5 + 1e-6)))
    for kept, now in ((first, x[:1000]), (end, x[-1000:])):
        # half a step of bf16, 8 significant bits, is 2^-8 of the value at most; the factor and the product in fp32 add 2^-23
        assert ((now.double() - kept.double() * factor).abs() <= (2.0 ** -8 + 2.0 ** -22) * (kept.double() * factor).abs()).all()
