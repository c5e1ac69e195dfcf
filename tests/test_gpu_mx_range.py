"""Products of microscaled operands whose scales lie at the ends of their range."""
import pytest
import torch

from tests import mx_reference as R
from tests.test_gpu_mx import FORMS, exact_operand
from dhellam_amd.operators.mx import mx_gemm_nt

pytestmark = pytest.mark.gpu

SIZES = [(3, 40, 512), (130, 300, 512), (600, 520, 1024), (2304, 2048, 1152)]


def shifted(rows, cols, form, seed, by):
    q = exact_operand(rows, cols, form, seed)
    q.scales += by % 256
    return q


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("fa,fb", [("e4m3", "e4m3"), ("e4m3", "e2m1"), ("e2m1", "e2m1")])
@pytest.mark.parametrize("da,db", [(-60, -66), (-60, -75), (-120, -10), (-20, -100)])
def test_results_around_the_smallest_normal_number(m, n, k, fa, fb, da, db):
    """Multiples of 2^-2 2^(da + db), which fp32 holds exactly, below its normal numbers too: no product or sum is lost."""
    a, b = shifted(m, k, fa, 7, da), shifted(n, k, fb, 8, db)
    want = (R.values(exact_operand(m, k, fa, 7)) @ R.values(exact_operand(n, k, fb, 8)).t()) * 2.0 ** (da + db)
    assert (want != 0).any() and want.abs().max() < 2.0 ** (da + db + 22)
    for dtype in (torch.float32, torch.bfloat16):
        assert torch.equal(mx_gemm_nt(a, b, out_dtype=dtype), want.to(dtype))


@pytest.mark.parametrize("m,n,k", SIZES)
@pytest.mark.parametrize("fa", FORMS)
@pytest.mark.parametrize("fb", FORMS)
def test_elements_past_fp32(m, n, k, fa, fb):
    """Elements times their scale from 2^128 on: 16-bit results, and fp32 ones of two 4-bit operands, are those of the sums; other fp32 results
    take such elements as infinite."""
    a, b = shifted(m, k, fa, 7, 126), shifted(n, k, fb, 8, -126)
    want = R.values(exact_operand(m, k, fa, 7)) @ R.values(exact_operand(n, k, fb, 8)).t()
    assert R.values(a).abs().max() >= 2.0 ** 128
    assert torch.equal(mx_gemm_nt(a, b, out_dtype=torch.bfloat16), want.bfloat16())
    got = mx_gemm_nt(a, b, out_dtype=torch.float32)
    if fa == fb == "e2m1":
        assert torch.equal(got, want.float())
    else:
        assert not got.isfinite().any()
