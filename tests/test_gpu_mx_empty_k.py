"""Products over no columns whose results take more than one round of a launch of a limited size."""
import pytest
import torch

from dhellam_amd.operators.mx import MXTensor, mx_gemm_nt

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("m,n", [(40001, 7001), (3, 5)])
def test_zeros_everywhere(m, n):
    none = lambda rows: MXTensor(torch.empty(rows, 0, dtype=torch.uint8, device="cuda"), torch.empty(0, (rows + 3) // 4, 4, 4, dtype=torch.uint8, device="cuda"),
                                 rows, 0, "e4m3")
    whole = torch.full((m + 2, n + 3), 7.0, dtype=torch.bfloat16, device="cuda")
    mx_gemm_nt(none(m), none(n), out=whole[1:m + 1, 2:n + 2])
    assert (whole[1:m + 1, 2:n + 2] == 0).all()
    whole[1:m + 1, 2:n + 2] = 7.0
    assert (whole == 7.0).all()
