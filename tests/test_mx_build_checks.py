"""The generated code of the tiled products of microscaled operands keeps the order that the source lays down (no GPU needed)."""
import os
import shutil

import pytest

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")


@pytest.fixture(scope="module")
def kernels():
    from dhellam_amd.build import mx_gemm_assembly
    return mx_gemm_assembly()


def test_every_instantiation(kernels):
    from dhellam_amd.build import check_mx_gemm_order
    assert sum("mx_w8" in n for n in kernels) == 9 and sum("mx_t128" in n for n in kernels) == 12
    for name, fn in kernels.items():
        assert check_mx_gemm_order(name, fn) > 100


def test_a_missing_wait_or_barrier_is_found(kernels):
    """The first barrier between matrix instructions, the waits for reads and the waits for the last copies, taken out in turn.  (The compiler
    waits for some reads by itself as well, so all of these waits go.)"""
    from dhellam_amd.build import check_mx_gemm_order
    for name, fn in kernels.items():
        strip = [l.split(";")[0].strip() for l in fn]
        first, last = (f([i for i, l in enumerate(strip) if "v_mfma" in l]) for f in (min, max))
        half = (first + last) // 2
        bad = list(fn)
        bad[next(i for i in range(first, half) if strip[i] == "s_barrier")] = ""
        with pytest.raises(RuntimeError):
            check_mx_gemm_order(name, bad)
        bad = ["" if l == "s_waitcnt lgkmcnt(0)" else f for l, f in zip(strip, fn)]
        with pytest.raises(RuntimeError):
            check_mx_gemm_order(name, bad)
        bad = list(fn)
        for i in range(last, len(fn)):
            if strip[i].startswith("s_waitcnt vmcnt(0)"):
                bad[i] = ""
        with pytest.raises(RuntimeError):
            check_mx_gemm_order(name, bad)
