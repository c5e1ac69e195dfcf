"""Which kernel a product of microscaled operands takes (no GPU needed: the rule is asked, nothing is launched)."""
import itertools

from dhellam_amd import _lib


def test_tiles_of_256_take_k_whole():
    """The kernel of 256 x 256 tiles has no split of k, and no rule gives it one; the others have 16 pieces at most, and a workspace for them."""
    if not _lib.LIB_PATH.exists():
        from dhellam_amd.build import build
        build()
    lib = _lib.load()
    sizes = [1, 16, 17, 33, 100, 128, 300, 512, 1000, 1999, 2048, 4096, 5000, 8192, 16384]
    seen = set()
    for m, n, k in itertools.product(sizes, sizes, (1, 128, 1000, 2080, 4096, 8192, 16384, 131072)):
        for fa, fb, out in ((0, 0, 1), (0, 1, 2), (1, 0, 1), (1, 1, 1), (0, 0, 0), (1, 1, 0)):
            side, pieces = divmod(lib.dh_mx_gemm_path(m, n, k, fa, fb, out), 100)
            seen.add(side)
            assert 1 <= pieces <= 16 and (side != 256 or pieces == 1)
            assert lib.dh_mx_gemm_workspace_bytes(m, n, k, fa, fb, out) == (pieces * m * ((n + 3) // 4 * 4) * 4 if pieces > 1 else 0)
    assert seen == {256, 128, 11, 12, 22, 42, 44}
