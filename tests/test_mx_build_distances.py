"""The generated code of the tiled products of microscaled operands: the slice behind the main loop keeps the order of the others, and instructions
from assembly keep their distance from what the compiler puts around them (no GPU needed)."""
import os
import re
import shutil

import pytest

pytestmark = pytest.mark.skipif(shutil.which("hipcc") is None and not os.path.exists("/opt/rocm/bin/hipcc"), reason="needs hipcc")


@pytest.fixture(scope="module")
def kernels():
    from dhellam_amd.build import mx_gemm_assembly
    return mx_gemm_assembly()


def _formats(kernels):
    """Every kernel with every pair of formats, for one type of its results."""
    return {n: f for n, f in kernels.items() if "DF16b" in n or "Lb1E" in n}


def _by_assembly(kernels):
    """Of the kernels whose products are assembly one of each kind of matrix instruction."""
    return {n: f for n, f in kernels.items() if "DF16b" in n and ("ILi8ELi8E" in n or "ILi4ELi4E" in n)}


def _plain(fn):
    return [l.split(";")[0].strip() for l in fn]


def _mfmas(fn):
    return [i for i, l in enumerate(_plain(fn)) if "v_mfma" in l]


def _operands(line):
    return re.split(r",\s*(?![^\[]*\])", line.split(None, 1)[1].split(" op_sel")[0])


def _first(operand):
    m = re.match(r"v\[(\d+):|v(\d+)", operand)
    return int(m.group(1) or m.group(2))


def test_as_built(kernels):
    from dhellam_amd.build import check_mx_gemm_distances, check_mx_gemm_order
    assert len(kernels) == 21
    for name, fn in kernels.items():
        assert check_mx_gemm_order(name, fn) > 100 and check_mx_gemm_distances(name, fn) > 30


def test_the_last_slice_keeps_the_order(kernels):
    """In the slice behind the main loop: a barrier away, its counted waits away, a copy among the matrix instructions."""
    from dhellam_amd.build import check_mx_gemm_order
    for name, fn in _formats(kernels).items():
        code, at = _plain(fn), _mfmas(fn)
        of_slice = len(at) // 3
        eight = "mx_w8" in name
        lo, hi = at[2 * of_slice - 1] + 1, at[-1]
        barriers = [i for i in range(lo, hi) if code[i].startswith("s_barrier")]
        assert len(barriers) == (8 if eight else 1)          # (with the one that ends the loop)
        for i in barriers:
            bad = list(fn)
            bad[i] = ""
            with pytest.raises(RuntimeError):
                check_mx_gemm_order(name, bad)
        waits = [i for i in range(lo, hi) if code[i].startswith("s_waitcnt vmcnt")]
        assert waits
        for i in waits:
            bad = list(fn)
            bad[i] = ""
            with pytest.raises(RuntimeError):
                check_mx_gemm_order(name, bad)
        copies = [i for i in range(lo, hi) if code[i].startswith("buffer_load")]
        assert copies
        bad = list(fn)
        bad[copies[0]] = ""
        with pytest.raises(RuntimeError, match="cop"):
            check_mx_gemm_order(name, bad)
        if eight:
            bad = list(fn)
            bad.insert(at[2 * of_slice + 3], fn[copies[0]])
            with pytest.raises(RuntimeError):
                check_mx_gemm_order(name, bad)


def test_the_first_slices_are_published(kernels):
    from dhellam_amd.build import check_mx_gemm_order
    for name, fn in _formats(kernels).items():
        code, first = _plain(fn), _mfmas(fn)[0]
        copies = [i for i in range(first) if code[i].startswith("buffer_load")]
        read = next(i for i in range(first) if code[i].startswith("ds_read"))
        for what in ("s_barrier", "s_waitcnt vmcnt"):
            bad = list(fn)
            bad[next(i for i in range(copies[0], read) if code[i].startswith(what))] = ""
            with pytest.raises(RuntimeError):
                check_mx_gemm_order(name, bad)


def test_an_operand_written_too_late_is_found(kernels):
    """Of several products in the loop and behind it: a vector instruction that writes a fragment's, a scale's or a sum's register before the
    product, at distances of 0 and 1; 2 is enough."""
    from dhellam_amd.build import check_mx_gemm_distances
    for name, fn in _by_assembly(kernels).items():
        at = _mfmas(fn)
        for i in (at[0], at[len(at) // 3], at[-1]):
            parts = _operands(_plain(fn)[i])
            for n in (1, 2, 4, 5):
                write = f"\tv_perm_b32 v{_first(parts[n])}, v0, v0, v0"
                for gap in ([], ["\ts_nop 0"]):
                    with pytest.raises(RuntimeError, match="operand"):
                        check_mx_gemm_distances(name, fn[:i] + [write] + gap + fn[i:])
            check_mx_gemm_distances(name, fn[:i] + [f"\tv_perm_b32 v{_first(parts[5])}, v0, v0, v0", "\ts_nop 1"] + fn[i:])


def test_a_sum_used_too_early_is_found(kernels):
    from dhellam_amd.build import check_mx_gemm_distances
    for name, fn in _by_assembly(kernels).items():
        i = _mfmas(fn)[-1]
        d = _first(_operands(_plain(fn)[i])[0])
        for line in (f"\tv_mov_b32_e32 v{d}, 0", f"\tv_add_f32_e32 v0, v0, v{d + 3}", f"\tglobal_store_dwordx4 v[0:1], v[{d}:{d + 3}], off"):
            with pytest.raises(RuntimeError, match="sum"):
                check_mx_gemm_distances(name, fn[:i + 1] + ["\ts_nop 7", line] + fn[i + 1:])
        # without the wait behind the last product the stores' preparation comes too early
        code = _plain(fn)
        waits = [j for j in range(i, len(fn)) if code[j] == "s_nop 15"][:2]
        assert len(waits) == 2
        behind = fn[:waits[0]] + [f"\tv_mov_b32_e32 v0, v{d}"] + fn[waits[1] + 1:]
        with pytest.raises(RuntimeError, match="sum"):
            check_mx_gemm_distances(name, behind)


def test_a_copy_behind_a_read_of_a_lane_is_found(kernels):
    from dhellam_amd.build import check_mx_gemm_distances
    for name, fn in _by_assembly(kernels).items():
        code = _plain(fn)
        i = next(j for j, l in enumerate(code) if l.startswith("buffer_load"))
        descriptor, offset = re.search(r"s\[(\d+):\d+\], (s\d+)", code[i]).groups()
        for register in (f"s{descriptor}", offset):
            with pytest.raises(RuntimeError, match="copy"):
                check_mx_gemm_distances(name, fn[:i] + [f"\tv_readlane_b32 {register}, v0, 1", "\ts_nop 3"] + fn[i:])
        check_mx_gemm_distances(name, fn[:i] + [f"\tv_readlane_b32 s{descriptor}, v0, 1", "\ts_nop 4"] + fn[i:])
