"""The waits of the distillation's backward in the assembly that is built (no GPU needed): what a run cannot show, for the memory
keeps the order nearly always."""
import re
import subprocess

import pytest

from dhellam_amd import build as B


def test_barriers_of_global_memory_wait_for_it(tmp_path):
    """A workgroup clears its bits (LDS), reads the listed logits, lets no wavefront store before they are there where the gradient takes their
    place, and corrects the listed columns behind all stores: three barriers, the last two behind a wait for global memory."""
    out = tmp_path / "distill.s"
    flags = [f for f in B.CXXFLAGS if f != "-fPIC"]
    try:
        res = subprocess.run([B.HIPCC, *flags, "--cuda-device-only", "-S", str(B.CSRC / "distill.hip"), "-o", str(out)], capture_output=True, text=True)
    except FileNotFoundError:
        pytest.skip("no hipcc")
    assert res.returncode == 0, res.stderr
    lines = [l.split(";")[0].strip() for l in out.read_text().split("\n")]
    starts = [i for i, l in enumerate(lines) if re.match(r"^_ZN2dh\w*distill_bwd_kernel\w+:", l)]
    assert len(starts) == 3 * 4 * 3                       # types, exponentials, (64 threads, 256, 256 past the caches)
    for at in starts:
        body = lines[at:next(i for i in range(at, len(lines)) if lines[i].startswith(".Lfunc_end"))]
        barriers = [i for i, l in enumerate(body) if l.startswith("s_barrier")]
        if len(barriers) == 0:                            # one wavefront: its barriers order its own accesses
            assert "Li64E" in lines[at]
            waits = [l for l in body if re.match(r"s_waitcnt.*vmcnt\(0\)", l)]
            assert len(waits) >= 2
            continue
        assert len(barriers) == 3, (lines[at], len(barriers))
        for b in barriers[1:]:
            before = [l for l in body[max(0, b - 6):b] if l.startswith("s_waitcnt")]
            assert any("vmcnt(0)" in l for l in before), (lines[at], body[b - 6:b + 1])
            assert not any(re.match(r"(global|buffer|flat)_(load|store)", l) for l in body[b - 3:b]), body[b - 3:b]
