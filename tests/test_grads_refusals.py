"""What the C entries of the gradients' norm and clipping refuse anywhere in a list (no GPU needed: the whole list is looked at on the host
before anything is launched, so that a refused call has changed no gradient)."""
import ctypes as C

import pytest

from dhellam_amd import _lib

P = 4096      # an address that is never read
N = 200       # more than two launches take


def _lib_():
    if not _lib.LIB_PATH.exists():
        from dhellam_amd.build import build
        build()
    return _lib.load()


def _lists(at, pointer, count, dtype, out_pointer, out_dtype):
    values = [[P] * N, [8] * N, [1] * N, [P] * N, [1] * N]
    for v, x in zip(values, (pointer, count, dtype, out_pointer, out_dtype)):
        v[at] = x
    return [(t * N)(*v) for t, v in zip((C.c_void_p, C.c_int64, C.c_int, C.c_void_p, C.c_int), values)]


@pytest.mark.parametrize("at", [0, 79, 80, 100, N - 1])
@pytest.mark.parametrize("what,text", [(dict(dtype=7, out_dtype=7), "dtype"), (dict(pointer=None), "null"), (dict(count=-2), "elements"),
                                       (dict(count=1 << 50), "too large"), (dict(count=(1 << 63) - 1), "too large")])
def test_lists_of_either_entry(at, what, text):
    lib = _lib_()
    g, n, t, o, ot = _lists(at, **{**dict(pointer=P, count=8, dtype=1, out_pointer=P, out_dtype=1), **what})
    for rc in (lambda: lib.dh_grad_norm(g, n, t, N, P, P, 1 << 62, None), lambda: lib.dh_grad_clip(g, o, n, t, ot, N, P, 1.0, 1.0, P, None)):
        assert rc() == -1 and text in lib.dh_last_error().decode() and f"tensor {at}" in lib.dh_last_error().decode()


@pytest.mark.parametrize("at", [0, 79, 80, 100, N - 1])
@pytest.mark.parametrize("what,text", [(dict(out_dtype=2), "own type"), (dict(out_pointer=None), "null")])
def test_results_of_the_clipping(at, what, text):
    lib = _lib_()
    g, n, t, o, ot = _lists(at, **{**dict(pointer=P, count=8, dtype=1, out_pointer=P, out_dtype=1), **what})
    assert lib.dh_grad_clip(g, o, n, t, ot, N, P, 1.0, 1.0, P, None) == -1
    assert text in lib.dh_last_error().decode() and f"tensor {at}" in lib.dh_last_error().decode()


@pytest.mark.parametrize("scale", [1e39, -1e39, 3.5e38])
def test_a_scale_past_fp32(scale):
    lib = _lib_()
    g, n, t, o, ot = _lists(0, P, 8, 1, P, 1)
    assert lib.dh_grad_clip(g, o, n, t, ot, N, P, 1.0, scale, P, None) == -1 and "scale" in lib.dh_last_error().decode()
