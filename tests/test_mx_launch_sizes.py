"""Sizes past what one launch holds (2^32 - 1 threads) are refused by name, before anything is launched (no GPU needed)."""
import ctypes as C

from dhellam_amd import _lib

P = 4096      # an address that is never read


def _lib_():
    if not _lib.LIB_PATH.exists():
        from dhellam_amd.build import build
        build()
    return _lib.load()


def _refused(rc, text):
    assert rc == -1 and text in _lib.load().dh_last_error().decode(), (rc, _lib.load().dh_last_error())


def test_quantise():
    lib = _lib_()
    call = lambda rows, cols: lib.dh_mx_quantise(P, rows, cols, cols, 1, 0, 0, None, None, P, P, None)
    _refused(call((1 << 31) - 1, 1), "tiles")
    _refused(call(1, (1 << 31) - 1), "tiles")
    _refused(call(1 << 19, 1 << 19), "tiles")


def test_product():
    lib = _lib_()
    call = lambda m, n, fb: lib.dh_mx_gemm_nt(P, P, 0, P, P, fb, P, m, n, 128, n, 1, 0, P, 1 << 62, None)
    _refused(call(1, 1 << 28, 1), "tiles")
    _refused(call(16, 1 << 28, 0), "tiles")
    _refused(call(20, (1 << 28) + 1, 0), "tiles")


def test_gradients():
    lib = _lib_()
    arr = lambda t, *v: (t * len(v))(*v)
    n = 1 << 38
    _refused(lib.dh_grad_norm(arr(C.c_void_p, P, P), arr(C.c_int64, 8, n), arr(C.c_int, 1, 1), 2, P, P, 1 << 62, None), "too large")
    _refused(lib.dh_grad_clip(arr(C.c_void_p, P, P), arr(C.c_void_p, P, P), arr(C.c_int64, 8, n), arr(C.c_int, 1, 1), arr(C.c_int, 1, 1), 2, P, 1.0, 1.0, P, None),
             "too large")
