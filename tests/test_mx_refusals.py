"""What the C entries of the microscaled operators and of the gradients' norm and clipping refuse, and their operators off the GPU (no GPU
needed: every check is made on the host before anything is launched)."""
import ctypes as C

import pytest
import torch

from dhellam_amd import _lib
from dhellam_amd.operators.grads import clip_grads, grad_norm
from dhellam_amd.operators.layernorm import pyrmsnorm_mx_fwd
from dhellam_amd.operators.mx import MXTensor, mx_gemm_nt, mx_quantise


def _lib_():
    if not _lib.LIB_PATH.exists():
        from dhellam_amd.build import build
        build()
    return _lib.load()


def _refused(rc, text):
    assert rc == -1 and text in _lib.load().dh_last_error().decode(), (rc, _lib.load().dh_last_error())


P = 4096      # an address that is never read: every one of these calls is refused before anything is launched


def test_quantise_refusals():
    lib = _lib_()
    call = lambda x=P, rows=4, cols=64, ldx=64, dtype=1, form=0, c=P, s=P, ct=None, st=None: lib.dh_mx_quantise(
        x, rows, cols, ldx, dtype, form, 0, c, s, ct, st, None)
    _refused(call(rows=-1), "rows")
    _refused(call(form=2), "format")
    _refused(call(dtype=3), "dtype")
    _refused(call(rows=1 << 31), "2^31")
    _refused(call(cols=1 << 31, ldx=1 << 31), "2^31")
    _refused(call(rows=(1 << 31) - 1, cols=1 << 20, ldx=1 << 20), "tiles")
    _refused(call(x=None), "null")
    _refused(call(c=None, s=None), "null")
    _refused(call(s=None), "pairs")
    _refused(call(ct=P), "pairs")
    _refused(call(ldx=63), "stride")
    _refused(call(c=P + 8), "aligned")
    _refused(call(ct=P, st=P + 4), "aligned")
    assert call(rows=0, x=None) == 0 and call(cols=0, x=None) == 0


def test_norm_refusals():
    lib = _lib_()
    call = lambda x=P, r=None, t=None, g=P, c=P, s=P, rs=P, rows=4, cols=64, dtype=1: lib.dh_rmsnorm_mx(x, r, t, g, None, c, s, rs, rows, cols, 1e-5, 0, 0, dtype, None)
    _refused(call(cols=-1), "cols")
    _refused(call(dtype=9), "dtype")
    _refused(call(cols=(1 << 24) + 1), "cols")
    _refused(call(rows=1 << 31), "rows")
    _refused(call(g=None), "null")
    _refused(call(rs=None), "null")
    _refused(call(r=P), "residual")
    _refused(call(t=P), "residual")
    _refused(call(c=P + 4), "aligned")
    assert call(rows=0, x=None) == 0


def test_product_refusals():
    lib = _lib_()
    call = lambda a=P, sa=P, fa=0, b=P, sb=P, fb=1, c=P, m=300, n=300, k=256, ldc=300, dtype=1, ws=None, wsb=0: lib.dh_mx_gemm_nt(
        a, sa, fa, b, sb, fb, c, m, n, k, ldc, dtype, 0, ws, wsb, None)
    _refused(call(m=-1), "m -1")
    _refused(call(k=(1 << 22) + 1), "k")
    _refused(call(m=1 << 31), "m")
    _refused(call(m=(1 << 31) - 1, n=1 << 20, ldc=1 << 20), "tiles")
    _refused(call(fa=2), "format")
    _refused(call(dtype=5), "dtype")
    _refused(call(c=None), "null")
    _refused(call(ldc=299), "stride")
    _refused(call(a=None), "null")
    _refused(call(sb=None), "null")
    _refused(call(b=P + 8), "aligned")
    _refused(call(m=1 << 30, k=1 << 12), "2 GiB")
    need = lib.dh_mx_gemm_workspace_bytes(1, 64, 1 << 16, 0, 1, 1)
    assert need > 0 and lib.dh_mx_gemm_workspace_bytes(0, 8, 8, 0, 1, 1) == 0 and lib.dh_mx_gemm_workspace_bytes(-1, 8, 8, 0, 1, 1) == 0
    _refused(call(m=1, n=64, k=1 << 16), "workspace")
    _refused(call(m=1, n=64, k=1 << 16, ws=P, wsb=need - 1), "workspace")
    assert call(m=0, c=None) == 0 and call(n=0, c=None, ldc=0) == 0


def test_gradient_refusals():
    lib = _lib_()
    arr = lambda t, *v: (t * len(v))(*v)
    norm = lambda p=P, n=8, dtype=0, out=P, ws=P, wsb=64: lib.dh_grad_norm(arr(C.c_void_p, p), arr(C.c_int64, n), arr(C.c_int, dtype), 1, out, ws, wsb, None)
    _refused(norm(n=-1), "elements")
    _refused(norm(dtype=4), "dtype")
    _refused(norm(p=None), "null")
    _refused(norm(out=None), "bad list")
    _refused(norm(ws=None), "workspace")
    _refused(norm(wsb=7), "workspace")
    _refused(norm(n=1 << 50, wsb=1 << 60), "too large")
    assert lib.dh_grad_norm_workspace_bytes(arr(C.c_int64, 1, 0, 32769), 3) == 24
    clip = lambda p=P, o=P, n=8, dtype=1, odtype=1, ss=P, max_norm=1.0, scale=1.0, found=P: lib.dh_grad_clip(
        arr(C.c_void_p, p), arr(C.c_void_p, o), arr(C.c_int64, n), arr(C.c_int, dtype), arr(C.c_int, odtype), 1, ss, max_norm, scale, found, None)
    _refused(clip(ss=None), "bad list")
    _refused(clip(found=None), "bad list")
    _refused(clip(max_norm=-1.0), "max_norm")
    _refused(clip(max_norm=float("nan")), "max_norm")
    _refused(clip(scale=float("inf")), "scale")
    _refused(clip(odtype=2), "own type")
    _refused(clip(dtype=0, odtype=1), "own type")
    _refused(clip(o=None), "null")
    _refused(clip(n=-3), "elements")


def test_operators_refuse_what_is_not_on_the_gpu():
    x = torch.zeros(4, 128)
    q = MXTensor(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 1, 4, 4, dtype=torch.uint8), 4, 128, "e4m3")
    for call in (lambda: mx_quantise(x), lambda: mx_gemm_nt(q, q), lambda: pyrmsnorm_mx_fwd(x, x[0], 1e-5, False), lambda: grad_norm([x]),
                 lambda: clip_grads([x], torch.zeros(1, dtype=torch.float64), 1.0)):
        with pytest.raises(RuntimeError, match="GPU"):
            call()


def test_operators_refuse_names_and_sizes():
    x = torch.zeros(4, 128)
    q = MXTensor(torch.zeros(4, 128, dtype=torch.uint8), torch.zeros(1, 1, 4, 4, dtype=torch.uint8), 4, 128, "e4m3")
    with pytest.raises(RuntimeError, match="format 'e5m2'"):
        mx_quantise(x, "e5m2")
    with pytest.raises(RuntimeError, match="along"):
        mx_quantise(x, along="row")
    with pytest.raises(RuntimeError, match="scale_rule"):
        mx_quantise(x, scale_rule="ceil")
    with pytest.raises(RuntimeError, match="scale_rule"):
        pyrmsnorm_mx_fwd(x, x[0], 1e-5, False, scale_rule="ceil")
    with pytest.raises(RuntimeError, match="columns"):
        mx_gemm_nt(q, MXTensor(q.codes, q.scales, 4, 64, "e4m3"))
    with pytest.raises(RuntimeError, match="format"):
        mx_gemm_nt(q, MXTensor(q.codes, q.scales, 4, 128, "fp8"))
