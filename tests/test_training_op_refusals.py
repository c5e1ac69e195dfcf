"""What the C entries of the rotary positions, the router's losses and the distillation loss refuse, and their operators off the GPU (no
GPU needed: every check is made on the host before anything is launched)."""
import math

import pytest
import torch

from dhellam_amd import _lib
from dhellam_amd.operators.rope import rotary_table


def _lib_():
    if not _lib.LIB_PATH.exists():
        from dhellam_amd.build import build
        build()
    return _lib.load()


def _refused(rc, text):
    assert rc == -1 and text in _lib.load().dh_last_error().decode(), (rc, _lib.load().dh_last_error())


P = 4096      # an address that is never read: every one of these calls is refused before anything is launched


def test_rotary_refusals():
    lib = _lib_()
    call = lambda tokens=4, hq=2, hk=1, d=8, rot=8, q=P, steps=P, pos=None, pos_bytes=0, dtype=1: lib.dh_rotary(
        q, P, P, P, steps, pos, pos_bytes, tokens, hq, hk, d, rot, 16, 8, 8, 8, 16, 8, 8, 8, 0, 0, 0, 1.0, dtype, None)
    _refused(call(tokens=-1), "bad shape")
    _refused(call(d=0), "bad shape")
    _refused(call(rot=3), "even")
    _refused(call(rot=0), "even")
    _refused(call(rot=10), "even")
    _refused(call(q=None), "null")
    _refused(call(steps=None), "steps")
    _refused(call(pos=P, pos_bytes=2), "positions")
    _refused(call(dtype=7), "dtype")
    assert call(tokens=0, q=None, steps=None) == 0 and call(hq=0, hk=0) == 0


def test_balance_refusals():
    lib = _lib_()
    fwd = lambda tokens=4, e=8, k=2, logits=P, losses=P, ws=None, ws_bytes=0: lib.dh_balance_loss_fwd(
        logits, P, None, tokens, e, k, 1.0, 0.0, losses, P, P, P, P, ws, ws_bytes, None)
    _refused(fwd(e=65), "experts")
    _refused(fwd(e=0), "experts")
    _refused(fwd(k=9, e=16), "k=9")
    _refused(fwd(k=3, e=2), "k=3")
    _refused(fwd(tokens=-1), "tokens")
    _refused(fwd(tokens=1 << 28), "tokens")
    _refused(fwd(logits=None), "null")
    _refused(fwd(losses=None), "null")
    need = lib.dh_balance_loss_workspace_bytes(100000, 64)
    assert need > 0 and lib.dh_balance_loss_workspace_bytes(1, 8) == 0 and lib.dh_balance_loss_workspace_bytes(0, 8) == 0
    _refused(fwd(tokens=100000, e=64), "workspace")
    _refused(fwd(tokens=100000, e=64, ws=P, ws_bytes=need - 1), "workspace")
    bwd = lambda tokens=4, e=8, k=2, gates=P, dgates=P, lse=P, counts=P, out=P: lib.dh_moe_route_bwd(
        P, P, gates, dgates, None, lse, counts, P, None, tokens, e, k, 1.0, 0.0, out, None)
    _refused(bwd(e=65), "experts")
    _refused(bwd(k=0), "k=0")
    _refused(bwd(gates=None), "dgates without gates")
    _refused(bwd(counts=None), "counts")
    _refused(bwd(dgates=None, lse=None), "neither")
    _refused(bwd(out=None), "null")
    assert bwd(tokens=0, out=None) == 0


def test_distill_refusals():
    lib = _lib_()

    def call(back, rows=4, cols=16, k=2, ld=16, logits=P, idb=8, td=0, target=P, start=0, total=16, tau=1.0, alpha=0.5, dtype=1, pitch=4,
             ws=None, nbytes=0, dout=P, grad=P + 4096, ldg=16):
        if back:
            return lib.dh_distill_bwd(logits, ld, P, idb, P, td, target, P, pitch, dout, rows, cols, k, start, total, tau, alpha, dtype, grad, ldg, None)
        return lib.dh_distill_fwd(logits, ld, P, idb, P, td, None, target, rows, cols, k, start, total, tau, alpha, dtype, P, pitch, ws, nbytes, None)
    for back in (False, True):
        _refused(call(back, rows=-1), "rows")
        _refused(call(back, cols=0), "rows")
        _refused(call(back, ld=15), "ld")
        _refused(call(back, rows=1 << 24, pitch=1 << 24), "rows")
        _refused(call(back, k=0), "entries")
        _refused(call(back, k=1025), "entries")
        _refused(call(back, idb=2), "ids")
        _refused(call(back, td=5), "teacher dtype")
        _refused(call(back, dtype=5), "dtype")
        _refused(call(back, start=8), "vocabulary")
        _refused(call(back, start=-1), "vocabulary")
        for tau in (0.0, -1.0, math.nan, math.inf):
            _refused(call(back, tau=tau), "temperature")
        for alpha in (-0.1, 1.1, math.nan):
            _refused(call(back, alpha=alpha), "alpha")
        _refused(call(back, target=None), "without targets")
        _refused(call(back, logits=None), "null")
        _refused(call(back, pitch=3), "pitch")
        assert call(back, rows=0, target=None, logits=None, pitch=0) == 0
    _refused(call(True, dout=None), "dout")
    _refused(call(True, ldg=15), "ld_grad")
    _refused(call(True, grad=P + 16), "overlap")
    _refused(call(True, grad=P, ldg=32), "overlap")
    need = lib.dh_distill_workspace_bytes(2, 100000)
    assert need > 0 and lib.dh_distill_workspace_bytes(0, 100000) == 0
    _refused(call(False, rows=2, cols=100000, ld=100000, total=100000, ws=P, nbytes=need - 1), "workspace")


@pytest.mark.parametrize("where", ["rotary", "balance", "route_bwd", "distill"])
def test_operands_off_the_gpu_are_refused(where):
    from dhellam_amd.operators.loss import distill_fwd
    from dhellam_amd.operators.moe import balance_loss_fwd, route_bwd
    from dhellam_amd.operators.rope import rotary_fwd
    x, idx = torch.zeros(4, 2, 8), torch.zeros(4, 2, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="GPU"):
        if where == "rotary":
            rotary_fwd(x, x, rotary_table(10000.0, 8, "cpu"))
        elif where == "balance":
            balance_loss_fwd(x[:, 0], idx)
        elif where == "route_bwd":
            route_bwd(x[:, 0], idx, x[:, 0, :2], x[:, 0, :2])
        else:
            distill_fwd({"vocab_parallel_logits": x[:, 0], "teacher_ids": idx, "teacher_logits": x[:, 0, :2]})
