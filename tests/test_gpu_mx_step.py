"""Low precision as a training step uses it: the quantising norm, products forward and backward, weight gradients into ``main_grad``, the
global norm and clipping, against 64 bits on the same quantised operands and against differences."""
import math

import pytest
import torch

from dhellam_amd.operators.grads import clip_grads, grad_norm
from dhellam_amd.operators.layernorm import pylayernorm_bwd, pyrmsnorm_mx_fwd
from dhellam_amd.operators.mx import mx_gemm_nt, mx_quantise
from dhellam_amd.operators.swiglu import swiglu, swiglu_back
from tests import mx_reference as R

pytestmark = pytest.mark.gpu

EPS = 1e-5


def rel(a, b):
    return ((a.double() - b).norm() / b.norm()).item()


@pytest.mark.parametrize("tokens,hidden,ffn", [(1, 256, 384), (77, 520, 264), (512, 1024, 1408)])
@pytest.mark.parametrize("fw", ["e4m3", "e2m1"])
@pytest.mark.parametrize("main", [torch.float32, torch.bfloat16])
def test_feed_forward_block(tokens, hidden, ffn, fw, main):
    """h = a + r; y = norm(h); z = swiglu(y W1^T) W2^T, straight through the quantisations; two micro-batches into the same main_grad.

    Tolerances: what goes into a product is the same on both sides, what comes out is rounded to bf16 (2^-9 in the norm of the error on
    average, 2^-8 at most) and formed from sums that are off by less than 2^-12 of themselves in the norm; behind it the activation and its
    gradient are rounded once more, and quantised from there: what the reference quantises is the same rounded tensor."""
    g = torch.Generator(device="cuda").manual_seed(tokens)
    bf = torch.bfloat16
    draw = lambda *s, std=1.0: (torch.randn(*s, generator=g, device="cuda") * std).to(bf)
    gamma, w1, w2 = draw(hidden, std=0.1) + 1, draw(2 * ffn, hidden, std=0.05), draw(hidden, ffn, std=0.05)
    (q1, q1t), _ = mx_quantise(w1, fw, "both", "cover")
    (q2, q2t), _ = mx_quantise(w2, fw, "both", "cover")
    v1, v2, v1t, v2t = R.values(q1)[:, :hidden], R.values(q2)[:, :ffn], R.values(q1t)[:, :2 * ffn], R.values(q2t)[:, :hidden]
    g1, g2, ggamma = torch.zeros_like(w1, dtype=main), torch.zeros_like(w2, dtype=main), torch.zeros_like(gamma)
    want1, want2, wantg = (torch.zeros_like(t, dtype=torch.float64) for t in (w1, w2, gamma))
    tol = 1.5 * (2.0 ** -8 + 2.0 ** -12)
    for _ in range(2):
        a, r, dz = draw(tokens, hidden), draw(tokens, hidden), draw(tokens, hidden, std=0.1)
        # forward
        y_kept = torch.empty_like(a)
        y, rsigma, h, _ = pyrmsnorm_mx_fwd(a, gamma, EPS, False, residual=r, ln_out=y_kept)
        u = mx_gemm_nt(y, q1)
        act, _ = swiglu(u, None)
        (s, st), _ = mx_quantise(act, "e4m3", "both")
        z = mx_gemm_nt(s, q2)
        vy = R.values(y)[:, :hidden]
        assert rel(u, vy @ v1.t()) <= tol
        sv = R.values(s)[:, :ffn]
        assert rel(z, sv @ v2.t()) <= tol
        # backward
        (d, dt), _ = mx_quantise(dz, "e4m3", "both")
        dact = mx_gemm_nt(d, q2t)
        assert rel(dact, R.values(d)[:, :hidden] @ v2t.t()) <= tol
        mx_gemm_nt(dt, st, out=g2, accumulate=True)
        want2 += R.values(dt)[:, :tokens] @ R.values(st)[:, :tokens].t()
        du, _ = swiglu_back(dact, u, None, None)
        (e, et), _ = mx_quantise(du, "e4m3", "both")
        dy = mx_gemm_nt(e, q1t)
        assert rel(dy, R.values(e)[:, :2 * ffn] @ v1t.t()) <= tol
        yt, _ = mx_quantise(y_kept, "e4m3", "columns")
        mx_gemm_nt(et, yt, out=g1, accumulate=True)
        want1 += R.values(et)[:, :tokens] @ R.values(yt)[:, :tokens].t()
        dh, _, _, _ = pylayernorm_bwd(dy, h, None, rsigma, gamma, 0, False, None, add_to_dgrad=dz, dgamma_out=ggamma)
        h64, gam = h.double().requires_grad_(True), gamma.double().requires_grad_(True)
        n64 = h64 * torch.rsqrt(h64.square().mean(1, keepdim=True) + EPS) * gam
        dh64, dg64 = torch.autograd.grad(n64, (h64, gam), dy.double())
        assert rel(dh, dh64 + dz.double()) <= tol
        wantg += dg64
    gtol = 2.0 ** -18 if main == torch.float32 else 2 * tol       # two roundings of the sum in bf16
    assert rel(g1, want1) <= gtol and rel(g2, want2) <= gtol and rel(ggamma, wantg) <= 2 * tol
    grads = [g1, g2, ggamma]
    kept = [t.clone() for t in grads]
    norm = math.sqrt(sum(float(t.double().square().sum()) for t in grads)) / 8
    found, _ = clip_grads(grads, grad_norm(grads)[0], norm / 3, scale=1 / 8)
    assert abs(found[0].item() - norm) <= 1e-6 * norm and abs(found[1].item() - 1 / 24) <= 1e-5 / 24
    for t, k in zip(grads, kept):
        assert rel(t, k.double() / 24) <= 1e-5 + torch.finfo(t.dtype).eps / 2
    assert abs(math.sqrt(grad_norm(grads)[0].item()) - norm / 3) <= 1e-2 * norm


@pytest.mark.parametrize("m,n,k", [(5, 40, 96), (130, 200, 300)])
@pytest.mark.parametrize("fw", ["e4m3", "e2m1"])
def test_gradients_against_differences(m, n, k, fw):
    """Whole numbers that every format and both directions hold exactly: f = <dY, X W^T> is linear in X and in W, so its central differences are
    its derivatives, and sums below 2^24 are exact."""
    g = torch.Generator(device="cuda").manual_seed(m)
    small = lambda *s: torch.randint(-2, 3, s, generator=g, device="cuda").bfloat16()
    x, w, dy, dx_dir, dw_dir = small(m, k), small(n, k), small(m, n), small(m, k), small(n, k)
    q = lambda t, f, along="rows": mx_quantise(t, f, along, "cover")[0]
    f = lambda x, w: (mx_gemm_nt(q(x, "e4m3"), q(w, fw), out_dtype=torch.float32).double() * dy.double()).sum().item()
    (d, dt), (s, st) = q(dy, "e4m3", "both"), q(x, "e4m3", "both")
    dx = mx_gemm_nt(d, q(w, fw, "columns"), out_dtype=torch.float32)
    dw = mx_gemm_nt(dt, st, out=torch.ones(n, k, device="cuda"), accumulate=True) - 1
    assert torch.equal(R.values(s)[:, :k].float(), x.float())
    assert (dx.double() * dx_dir.double()).sum().item() == (f(x + dx_dir, w) - f(x - dx_dir, w)) / 2
    assert (dw.double() * dw_dir.double()).sum().item() == (f(x, w + dw_dir) - f(x, w - dw_dir)) / 2


def test_model_shells_clip_their_gradients():
    from dhellam_amd.core.dsllm import DSLLM, DSLLMStep, clip_main_grads, run_microbatches
    from dhellam_amd.core.dstb import LayerConfig
    cfg = LayerConfig(hidden_size=256, num_attention_heads=4, num_query_groups=2, ffn_hidden_size=192, seq_length=64, micro_batch_size=1,
                      params_dtype=torch.bfloat16)
    ids = torch.randint(0, 100, (1, 65), device="cuda")
    batch = {"token_ids": ids[:, :-1].contiguous(), "labels": ids[:, 1:].contiguous(), "loss_mask": torch.ones(1, 64, device="cuda")}
    step, shell = DSLLMStep(cfg, 2, 100), DSLLM(cfg, 100, 2)
    step.step([batch, batch], loss_scale=16.0)
    run_microbatches(shell, [batch, batch])
    for params, clip in (([t for _, t in step.named_parameters()], lambda *a: step.clip_grads(*a)),
                         ([p for p in shell.parameters() if getattr(p, "main_grad", None) is not None], lambda *a: clip_main_grads(shell.parameters(), *a))):
        kept = [p.main_grad.clone() for p in params]
        norm = math.sqrt(sum(float(t.double().square().sum()) for t in kept)) / 16
        assert norm > 0
        found = clip(norm / 4, 1 / 16)
        assert abs(found[0].item() - norm) <= 1e-6 * norm
        for p, k in zip(params, kept):
            assert (p.main_grad.double() - k.double() / 64).abs().max() <= 2.0 ** -8 * (k.double() / 64).abs().max() + 1e-30
    with pytest.raises(ValueError, match="main_grad"):
        clip_main_grads([torch.zeros(3, device="cuda")], 1.0)


def test_binding_names_and_elapsed_time():
    from dhellam_amd import _Clib
    x, gamma = torch.randn(64, 256, device="cuda").bfloat16(), torch.ones(256, device="cuda").bfloat16()
    q, ms = _Clib.pymx_quantise(x, profiling=True)
    a, b = _Clib.pymx_quantise(x, "e2m1", "both")
    assert ms > 0 and (a.rows, b.rows) == (64, 256) and _Clib.pymx_gemm_nt(q, q).shape == (64, 64)
    n, rsigma, total, ms = _Clib.pyrmsnorm_mx_fwd(x, gamma, EPS, x, True)
    assert ms > 0 and total.shape == x.shape and rsigma.shape == (64,) and n.format == "e4m3"
    (s,), (f, ms) = _Clib.pygrad_norm([x]), _Clib.pyclip_grads([x], _Clib.pygrad_norm([x])[0], 1.0, profiling=True)
    assert s.dtype == torch.float64 and f.shape == (2,) and ms > 0
