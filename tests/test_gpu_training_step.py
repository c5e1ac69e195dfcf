"""Rotary positions, router losses and the distillation loss where they are used: in the decoder layer, in the head block, and together in
one step of a small mixture model, against 64-bit autograd."""
import math

import pytest
import torch

from dhellam_amd.operators.rope import rotary_frequencies
from oracle import layer as OL
from tests.util import assert_close, rel_err

pytestmark = pytest.mark.gpu

PARTS = {"kind": "parts", "factor": 4.0, "original_length": 64}


def turn(x, at, theta, rot, interleaved, scaling):
    """[tokens, heads, d] in 64 bits, pair by pair."""
    f, factor = rotary_frequencies(theta, rot, scaling)
    angle = at.double()[:, None] * torch.tensor(f, dtype=torch.float64, device=x.device)
    c, s = (torch.cos(angle) * factor)[:, None], (torch.sin(angle) * factor)[:, None]
    a, b = (x[..., 0:rot:2], x[..., 1:rot:2]) if interleaved else (x[..., :rot // 2], x[..., rot // 2:rot])
    a, b = a * c - b * s, b * c + a * s
    front = torch.stack((a, b), -1).flatten(-2) if interleaved else torch.cat((a, b), -1)
    return torch.cat((front, x[..., rot:]), -1)


@pytest.mark.parametrize("groups,cp,strands", [(1, 1, 1), (2, 1, 1), (4, 1, 2), (1, 2, 1), (2, 2, 2), (1, 1, 2)])
@pytest.mark.parametrize("rot,interleaved,scaling", [(None, True, None), (24, False, None), (16, True, PARTS), (None, False, {"kind": "linear", "factor": 4.0})])
def test_layer_with_other_rotary_positions(groups, cp, strands, rot, interleaved, scaling, monkeypatch):
    """One kv group (turned as views of the packed projection) and several (inside attention), plain and round the ring, serial and double
    strand: every form runs where the halves of whole heads do."""
    from dhellam_amd.core.dstb import LayerConfig
    from dhellam_amd.core.layer import LayerRunner, make_microbatch, make_weights
    cfg = LayerConfig(hidden_size=256, num_attention_heads=4, num_query_groups=groups, ffn_hidden_size=192, seq_length=64, micro_batch_size=2,
                      context_parallel_size=cp, cp_rank=cp - 1, params_dtype=torch.float32, rotary_dim=rot, rotary_interleaved=interleaved,
                      rope_scaling=scaling)
    assert cfg.general_rotary
    w, mbs = make_weights(cfg, 0), [make_microbatch(cfg, i) for i in range(strands)]
    w_cpu = {k: v.detach().cpu() for k, v in w.items() if v.is_floating_point()}
    mb_cpu = [{k: v.detach().cpu() if isinstance(v, torch.Tensor) else [t.cpu() for t in v] for k, v in mb.items()} for mb in mbs]
    runner = LayerRunner(cfg, w)
    outs, dxs = (runner.run_double_strand if strands == 2 else runner.run_serial)(mbs)
    torch.cuda.synchronize()
    monkeypatch.setattr(OL.O, "rope", lambda x, at, theta, dtype=torch.float64: turn(x.to(dtype), at, theta, rot or 64, interleaved, scaling))
    oc = dict(hidden=256, heads=4, groups=groups, head_dim=64, ffn=192, seq=64, batch=2, tp=1, tp_rank=0, eps=cfg.layernorm_epsilon,
              theta=cfg.rope_theta, cp=cp, cp_rank=cp - 1)
    total = None
    for i in range(strands):
        out, g = OL.layer_fwd_bwd(oc, w_cpu, mb_cpu[i])
        assert_close(outs[i], out, torch.float32, "out")
        assert_close(dxs[i], g["x"], torch.float32, "dx")
        total = g if total is None else {k: total[k] + g[k] for k in g}
    for k in w_cpu:
        assert_close(w[k].main_grad, total[k], torch.float32, k)


def test_default_rotary_positions_are_what_they_were():
    """A configuration that names whole halves runs the operator of whole halves."""
    from dhellam_amd.core.dstb import LayerConfig
    base = dict(hidden_size=256, num_attention_heads=4, num_query_groups=4, ffn_hidden_size=192, seq_length=64)
    assert not LayerConfig(**base).general_rotary and not LayerConfig(**base, rotary_dim=64).general_rotary
    assert not LayerConfig(**base, rope_theta=None, rotary_interleaved=True).general_rotary


def plain_distill(x, ids, t, lse, target, tau, alpha):
    there = ids >= 0
    logp = t / tau - (lse[..., None] if lse is not None else torch.logsumexp((t / tau).masked_fill(~there, -math.inf), -1, keepdim=True))
    logp = logp.masked_fill(~there, 0.0)
    p = torch.exp(logp).masked_fill(~there, 0.0)
    loss = alpha * tau ** 2 * (p * (logp - torch.log_softmax(x / tau, -1).gather(-1, ids.clamp(min=0)))).sum(-1)
    return loss - (1 - alpha) * torch.log_softmax(x, -1).gather(-1, target[..., None])[..., 0]


@pytest.mark.parametrize("batch_first", [False, True])
@pytest.mark.parametrize("tau,alpha,whole", [(1.0, 1.0, False), (2.0, 0.3, True)])
def test_head_block_with_a_teacher(batch_first, tau, alpha, whole):
    from dhellam_amd.core import dshb
    b, s, h, v, k = 2, 33, 64, 500, 7
    g = torch.Generator(device="cuda").manual_seed(0)
    rand = lambda *n: torch.randn(*n, generator=g, device="cuda")
    hidden, table, ln = rand(b, s, h), rand(v, h) * 0.2, 1 + 0.1 * rand(h)
    labels, mask = torch.randint(0, v, (b, s), generator=g, device="cuda"), (torch.rand(b, s, generator=g, device="cuda") < 0.8).float()
    ids = torch.rand(b, s, v, generator=g, device="cuda").argsort(-1)[..., :k]
    ids[0, 3, 4:] = -1
    t = rand(b, s, k)
    teacher = {"ids": ids, "logits": t, "temperature": tau, "alpha": alpha}
    if whole:
        teacher["lse"] = torch.logsumexp(t / tau, -1) + 0.3
    leaves = [x.double().requires_grad_(True) for x in (hidden, table, ln)]
    hd, td, ld = leaves
    logits = hd * torch.rsqrt((hd * hd).mean(-1, keepdim=True) + 1e-5) * ld @ td.T
    loss = (plain_distill(logits, ids, t.double(), teacher["lse"].double() if whole else None, labels, tau, alpha) * mask).sum() / mask.sum()
    want = torch.autograd.grad(loss, leaves)
    for w in (table, ln):
        w.main_grad = torch.zeros_like(w)
    x = hidden if batch_first else hidden.transpose(0, 1).contiguous()
    got, ctx = dshb.post_process(x, ln, None, labels, mask, table, 1, batch_first=batch_first, teacher=teacher)
    d = dshb.post_process_bwd(ctx)
    assert abs(got.item() - loss.item()) <= 1e-5 * abs(loss.item())
    assert_close(d if batch_first else d.transpose(0, 1), want[0], torch.float32, "d hidden")
    assert_close(table.main_grad, want[1], torch.float32, "d table")
    assert_close(ln.main_grad, want[2], torch.float32, "d norm")
    with pytest.raises(ValueError):
        dshb.post_process(x, ln, None, labels, mask, table, 1, label_smoothing=0.1, batch_first=batch_first, teacher=teacher)


def test_a_step_of_a_mixture_model():
    """Rotary attention, router, experts and a taught head, forward and backward by operators, in bf16, against 64-bit autograd with the same
    choices of experts.  Bound: 16 tensors are stored in 16 bits on the way there and back, each off by 2^-9 of itself (root mean square
    half of that); in quadrature below 2^-9 4, taken twice."""
    from dhellam_amd.core import dshb
    from dhellam_amd._Clib import pymha_varlen_bwd, pymha_varlen_fwd
    from dhellam_amd.operators import moe
    from dhellam_amd.operators.layernorm_column import dgrad_bwd, gemm_fwd, wgrad_bwd
    from dhellam_amd.operators.rope import rotary_bwd, rotary_fwd, rotary_table
    T, H, hq, hk, d, F, E, K, V, KT = 192, 256, 4, 1, 64, 128, 8, 2, 1000, 16
    theta, rot, tau, alpha, ca, cz = 10000.0, 32, 2.0, 0.5, 0.02, 0.002
    g = torch.Generator(device="cuda").manual_seed(0)
    bf = torch.bfloat16
    rand = lambda *n, std=1.0: (torch.randn(*n, generator=g, device="cuda") * std).to(bf)
    x, wqkv, wo = rand(T, H), rand((hq + 2 * hk) * d, H, std=H ** -0.5), rand(H, hq * d, std=(hq * d) ** -0.5)
    wr = torch.randn(E, H, generator=g, device="cuda") * H ** -0.5
    w1, w2, table = rand(E, 2 * F, H, std=H ** -0.5), rand(E, H, F, std=F ** -0.5), rand(V, H, std=H ** -0.5)
    ln = (1 + 0.1 * torch.randn(H, generator=g, device="cuda")).to(bf)
    at = torch.cat((torch.arange(128), torch.arange(64))).cuda()
    cu = torch.tensor([0, 128, T], dtype=torch.int32, device="cuda")
    labels = torch.randint(0, V, (1, T), generator=g, device="cuda")
    mask = torch.rand(1, T, generator=g, device="cuda") < 0.9
    ids = torch.rand(1, T, V, generator=g, device="cuda").argsort(-1)[..., :KT]
    teacher = {"ids": ids, "logits": torch.randn(1, T, KT, generator=g, device="cuda"), "temperature": tau, "alpha": alpha}
    for w in (wqkv, wo, table, ln):
        w.main_grad = torch.zeros_like(w)
    # ---- forward
    tab = rotary_table(theta, rot, "cuda", True, PARTS)
    qkv, _ = gemm_fwd(None, x, wqkv, None, "TN", False, 0, True, None)
    split = lambda p: (p[:, :hq * d].view(T, hq, d), p[:, hq * d:(hq + 1) * d].view(T, 1, d), p[:, (hq + 1) * d:].view(T, 1, d))
    q, k, v = split(qkv)
    rotary_fwd(q, k, tab, at, inplace=True)
    scale = d ** -0.5
    o, _, _, _, _, lse, _, rng = pymha_varlen_fwd(q, k, v, cu, cu, 128, 128, 0.0, scale, True, False, 0, False)
    a, _ = gemm_fwd(None, o.view(T, -1), wo, None, "TN", False, 0, True, None)
    x2 = x + a
    logits = x2.float() @ wr.T
    idx, gates, _ = moe.route_topk(logits, K)
    losses, balance, _ = moe.balance_loss_fwd(logits, idx, mask[0], ca, cz)
    plan, _ = moe.sort_assignments(idx, E)
    xp, _ = moe.permute_fwd(x2, plan, 0, E, T * K)
    y, saved, _ = moe.expert_ffn_fwd(xp, w1, w2, plan.expert_offsets)
    m, _ = moe.unpermute_fwd(y, plan, gates, 0, E)
    x3 = (x2 + m).view(1, T, H)
    loss, ctx = dshb.post_process(x3, ln, None, labels, mask, table, 1, batch_first=True, teacher=teacher)
    # ---- backward
    dx3 = dshb.post_process_bwd(ctx).view(T, H)
    dy, dgates, _ = moe.unpermute_bwd(dx3, y, plan, gates, 0, E, T * K)
    dxp, dw1, dw2, _ = moe.expert_ffn_bwd(dy, xp, w1, w2, plan.expert_offsets, saved)
    dx2, _ = moe.permute_bwd(dxp, plan, 0, E)
    dlogits, _ = moe.route_bwd(logits, idx, gates, dgates, balance)
    dx2 = (dx3.float() + dx2.float() + dlogits @ wr).to(bf)
    dwr = dlogits.T @ x2.float()
    da, _ = dgrad_bwd(None, dx2, wo, None, "NN", False, 0, True, None)
    wgrad_bwd(None, dx2, o.view(T, -1), wo.main_grad, True, "NT", False, 0, True, None)
    dq, dk, dv, _ = pymha_varlen_bwd(da.view(T, hq, d), q, k, v, o, lse, cu, cu, 128, 128, 0.0, scale, True, rng, True, 0, False,
                                     torch.cuda.current_stream().cuda_stream)
    dq, dk, _ = rotary_bwd(dq, dk, tab, at)
    dqkv = torch.cat((dq.view(T, -1), dk.view(T, -1), dv.view(T, -1)), 1)
    dx, _ = dgrad_bwd(None, dqkv, wqkv, None, "NN", False, 0, True, None)
    wgrad_bwd(None, dqkv, x, wqkv.main_grad, True, "NT", False, 0, True, None)
    dx = dx.float() + dx2.float()
    # ---- 64 bits
    leaf = {n: t.double().requires_grad_(True) for n, t in dict(x=x, wqkv=wqkv, wo=wo, wr=wr, w1=w1, w2=w2, table=table, ln=ln).items()}
    q, k, v = split(leaf["x"] @ leaf["wqkv"].T)
    q, k = turn(q, at, theta, rot, True, PARTS), turn(k, at, theta, rot, True, PARTS)
    outs = []
    for lo, hi in ((0, 128), (128, T)):
        sc = torch.einsum("qhd,kd->hqk", q[lo:hi], k[lo:hi, 0]) * scale
        sc = sc.masked_fill(torch.triu(torch.ones(hi - lo, hi - lo, dtype=torch.bool, device="cuda"), 1), -math.inf)
        outs.append(torch.einsum("hqk,kd->qhd", torch.softmax(sc, -1), v[lo:hi, 0]))
    x2 = leaf["x"] + torch.cat(outs).reshape(T, -1) @ leaf["wo"].T
    lg = x2 @ leaf["wr"].T
    gate = torch.softmax(lg.gather(1, idx.long()), 1)
    mm = torch.zeros_like(x2)
    for e in range(E):
        h1 = x2 @ leaf["w1"][e].T
        ye = torch.nn.functional.silu(h1[:, :F]) * h1[:, F:] @ leaf["w2"][e].T
        mm = mm + ye * (gate * (idx == e)).sum(1, keepdim=True)
    x3 = x2 + mm
    keep = mask[0]
    n = keep.sum()
    counts = torch.stack([((idx == e) & keep[:, None]).sum() for e in range(E)]).double()
    aux = ca * E / (K * n * n) * (counts * (torch.softmax(lg, 1) * keep[:, None]).sum(0)).sum()
    zl = cz / n * (torch.logsumexp(lg, 1) ** 2 * keep).sum()
    hd = x3 * torch.rsqrt((x3 * x3).mean(-1, keepdim=True) + 1e-5) * leaf["ln"] @ leaf["table"].T
    main = (plain_distill(hd, ids[0], teacher["logits"][0].double(), None, labels[0], tau, alpha) * keep).sum() / n
    (main + aux + zl).backward()
    assert torch.equal(balance.counts.double(), counts)
    # (each value is a mean over the tokens: what the roundings do to it is below what they do to the gradients)
    assert abs(loss.item() - main.item()) <= 2e-2 * main.item()
    assert abs(losses[0].item() - aux.item()) <= 2e-2 * aux.item() and abs(losses[1].item() - zl.item()) <= 2e-2 * zl.item()
    got = dict(x=dx, wqkv=wqkv.main_grad, wo=wo.main_grad, wr=dwr, w1=dw1, w2=dw2, table=table.main_grad, ln=ln.main_grad)
    far = {name: rel_err(got[name], leaf[name].grad) for name in got}
    assert max(far.values()) <= 2 * 4 * 2.0 ** -9, far


def test_binding_level_names():
    """They forward to the operators of the same kind."""
    from dhellam_amd import _Clib as C
    from dhellam_amd.operators import loss, moe, rope
    g = torch.Generator(device="cuda").manual_seed(1)
    rand = lambda *n: torch.randn(*n, generator=g, device="cuda")
    t, q, k, at = rope.rotary_table(10000.0, 32, "cuda", True), rand(9, 4, 64), rand(9, 1, 64), torch.arange(9, device="cuda")
    for name, f in (("pyrotary_fwd", rope.rotary_fwd), ("pyrotary_bwd", rope.rotary_bwd)):
        got = getattr(C, name)(q, k, t, at, True)
        assert all(torch.equal(a, b) for a, b in zip(got, f(q, k, t, at)[:2])) and got[2] > 0
    lg = rand(9, 8)
    idx, gates, _ = moe.route_topk(lg, 2)
    losses, bal = C.pymoe_balance_loss(lg, idx, None, 0.1, 0.01)
    assert torch.equal(losses, moe.balance_loss_fwd(lg, idx, None, 0.1, 0.01)[0])
    assert torch.equal(C.pymoe_route_bwd(lg, idx, gates, gates, bal, None)[0], moe.route_bwd(lg, idx, gates, gates, bal)[0])
    x, ids, tl, target = rand(9, 50), torch.randint(0, 50, (9, 3), generator=g, device="cuda"), rand(9, 3), torch.arange(9, device="cuda")
    inputs = {"vocab_parallel_logits": x, "teacher_ids": ids, "teacher_logits": tl, "target": target}
    out, want = C.pydistill_fwd(x, ids, tl, None, target, 2.0, 0.5), loss.distill_fwd(inputs, 2.0, 0.5)
    assert torch.equal(out["loss"], want["loss"])
    assert torch.equal(C.pydistill_bwd(x, ids, tl, target, out, losses.new_ones(9)), loss.distill_bwd([inputs, want], losses.new_ones(9)))


def test_sizes_past_an_int_are_refused():
    """Of tensors without an element, so that nothing that large is held: a size of 2^32 + n is not taken for n."""
    from dhellam_amd.operators.loss import distill_bwd, distill_fwd
    from dhellam_amd.operators.moe import balance_loss_fwd, route_bwd
    from dhellam_amd.operators.rope import rotary_fwd, rotary_table
    big = 1 << 32
    empty = lambda *n, dtype=torch.float32: torch.empty(*n, device="cuda", dtype=dtype)
    t = rotary_table(10000.0, 32, "cuda")
    idx = empty(0, big + 2, dtype=torch.int32)
    inputs = {"vocab_parallel_logits": empty(0, 50), "teacher_ids": empty(0, big + 3, dtype=torch.int64), "teacher_logits": empty(0, big + 3)}
    out = distill_fwd(dict(inputs, teacher_ids=inputs["teacher_ids"][:, :3], teacher_logits=inputs["teacher_logits"][:, :3]))
    for bad in [lambda: rotary_fwd(empty(0, big + 1, 64), None, t), lambda: rotary_fwd(empty(0, 1, 64), empty(0, big + 1, 64), t),
                lambda: rotary_fwd(empty(0, 1, big + 64), None, t), lambda: balance_loss_fwd(empty(0, 8), idx),
                lambda: route_bwd(empty(0, 8), idx, empty(0, big + 2), empty(0, big + 2)), lambda: distill_fwd(inputs),
                lambda: distill_bwd([inputs, out], empty(0))]:
        with pytest.raises(RuntimeError):
            bad()
