"""The router's losses, counts and gradients against 64-bit autograd and against differences."""
import pytest
import torch

from dhellam_amd.operators.moe import BalanceLoss, balance_loss_fwd, route_bwd, route_topk

pytestmark = pytest.mark.gpu

A, B = 0.01, 0.001


def router(t, e, k, seed=0, masked=False):
    g = torch.Generator(device="cuda").manual_seed(seed)
    logits = torch.randn(t, e, generator=g, device="cuda") * 2 + torch.randn(e, generator=g, device="cuda")
    idx, gates, _ = route_topk(logits, k)
    dgates = torch.randn(t, k, generator=g, device="cuda")
    mask = torch.rand(t, generator=g, device="cuda") < 0.7 if masked else None
    return logits, idx, gates, dgates, mask


def plain(logits, idx, gates, dgates, mask, w=(1.0, 1.0), a=A, b=B):
    """losses, counts, prob_sum, dlogits in 64 bits, and the size of the terms that the gradient is a sum of."""
    t, e = logits.shape
    k = idx.shape[1]
    m = mask if mask is not None else torch.ones(t, dtype=torch.bool, device=logits.device)
    x = torch.where(m[:, None], logits.double(), 0.0).requires_grad_(True)
    n = max(int(m.sum()), 1)
    counts = torch.stack([((idx == i) & m[:, None]).sum() for i in range(e)])
    lse, p = torch.logsumexp(x, 1), torch.softmax(x, 1)
    probs = (p * m[:, None]).sum(0)
    losses = torch.stack((a * e / (k * n * n) * (counts * probs).sum(), b / n * (lse ** 2 * m).sum()))
    (d,) = torch.autograd.grad((losses * torch.tensor(w, dtype=torch.float64, device=x.device)).sum(), x)
    p, lse = p.detach() * m[:, None], lse.detach() * m
    size = abs(w[0]) * a * e / (k * n * n) * p * (counts + (counts * p).sum(1, keepdim=True)) + abs(w[1]) * 2 * b / n * lse.abs()[:, None] * p
    if dgates is not None:
        g, dg = gates.double(), dgates.double()
        d = d.scatter_add(1, idx.long(), g * (dg - (g * dg).sum(1, keepdim=True)))
        size = size.scatter_add(1, idx.long(), g * (dg.abs() + (g * dg.abs()).sum(1, keepdim=True)))
    return losses.detach(), counts, probs.detach(), d, size


def close(got, want, size, tol=1e-5):
    """An exponential's relative error is (|x - max| + 3) 2^-24, at most 20 2^-24 here; sums are of at most 100 terms one behind the other
    (16 of a lane, 6 exchanges, 4 and 32 and 16 partial sums): 120 2^-24 = 7e-6 of the terms' size."""
    assert ((got.double() - want).abs() <= tol * size + 1e-30).all(), ((got.double() - want).abs() / (size + 1e-30)).max()


SIZES = [(1, 1, 1), (1, 8, 2), (3, 2, 1), (64, 5, 3), (63, 64, 8), (1000, 8, 2), (257, 24, 2), (4096, 16, 4), (5000, 60, 6), (2049, 7, 7), (20011, 64, 8),
         (70001, 8, 2), (131072, 33, 5)]


@pytest.mark.parametrize("t,e,k", SIZES)
@pytest.mark.parametrize("masked", [False, True])
def test_losses_counts_and_gradients(t, e, k, masked):
    logits, idx, gates, dgates, mask = router(t, e, k, seed=t, masked=masked)
    losses, bal, ms = balance_loss_fwd(logits, idx, mask, A, B)
    want = plain(logits, idx, gates, dgates, mask)
    assert ms == 0 and bal.counts.dtype == torch.int32 and torch.equal(bal.counts.long(), want[1])
    assert bal.tokens.item() == (t if mask is None else int(mask.sum()))
    close(losses, want[0], want[0].abs())
    close(bal.prob_sum, want[2], want[2])
    d, _ = route_bwd(logits, idx, gates, dgates, bal)
    close(d, want[3], want[4])
    # each part alone, and the losses' gradients scaled
    none = plain(logits, idx, gates, None, mask, (0.5, -3.0))
    close(route_bwd(logits, idx, gates, None, bal, torch.tensor([0.5, -3.0], device="cuda"))[0], none[3], none[4])
    alone = plain(logits, idx, gates, dgates, mask, (0.0, 0.0))
    close(route_bwd(logits, idx, gates, dgates)[0], alone[3], alone[4])


def test_gradient_against_differences():
    """The losses as a function of the logits with the choices held fixed; a step of h errs by its third derivative, below h^2."""
    logits, idx, gates, dgates, _ = router(6, 8, 2)
    _, bal, _ = balance_loss_fwd(logits, idx, None, 1.0, 0.1)
    d = route_bwd(logits, idx, gates, None, bal)[0]
    f = lambda x: plain(x, idx, gates, None, None, a=1.0, b=0.1)[0].sum().item()
    h = 1e-4
    for t in range(6):
        for e in range(8):
            up, down = logits.double().clone(), logits.double().clone()
            up[t, e] += h
            down[t, e] -= h
            assert abs((f(up) - f(down)) / (2 * h) - d[t, e].item()) <= 1e-6


def test_an_even_router_has_the_coefficient_as_its_loss():
    logits = torch.zeros(64, 8, device="cuda")
    idx = (torch.arange(64, device="cuda", dtype=torch.int32)[:, None] * 2 + torch.arange(2, device="cuda", dtype=torch.int32)) % 8
    losses, bal, _ = balance_loss_fwd(logits, idx, None, 0.5, 1.0)
    torch.testing.assert_close(losses, torch.tensor([0.5, torch.tensor(8.0).log() ** 2], device="cuda"), rtol=1e-6, atol=0)
    assert (bal.counts == 16).all()
    assert route_bwd(logits, idx, balance=BalanceLoss(bal.counts, bal.prob_sum, bal.tokens, bal.lse, None, 0.5, 0.0))[0].abs().max() <= 1e-8


@pytest.mark.parametrize("t,e,k", [(40, 8, 2), (9000, 64, 4), (5, 5, 2)])
def test_masked_tokens_may_hold_anything(t, e, k):
    logits, idx, gates, dgates, mask = router(t, e, k, masked=True)
    mask[0], mask[-1] = False, True
    want = balance_loss_fwd(logits, idx, mask, A, B)
    dwant = route_bwd(logits, idx, gates, None, want[1])[0]
    bad = logits.clone()
    bad[~mask] = torch.tensor([torch.nan, torch.inf, -torch.inf, torch.finfo(torch.float32).min], device="cuda").repeat(t)[:e * t].view(-1)[:e]
    worse = idx.clone()
    worse[~mask] = -7
    got = balance_loss_fwd(bad, worse, mask, A, B)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1].counts, want[1].counts) and torch.equal(got[1].prob_sum, want[1].prob_sum)
    d = route_bwd(bad, worse, gates, None, got[1])[0]
    assert torch.equal(d, dwant) and (d[~mask] == 0).all()


@pytest.mark.parametrize("t", [30, 5000])
def test_logits_that_do_not_start_a_vector(t):
    """Contiguous logits four bytes off the 16-byte grid: the same results."""
    logits, idx, gates, dgates, mask = router(t, 8, 2, masked=True)
    room = torch.zeros(8 * t + 1, device="cuda")
    off = room[1:].view(t, 8).copy_(logits)
    want, got = balance_loss_fwd(logits, idx, mask, A, B), balance_loss_fwd(off, idx, mask, A, B)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1].prob_sum, want[1].prob_sum)
    assert torch.equal(route_bwd(off, idx, gates, dgates, got[1])[0], route_bwd(logits, idx, gates, dgates, want[1])[0])


def test_nothing_counts():
    logits, idx, gates, dgates, _ = router(100, 8, 2)
    off = torch.zeros(100, dtype=torch.bool, device="cuda")
    losses, bal, _ = balance_loss_fwd(logits * torch.nan, idx, off, A, B)
    assert (losses == 0).all() and (bal.counts == 0).all() and (bal.prob_sum == 0).all() and bal.tokens.item() == 0
    assert (route_bwd(logits, idx, gates, None, bal)[0] == 0).all()
    losses, bal, _ = balance_loss_fwd(logits[:0], idx[:0], None, A, B)
    assert (losses == 0).all() and (bal.counts == 0).all() and bal.tokens.item() == 0
    assert route_bwd(logits[:0], idx[:0], gates[:0], dgates[:0], bal)[0].shape == (0, 8)


def test_experts_that_are_switched_off():
    """Logits of -inf, and of the type's lowest value, are probabilities of zero; choices outside [0, E) are not counted."""
    logits, idx, gates, dgates, _ = router(500, 8, 2)
    for low in (-torch.inf, torch.finfo(torch.float32).min):
        x = logits.clone()
        x[:, 5] = low
        i, g, _ = route_topk(x, 2)
        losses, bal, _ = balance_loss_fwd(x, i, None, A, B)
        assert bal.counts[5] == 0 and bal.prob_sum[5] == 0 and torch.isfinite(losses).all()
        d = route_bwd(x, i, g, dgates, bal)[0]
        assert (d[:, 5] == 0).all()
        keep = [0, 1, 2, 3, 4, 6, 7]
        small = i - (i > 5).int()
        want = plain(x[:, keep], small, g, dgates, None, a=A * 8 / 7)
        close(d[:, keep], want[3], want[4])
    out = idx.clone()
    out[::2, 0], out[1::2, 1] = -1, 8
    _, bal, _ = balance_loss_fwd(logits, out, None, A, B)
    assert bal.counts.sum() == 500


@pytest.mark.parametrize("e,k", [(8, 2), (24, 2), (32, 5), (64, 8)])
def test_an_expert_chosen_twice_counts_twice(e, k):
    """In some tokens, beside others that choose each expert once; once three times."""
    logits, idx, gates, dgates, _ = router(150, e, k)
    idx[::3, 1] = idx[::3, 0]
    idx[5, :3] = idx[5, 0].clone()
    losses, bal, _ = balance_loss_fwd(logits, idx, None, A, B)
    assert torch.equal(bal.counts.long(), torch.bincount(idx.flatten().long(), minlength=e))
    d = route_bwd(logits, idx, gates, dgates)[0]
    g, dg = gates.double(), dgates.double()
    ref = torch.zeros(150, e, dtype=torch.float64, device="cuda").scatter_add(1, idx.long(), g * (dg - (g * dg).sum(1, keepdim=True)))
    close(d, ref, torch.zeros_like(ref).scatter_add(1, idx.long(), g * (dg.abs() + (g * dg.abs()).sum(1, keepdim=True))))
    out = idx.clone()
    out[1::4, 0] = -1
    out[2::4, 1] = e
    d = route_bwd(logits, out, gates, dgates)[0]                          # a choice that is none has no logit
    at = out.long().clamp(0, e - 1)
    val = (g * (dg - (g * dg).sum(1, keepdim=True))) * ((out >= 0) & (out < e))
    close(d, torch.zeros_like(ref).scatter_add(1, at, val), torch.zeros_like(ref).scatter_add(1, at, g * (dg.abs() + (g * dg.abs()).sum(1, keepdim=True))))


def test_ranks_join_their_counts():
    logits, idx, gates, dgates, mask = router(4000, 16, 2, masked=True)
    whole = balance_loss_fwd(logits, idx, mask, A, B)
    parts = [balance_loss_fwd(logits[s].contiguous(), idx[s].contiguous(), mask[s].contiguous(), A, B) for s in (slice(0, 1500), slice(1500, 4000))]
    counts, tokens = sum(p[1].counts for p in parts), sum(p[1].tokens for p in parts)
    assert torch.equal(counts, whole[1].counts) and torch.equal(tokens, whole[1].tokens)
    probs = sum(p[1].prob_sum for p in parts)
    n = tokens.double()
    torch.testing.assert_close((A * 16 / (2 * n * n) * (counts.double() * probs.double()).sum()).float()[0], whole[0][0], rtol=1e-5, atol=0)
    want = route_bwd(logits, idx, None, None, whole[1])[0]
    for p, s in zip(parts, (slice(0, 1500), slice(1500, 4000))):
        bal = BalanceLoss(counts, probs, tokens, p[1].lse, p[1].mask, A, B)
        assert torch.equal(route_bwd(logits[s].contiguous(), idx[s].contiguous(), None, None, bal)[0], want[s])


def test_tokens_past_32_bits_of_offset():
    """40 million tokens of 64 experts (10 GB): 5000 tokens over and over.  A lane adds 2500 terms one behind the other, half a step each
    at most: 2^-24 2500 = 1.5e-4 of a sum beside what ``close`` allows."""
    logits, idx, gates, dgates, mask = router(5000, 64, 8, masked=True)
    n = 8000
    many = lambda t: t.repeat(n, *[1] * (t.dim() - 1))
    x, i = many(logits), many(idx)
    losses, bal, _ = balance_loss_fwd(x, i, many(mask), A, B)
    want = plain(logits, idx, None, None, mask)
    assert torch.equal(bal.counts.long(), n * want[1]) and bal.tokens.item() == n * int(mask.sum())
    close(losses, want[0], want[0].abs(), 1.6e-4)
    close(bal.prob_sum, n * want[2], n * want[2], 1.6e-4)
    d = route_bwd(x, i, many(gates), many(dgates), bal)[0]
    ref = plain(logits, idx, gates, dgates, mask)
    losses_only, with_gates = plain(logits, idx, None, None, mask), ref[3] - want[3]
    for at in (slice(0, 5000), slice(-5000, None)):                       # (a mean over n times as many: the losses' share is n times smaller)
        close(d[at], losses_only[3] / n + with_gates, ref[4])


def test_the_same_every_time_on_streams_and_in_graphs():
    """Two graphs captured on one stream, replayed at the same time on two: neither shares scratch with the other."""
    data = [router(60000 + i, 64, 8, seed=i) for i in range(2)]
    want = []
    for logits, idx, gates, dgates, mask in data:
        losses, bal, _ = balance_loss_fwd(logits, idx, mask, A, B)
        want.append((losses, bal.counts, bal.prob_sum, route_bwd(logits, idx, gates, dgates, bal)[0]))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    logits, idx, gates, dgates, mask = data[0]
    losses, bal, ms = balance_loss_fwd(logits, idx, mask, A, B, stream=side, profiling=True)
    d, _ = route_bwd(logits, idx, gates, dgates, bal, stream=side)
    torch.cuda.synchronize()
    assert ms > 0 and torch.equal(losses, want[0][0]) and torch.equal(d, want[0][3])
    graphs, outs = [], []
    for logits, idx, gates, dgates, mask in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            losses, bal, _ = balance_loss_fwd(logits, idx, mask, A, B)
            outs.append((losses, bal.counts, bal.prob_sum, route_bwd(logits, idx, gates, dgates, bal)[0]))
        graphs.append(g)
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    for _ in range(3):
        for o in outs:
            for x in o:
                x.zero_()
        torch.cuda.synchronize()
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
        torch.cuda.synchronize()
        for got, ref in zip(outs, want):
            assert all(torch.equal(x, y) for x, y in zip(got, ref))


def test_refusals():
    logits, idx, gates, dgates, _ = router(10, 8, 2)
    _, bal, _ = balance_loss_fwd(logits, idx)
    ok = torch.ones(10, dtype=torch.bool, device="cuda")
    for bad in [lambda: balance_loss_fwd(logits.half(), idx), lambda: balance_loss_fwd(logits[:, :4], idx), lambda: balance_loss_fwd(logits, idx.long()),
                lambda: balance_loss_fwd(logits, idx[:9]), lambda: balance_loss_fwd(logits, idx, ok.float()), lambda: balance_loss_fwd(logits, idx, ok[:9]),
                lambda: route_bwd(logits, idx), lambda: route_bwd(logits, idx, None, dgates), lambda: route_bwd(logits, idx, gates.half(), dgates),
                lambda: route_bwd(logits, idx, gates[:9], dgates), lambda: route_bwd(logits[:9], idx[:9], None, None, bal),
                lambda: route_bwd(logits, idx, None, None, bal, torch.ones(3, device="cuda"))]:
        with pytest.raises(AssertionError):
            bad()
    for bad in [lambda: balance_loss_fwd(logits, idx.cpu()), lambda: balance_loss_fwd(torch.zeros(4, 65, device="cuda"), idx[:4]),
                lambda: balance_loss_fwd(logits, torch.zeros(10, 9, dtype=torch.int32, device="cuda")),
                lambda: route_bwd(logits, idx, gates, dgates.cpu()), lambda: balance_loss_fwd(logits, idx, stream=3)]:
        with pytest.raises(RuntimeError):
            bad()


@pytest.mark.parametrize("t,e,k", [(64, 3, 2), (500, 8, 2), (300, 16, 4), (5000, 24, 2), (9000, 60, 6)])
@pytest.mark.parametrize("offset", [20.0, -100.0, 1000.0, 30000.0])
def test_the_size_of_the_logits_costs_no_digits(t, e, k, offset):
    """A softmax does not depend on what all logits of a row have in common.  Probabilities: the argument's difference, product and constant
    are 2.5 half steps of up to 20, the exponential 2, the sum over 64 and its reciprocal 10, and they come twice (alone and in the
    mean): 2 (50 + 12) 2^-24 = 7.4e-6 of the terms, below what ``close`` allows."""
    logits, idx, gates, dgates, mask = router(t, e, k, seed=t, masked=True)
    logits += offset * torch.linspace(0.5, 1.0, t, device="cuda")[:, None]
    losses, bal, _ = balance_loss_fwd(logits, idx, mask, A, B)
    for w in ((1.0, 1.0), (1.0, 0.0), (0.0, 1.0)):
        want = plain(logits, idx, gates, None, mask, w)
        close(route_bwd(logits, idx, None, None, bal, torch.tensor(w, device="cuda"))[0], want[3], want[4])
    close(losses, want[0], want[0].abs())
    close(bal.prob_sum, want[2], want[2])


@pytest.mark.parametrize("e", [41, 63])
def test_equal_terms_of_many_tokens(e):
    """2^27 + 5 tokens that all say the same: 8192 terms a lane, whose roundings all go one way.  64 terms behind one another, then 128 sums of
    them, 2 exchanges, and 16, 16 and 16 partial sums: a half step of the running sum each, which is half the final one on average, 121 2^-24 =
    7.2e-6, and 2^-23 of a term."""
    t = (1 << 27) + 5
    idx = (torch.arange(t, device="cuda") % e).int()[:, None]
    losses, bal, _ = balance_loss_fwd(torch.zeros(t, e, device="cuda"), idx, None, A, B)
    assert torch.equal(bal.counts, torch.bincount(idx[:, 0], minlength=e).int()) and bal.tokens.item() == t
    want = torch.tensor([A, B * torch.log(torch.tensor(float(e), dtype=torch.float64)).item() ** 2], dtype=torch.float64, device="cuda")
    close(losses, want, want)
    close(bal.prob_sum, torch.full((e,), t / e, dtype=torch.float64, device="cuda"), t / e)


@pytest.mark.parametrize("t,e,k", [(4097, 1, 1), (5001, 2, 2), (9999, 3, 1), (70003, 4, 4), (2049, 8, 8), (1025, 9, 3), (513, 17, 5), (20001, 24, 2), (3001, 32, 8),
                                   (257, 33, 8), (30011, 63, 8)])
@pytest.mark.parametrize("masked", [False, True])
def test_every_number_of_lanes_in_two_launches(t, e, k, masked):
    test_losses_counts_and_gradients(t, e, k, masked)
