"""The distillation loss against 64-bit log-softmax and autograd, and against differences."""
import pytest
import torch

from dhellam_amd.common import parallel_state
from dhellam_amd.operators.loss import cross_entropy_bwd, cross_entropy_fwd, distill_bwd, distill_fwd, distill_statistics

pytestmark = pytest.mark.gpu

LOW = torch.finfo(torch.float32).min


def case(rows, cols, k, dtype, alpha=1.0, whole=False, padded=False, twice=False, tau=1.0, seed=0, ids=torch.int64, teacher=torch.float32):
    g = torch.Generator(device="cuda").manual_seed(seed)
    x = (torch.randn(rows, cols, generator=g, device="cuda") * 2).to(dtype)
    i = torch.rand(rows, cols, generator=g, device="cuda").argsort(1)[:, :k].contiguous() if rows * cols < 1 << 24 else (
        torch.randint(0, cols, (rows, 1), generator=g, device="cuda") + torch.arange(k, device="cuda") * (cols // k)) % cols
    if twice and k > 1:
        i[:, 1::2] = i[:, 0::2][:, :i[:, 1::2].shape[1]]
    t = (torch.randn(rows, k, generator=g, device="cuda") * 2 + 3).sort(1, descending=True).values.to(teacher)
    lse = torch.logsumexp(t.float() / tau, 1) + 0.2 if whole else None
    if padded:
        n = torch.randint(0, k + 1, (rows, 1), generator=g, device="cuda")
        n[0] = 0
        i = i.masked_fill(torch.arange(k, device="cuda") >= n, -1)
    target = torch.randint(0, cols, (rows,), generator=g, device="cuda") if alpha < 1 else None
    if alpha < 1 and rows > 1:
        target[1] = i[1, 0].clamp(min=0)                    # the target among the teacher's entries
    inputs = {"vocab_parallel_logits": x, "teacher_ids": i.to(ids), "teacher_logits": t, "teacher_lse": lse, "target": target}
    return inputs, torch.rand(rows, generator=g, device="cuda")


def plain(inputs, tau, alpha):
    """(loss, d loss / d logits, size of the loss' terms, size of the gradient's), 64 bits, entries one at a time."""
    x = inputs["vocab_parallel_logits"].double().requires_grad_(True)
    cols = x.shape[-1]
    ids, t = inputs["teacher_ids"].long(), inputs["teacher_logits"].double() / tau
    there = (ids >= 0) & (ids < cols)
    t = t.masked_fill(~there, -torch.inf)
    norm = inputs["teacher_lse"].double()[..., None] if inputs["teacher_lse"] is not None else torch.logsumexp(t, -1, keepdim=True)
    logp = (t - norm).masked_fill(~there, 0.0)
    p = torch.exp(logp).masked_fill(~there, 0.0)
    logq = torch.log_softmax(x / tau, -1)
    col = ids.clamp(0, cols - 1)
    at = logq.gather(-1, col)
    some = p > 0
    terms = torch.where(some, p * (torch.where(some, logp, 0.0) - torch.where(some, at, 0.0)), 0.0)
    loss = alpha * tau ** 2 * terms.sum(-1)
    # the parts that logq is the difference of: (x - max) / tau and log sum
    top = x.detach().max(-1, keepdim=True).values
    logs = torch.logsumexp(x.detach() / tau, -1, keepdim=True) - top / tau
    size = alpha * tau ** 2 * (p * (torch.where(some, logp.abs(), 0.0) + ((x.detach().gather(-1, col) - top) / tau).abs().nan_to_num(0, 0, 0) + logs.abs() + 1)).sum(-1)
    q = torch.exp(logq.detach())
    gsize = alpha * tau * p.sum(-1, keepdim=True) * q
    gsize = gsize.scatter_add(-1, col, alpha * tau * p)
    if alpha < 1:
        hard = torch.log_softmax(x, -1)
        pick = hard.gather(-1, inputs["target"][..., None])[..., 0]
        loss = loss - (1 - alpha) * pick
        size = size + (1 - alpha) * (pick.detach().abs() + (torch.logsumexp(x.detach(), -1) - top[..., 0]).abs() + 1)
        gsize = gsize + (1 - alpha) * torch.exp(hard.detach())
        gsize = gsize.scatter_add(-1, inputs["target"][..., None], torch.full_like(top, 1 - alpha))
    (d,) = torch.autograd.grad(loss.sum(), x)
    return loss.detach(), d, size, gsize


def tolerance(cols, tau):
    """Sums of cols / 256 terms one behind the other and 20 joins, an exponential of an argument of up to 40 / tau: half steps of 2^-23."""
    return (cols / 256 + 20 + 2 * 40 / min(tau, 1.0) + 10) * 2.0 ** -24


def compare(out, d, want, dout, dtype, cols, tau):
    tol = tolerance(cols, tau)
    loss, grad, size, gsize = want
    assert out["loss"].dtype == torch.float32 and out["loss"].shape == loss.shape
    assert ((out["loss"].double() - loss).abs() <= tol * size + 1e-30).all(), ((out["loss"].double() - loss).abs() / size).max()
    w = dout.double()[..., None]
    bound = (grad * w).abs() * torch.finfo(dtype).eps / 2 + 1.01 * tol * gsize * w.abs() + torch.finfo(dtype).tiny * torch.finfo(dtype).eps
    err = (d.double() - grad * w).abs()
    assert d.dtype == dtype and (err <= bound).all(), (err / bound).max()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols,k", [(1, 1, 1), (1, 2, 2), (3, 7, 3), (5, 1000, 64), (2, 4097, 1), (33, 4001, 100), (2, 50257, 300), (1, 128256, 1024),
                                         (1030, 1000, 20), (1024, 515, 257), (300, 2048, 256), (70, 2049, 255), (4100, 3000, 5), (101, 65600, 300), (520, 9001, 3)])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 1.0), (1.0, 0.5), (0.7, 0.3), (4.0, 0.0)])
def test_loss_and_gradient(rows, cols, k, tau, alpha, dtype):
    inputs, dout = case(rows, cols, k, dtype, alpha, tau=tau, seed=cols + k)
    out = distill_fwd(inputs, tau, alpha)
    compare(out, distill_bwd([inputs, out], dout), plain(inputs, tau, alpha), dout, dtype, cols, tau)


@pytest.mark.parametrize("padded,twice,whole", [(True, False, False), (False, True, False), (False, False, True), (True, True, True)])
@pytest.mark.parametrize("rows,cols,k", [(40, 1000, 8), (6, 30001, 130), (1100, 777, 33), (2, 9000, 1024)])
@pytest.mark.parametrize("alpha", [1.0, 0.4])
@pytest.mark.parametrize("ids,teacher", [(torch.int64, torch.float32), (torch.int32, torch.bfloat16), (torch.int32, torch.float16)])
def test_padded_repeated_and_unnormalised_lists(rows, cols, k, padded, twice, whole, alpha, ids, teacher):
    inputs, dout = case(rows, cols, k, torch.bfloat16, alpha, whole, padded, twice, 1.5, ids=ids, teacher=teacher)
    out = distill_fwd(inputs, 1.5, alpha)
    d = distill_bwd([inputs, out], dout)
    compare(out, d, plain(inputs, 1.5, alpha), dout, torch.bfloat16, cols, 1.5)
    if padded and alpha == 1.0:
        assert out["loss"][0] == 0 and (d[0] == 0).all()                 # nothing listed: nothing learnt
    if padded:                                                           # what a padded entry holds is not looked at
        other = dict(inputs)
        gone = inputs["teacher_ids"] < 0
        other["teacher_logits"] = inputs["teacher_logits"].masked_fill(gone, torch.nan)
        other["teacher_ids"] = inputs["teacher_ids"].masked_fill(gone, 1 << 30)
        again = distill_fwd(other, 1.5, alpha)
        assert torch.equal(again["loss"], out["loss"]) and torch.equal(distill_bwd([other, again], dout), d)


def test_gradient_against_differences():
    """fp64 differences of the 64-bit loss: h^2 of a third derivative of order one, and the rounding 1e-16 / h."""
    inputs, dout = case(2, 30, 5, torch.float32, 0.4, padded=False, twice=True, tau=1.3)
    out = distill_fwd(inputs, 1.3, 0.4)
    d = distill_bwd([inputs, out], torch.ones(2, device="cuda"))
    h = 1e-4
    for c in range(30):
        f = []
        for s in (h, -h):
            moved = dict(inputs)
            moved["vocab_parallel_logits"] = inputs["vocab_parallel_logits"].double()
            moved["vocab_parallel_logits"][:, c] += s
            f.append(plain(moved, 1.3, 0.4)[0])
        assert ((f[0] - f[1]) / (2 * h) - d[:, c].double()).abs().max() <= 2e-6


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,cols", [(3, 1001), (1025, 130)])
def test_shapes_strides_and_in_place(rows, cols, dtype):
    inputs, dout = case(2 * rows, cols, 9, dtype, 0.5)
    out = distill_fwd(inputs, 2.0, 0.5)
    want = distill_bwd([inputs, out], dout)
    folded = {n: (v.unflatten(0, (2, rows)) if v is not None else None) for n, v in inputs.items()}
    pitched = torch.zeros(2 * rows, cols + 5, device="cuda", dtype=dtype)
    pitched[:, 3:cols + 3] = inputs["vocab_parallel_logits"]
    folded["vocab_parallel_logits"] = pitched[:, 3:cols + 3].unflatten(0, (2, rows))
    folded["teacher_ids"] = folded["teacher_ids"].transpose(-1, -2).contiguous().transpose(-1, -2)
    o2 = distill_fwd(folded, 2.0, 0.5)
    assert o2["loss"].shape == (2, rows) and torch.equal(o2["loss"].flatten(), out["loss"])
    d2 = distill_bwd([folded, o2], dout.view(2, rows))
    assert d2.shape == (2, rows, cols) and torch.equal(d2.flatten(0, 1), want)
    d3 = distill_bwd([folded, o2], dout.view(2, rows), grad_out=folded["vocab_parallel_logits"])
    assert d3.data_ptr() == pitched[:, 3:].data_ptr() and torch.equal(pitched[:, 3:cols + 3], want)
    assert (pitched[:, :3] == 0).all() and (pitched[:, cols + 3:] == 0).all()


def test_it_is_the_cross_entropy_without_a_teacher_and_a_scaled_one_with_a_certain_teacher():
    inputs, dout = case(50, 3001, 4, torch.float32, 0.0)
    out = distill_fwd(inputs, 3.0, 0.0)
    ce_in = {"vocab_parallel_logits": inputs["vocab_parallel_logits"], "target": inputs["target"]}
    ce = cross_entropy_fwd(ce_in, keep_softmax=False)
    torch.testing.assert_close(out["loss"], ce["loss"], rtol=1e-5, atol=1e-6)
    torch.testing.assert_close(distill_bwd([inputs, out], dout), cross_entropy_bwd([ce_in, ce], dout), rtol=1e-4, atol=1e-7)
    sure = dict(inputs, teacher_ids=inputs["target"][:, None], teacher_logits=torch.zeros(50, 1, device="cuda"))
    out = distill_fwd(sure)
    torch.testing.assert_close(out["loss"], ce["loss"], rtol=1e-5, atol=1e-6)


@pytest.mark.parametrize("rows,cols", [(4, 2000), (1100, 2000), (4, 6000), (4, 40000)])
@pytest.mark.parametrize("alpha", [1.0, 0.5])
def test_rows_and_columns_that_are_switched_off(rows, cols, alpha):
    """Student columns of -inf or the lowest value have no probability; teacher entries of -inf neither; a row with dout 0 gets zeros
    whatever it holds; a listed column of -inf is an infinite loss with a finite gradient."""
    inputs, dout = case(rows, cols, 16, torch.float32, alpha)
    x, t = inputs["vocab_parallel_logits"], inputs["teacher_logits"]
    x[:, cols - 10:] = torch.tensor([-torch.inf, LOW], device="cuda").repeat(5)
    keep = (inputs["teacher_ids"] < cols - 10) & (torch.arange(16, device="cuda") % 3 != 2)
    inputs["teacher_logits"] = t.masked_fill(~keep, -torch.inf)
    if alpha < 1:
        inputs["target"].clamp_(max=cols - 11)
    out = distill_fwd(inputs, 1.0, alpha)
    d = distill_bwd([inputs, out], dout)
    compare(out, d, plain(inputs, 1.0, alpha), dout, torch.float32, cols, 1.0)
    assert torch.isfinite(out["loss"]).all() and (d[:, cols - 10:] == 0).all()
    x[2] = torch.tensor([torch.nan, torch.inf], device="cuda").repeat(cols // 2)
    dout[2] = 0
    again = distill_fwd(inputs, 1.0, alpha)
    d2 = distill_bwd([inputs, again], dout)
    assert (d2[2] == 0).all() and torch.equal(d2[3:], d[3:]) and torch.equal(again["loss"][3:], out["loss"][3:])
    inputs["teacher_ids"][0, 0], inputs["teacher_logits"][0, 0] = cols - 10, 5.0
    again = distill_fwd(inputs, 1.0, alpha)
    assert again["loss"][0] == torch.inf and torch.isfinite(distill_bwd([inputs, again], dout)[0]).all()


@pytest.mark.parametrize("low", [-torch.inf, LOW, -1e30])
@pytest.mark.parametrize("rows,cols", [(4, 40000), (3, 3000), (1100, 900)])
def test_a_switched_off_beginning_of_the_vocabulary(rows, cols, low):
    """Whole segments, and whole wavefronts' shares, without a value to compare with."""
    inputs, dout = case(rows, cols, 300 if cols > 3000 else 40, torch.float32, 0.5, tau=0.7)
    part = cols * 3 // 5
    inputs["vocab_parallel_logits"][:, :part] = low
    inputs["teacher_ids"].clamp_(min=part)
    inputs["target"].clamp_(min=part)
    out = distill_fwd(inputs, 0.7, 0.5)
    compare(out, distill_bwd([inputs, out], dout), plain(inputs, 0.7, 0.5), dout, torch.float32, cols, 0.7)


@pytest.mark.parametrize("rows,cols", [(6, 1200), (1200, 1200), (3, 34000)])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 0.4)])
def test_slices_of_the_vocabulary_join(rows, cols, tau, alpha):
    k = 20
    inputs, dout = case(rows, 2 * cols, k, torch.float32, alpha, padded=True, tau=tau)
    whole = distill_fwd(inputs, tau, alpha)
    want = distill_bwd([inputs, whole], dout)
    outs, parts = [], []
    try:
        for rank in range(2):
            parallel_state.set_tensor_model_parallel(rank, 2)
            part = dict(inputs, vocab_parallel_logits=inputs["vocab_parallel_logits"][:, rank * cols:(rank + 1) * cols])
            parts.append(part)
            outs.append(distill_statistics(distill_fwd(part, tau, alpha)))
        m = torch.maximum(outs[0]["row_max"], outs[1]["row_max"])
        s = sum(o["sum_exp_t"] * torch.exp((o["row_max"] - m) / tau) for o in outs)
        dot = sum(o["dot"] + o["mass_local"] * (o["row_max"] - m) / tau for o in outs)
        torch.testing.assert_close(outs[0]["mass"], outs[1]["mass"])
        loss = alpha * tau ** 2 * (outs[0]["entropy"] - dot + outs[0]["mass"] * torch.log(s))
        s1 = s
        if alpha < 1:
            s1 = sum(o["sum_exp"] * torch.exp(o["row_max"] - m) for o in outs)
            mine = [(inputs["target"] >= r * cols) & (inputs["target"] < (r + 1) * cols) for r in range(2)]
            pred = sum(torch.where(i, o["predicted"] + o["row_max"] - m, 0.0) for i, o in zip(mine, outs))
            loss = loss + (1 - alpha) * (torch.log(s1) - pred)
        torch.testing.assert_close(loss, whole["loss"], rtol=2e-5, atol=2e-5)
        for rank in range(2):
            parallel_state.set_tensor_model_parallel(rank, 2)
            o = distill_fwd(parts[rank], tau, alpha)
            for name, joined in (("row_max", m), ("sum_exp_t", s), ("sum_exp", s1)):
                distill_statistics(o)[name].copy_(joined)
            got = distill_bwd([parts[rank], o], dout)
            torch.testing.assert_close(got, want[:, rank * cols:(rank + 1) * cols], rtol=1e-4, atol=1e-7)
    finally:
        parallel_state.set_tensor_model_parallel(0, 1)


def test_logits_past_32_bits_of_offset():
    """20000 rows of 128256 in bf16 (5.1 GB): the last rows are what they are alone, in place too."""
    n, cols = 20000, 128256
    tail, dout = case(5, cols, 20, torch.bfloat16, 0.5, tau=2.0)
    inputs = {name: (v.repeat(n // 5, *[1] * (v.dim() - 1)) if v is not None else None) for name, v in tail.items()}
    out = distill_fwd(inputs, 2.0, 0.5)
    want = plain(tail, 2.0, 0.5)
    d = distill_bwd([inputs, out], dout.repeat(n // 5), grad_out=inputs["vocab_parallel_logits"])
    for at in (slice(0, 5), slice(n - 5, n)):
        compare({"loss": out["loss"][at]}, d[at], want, dout, torch.bfloat16, cols, 2.0)
    assert torch.equal(out["loss"], out["loss"][:5].repeat(n // 5)) and torch.equal(d[-5:], d[:5])


def test_the_same_every_time_in_graphs():
    """Two graphs captured behind one another replay at the same time on two streams; repeated columns are summed in the list's order."""
    data = [case(5 + i, 40000, 300, torch.bfloat16, 0.5, twice=True, seed=i) for i in range(2)]
    run = lambda inputs, dout: (lambda out: (out["loss"], distill_bwd([inputs, out], dout)))(distill_fwd(inputs, 2.0, 0.5))
    want = [run(*d) for d in data]
    graphs, outs = [], []
    for d in data:
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            outs.append(run(*d))
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
        for got, ref, d in zip(outs, want, data):
            assert all(torch.equal(x, y) for x, y in zip(got, ref))
            assert all(torch.equal(x, y) for x, y in zip(run(*d), ref))


def test_refusals():
    inputs, dout = case(4, 100, 3, torch.bfloat16, 0.5)
    out = distill_fwd(inputs, 1.0, 0.5)
    i, t, x = inputs["teacher_ids"], inputs["teacher_logits"], inputs["vocab_parallel_logits"]
    for change in [{"target": None}, {"target": inputs["target"].int()}, {"target": inputs["target"][:3]}, {"teacher_ids": i.float()}, {"teacher_ids": i[:3]},
                   {"teacher_logits": t[:, :2]}, {"teacher_lse": torch.zeros(3, device="cuda")}, {"teacher_lse": torch.zeros(4, device="cuda").half()},
                   {"vocab_parallel_logits": torch.zeros(100, 4, device="cuda").t()}]:
        with pytest.raises(AssertionError):
            distill_fwd(dict(inputs, **change), 1.0, 0.5)
    for change, args in [({"teacher_logits": t.double()}, (1.0, 0.5)), ({"vocab_parallel_logits": x.double()}, (1.0, 0.5)), ({"teacher_ids": i.cpu()}, (1.0, 0.5)),
                         ({}, (0.0, 0.5)), ({}, (1.0, 1.5)), ({}, (float("nan"), 0.5)),
                         ({"teacher_ids": i.repeat(1, 400), "teacher_logits": t.repeat(1, 400)}, (1.0, 0.5)),
                         ({"teacher_ids": i[:, :0], "teacher_logits": t[:, :0]}, (1.0, 0.5))]:
        with pytest.raises(RuntimeError):
            distill_fwd(dict(inputs, **change), *args)
    for bad in [lambda: distill_bwd([inputs, out], dout[:3]), lambda: distill_bwd([inputs, dict(out, stats=out["stats"][:, :3])], dout),
                lambda: distill_bwd([inputs, out], dout, x.float()), lambda: distill_bwd([inputs, out], dout, x[:3])]:
        with pytest.raises(AssertionError):
            bad()
    with pytest.raises(RuntimeError):                                    # a gradient that overlaps the logits in another place
        room = torch.zeros(405, device="cuda", dtype=torch.bfloat16)
        distill_bwd([dict(inputs, vocab_parallel_logits=room[:400].view(4, 100)), out], dout, room[5:].view(4, 100))
    none = {n: (v[:0] if v is not None else None) for n, v in inputs.items()}
    o = distill_fwd(none, 1.0, 0.5)
    assert o["loss"].shape == (0,) and distill_bwd([none, o], dout[:0]).shape == (0, 100)


@pytest.mark.parametrize("low", [-torch.inf, LOW, -1e30])
@pytest.mark.parametrize("rows,cols", [(3, 70000), (3, 30000)])
@pytest.mark.parametrize("tau", [1.0, 0.7])
def test_entries_without_a_weight_on_columns_that_are_switched_off(rows, cols, tau, low):
    """600 entries: the first 300 have no weight (the teacher's -inf) and columns without a probability, or are padding; what a row's
    segments are joined with must not be measured against those."""
    inputs, dout = case(rows, cols, 600, torch.float32, tau=tau)
    x, ids, t = inputs["vocab_parallel_logits"], inputs["teacher_ids"], inputs["teacher_logits"]
    x[:, :cols // 2] = low
    ids[:, :300] = torch.arange(300, device="cuda")
    ids[:, 300:] = cols - 1 - torch.arange(300, device="cuda")
    t[:, :300] = -torch.inf
    ids[1, :290] = -1
    x[2] = torch.where(x[2] == low, low, x[2] + 500.0)                  # a row far from zero
    out = distill_fwd(inputs, tau, 1.0)
    compare(out, distill_bwd([inputs, out], dout), plain(inputs, tau, 1.0), dout, torch.float32, cols, tau)


@pytest.mark.parametrize("rows,cols", [(6, 1200), (1200, 1200), (3, 34000), (2, 70000)])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (0.5, 0.4), (2.0, 0.4)])
@pytest.mark.parametrize("low", [-torch.inf, LOW])
def test_slices_that_are_switched_off_join(rows, cols, tau, alpha, low):
    """One rank's whole slice holds nothing but -inf (or the lowest float): what it leaves adds nothing, by the formula as it is written.  The loss of a
    row that lists a column of -inf there, or has its label there, is infinite.  The joined loss is a sum of the same terms as that of one
    call, each rounded once more: twice the tolerance of ``compare``."""
    inputs, dout = case(rows, 2 * cols, 20, torch.float32, alpha, padded=True, tau=tau)
    inputs["vocab_parallel_logits"][:, :cols] = low
    inputs["teacher_ids"] = torch.where(inputs["teacher_ids"] >= 0, inputs["teacher_ids"].clamp(min=cols), -1)
    inputs["teacher_ids"][0, 0] = cols                                   # (row 0 of a padded case lists nothing)
    if alpha < 1:
        inputs["target"].clamp_(min=cols)
    there = []
    if low == -torch.inf:                                                # the first row lists a column that is switched off, the second has its label there
        inputs["teacher_ids"][0, 0] = 5
        there = [0]
        if alpha < 1:
            inputs["target"][1] = 7
            there = [0, 1]
    want = plain(inputs, tau, alpha)
    slices = [dict(inputs, vocab_parallel_logits=inputs["vocab_parallel_logits"][:, r * cols:(r + 1) * cols]) for r in range(2)]
    try:
        outs = []
        for rank in range(2):
            parallel_state.set_tensor_model_parallel(rank, 2)
            outs.append(distill_fwd(slices[rank], tau, alpha))
        st = [distill_statistics(o) for o in outs]
        m = torch.maximum(st[0]["row_max"], st[1]["row_max"])
        s = sum(o["sum_exp_t"] * torch.exp((o["row_max"] - m) / tau) for o in st)
        d = sum(o["dot"] + o["mass_local"] * (o["row_max"] - m) / tau for o in st)
        loss = alpha * tau ** 2 * (st[0]["entropy"] - d + st[0]["mass"] * torch.log(s))
        s1 = s
        if alpha < 1:
            s1 = sum(o["sum_exp"] * torch.exp(o["row_max"] - m) for o in st)
            mine = [(inputs["target"] >= r * cols) & (inputs["target"] < (r + 1) * cols) for r in range(2)]
            loss = loss + (1 - alpha) * (torch.log(s1) - sum(torch.where(i, o["predicted"] + o["row_max"] - m, 0.0) for i, o in zip(mine, st)))
        fine = [r for r in range(rows) if r not in there]
        assert (loss[there] == torch.inf).all()
        assert ((loss.double() - want[0]).abs() <= 2 * tolerance(2 * cols, tau) * want[2] + 1e-30)[fine].all()
        for rank in range(2):
            parallel_state.set_tensor_model_parallel(rank, 2)
            for name, joined in (("row_max", m), ("sum_exp_t", s), ("sum_exp", s1)):
                st[rank][name].copy_(joined)
            got = distill_bwd([slices[rank], outs[rank]], dout)
            ref = want[1][:, rank * cols:(rank + 1) * cols] * dout[:, None]
            assert ((got - ref).abs() <= 2 * tolerance(2 * cols, tau) * want[3][:, rank * cols:(rank + 1) * cols] * dout[:, None]
                    + ref.abs() * 2.0 ** -24 + 1e-37)[fine].all()
            assert torch.isfinite(got).all()
            if rank == 0:                                                # (listed columns there have what is taken off them)
                got[there] = 0
                assert (got == 0).all()
    finally:
        parallel_state.set_tensor_model_parallel(0, 1)


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("rows,cols,k", [(64, 2000, 256), (300, 4001, 1024), (40, 70001, 1024)])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 0.5)])
def test_dense_lists_in_place(rows, cols, k, tau, alpha, dtype):
    """Every third column or so is listed, by wavefronts other than those that write it: over the logits the same bits as beside them."""
    inputs, dout = case(rows, cols, k, dtype, alpha, tau=tau)
    inputs["teacher_ids"] = (torch.arange(k, device="cuda") * 3 + torch.arange(rows, device="cuda")[:, None]) % cols
    out = distill_fwd(inputs, tau, alpha)
    want = distill_bwd([inputs, out], dout)
    compare(out, want, plain(inputs, tau, alpha), dout, dtype, cols, tau)
    assert torch.equal(distill_bwd([inputs, out], dout, grad_out=inputs["vocab_parallel_logits"]), want)


@pytest.mark.parametrize("rows,cols,k,dtype", [(300, 100003, 300, torch.bfloat16), (1500, 100003, 20, torch.float16), (2800, 50257, 64, torch.bfloat16),
                                               (130, 128256, 1024, torch.float32), (1400, 50257, 8, torch.float32), (7001, 3001, 33, torch.float16)])
@pytest.mark.parametrize("tau,alpha", [(1.0, 1.0), (2.0, 0.5), (4.0, 0.5), (0.7, 0.5)])
def test_logits_that_go_past_the_caches(rows, cols, k, dtype, tau, alpha):
    """More than a part of the last-level cache, with padded lists, repeated columns and the label among them; in place the same bits."""
    inputs, dout = case(rows, cols, k, dtype, alpha, padded=True, twice=True, tau=tau, teacher=torch.bfloat16)
    out = distill_fwd(inputs, tau, alpha)
    d = distill_bwd([inputs, out], dout)
    for at in range(0, rows, 500):
        s = slice(at, at + 500)
        part = {n: (v[s] if v is not None else None) for n, v in inputs.items()}
        compare({"loss": out["loss"][s]}, d[s], plain(part, tau, alpha), dout[s], dtype, cols, tau)
    assert torch.equal(distill_bwd([inputs, out], dout, grad_out=inputs["vocab_parallel_logits"]), d)
