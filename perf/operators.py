"""Timed cases of three operators of a training step: rotary positions in their general form, the router's losses and gradients,
and the distillation loss against a teacher's top logits.

``listed()`` names a dozen cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes a case's inputs, ``run`` takes ONE
pass over them, ``work`` says what a pass cannot do without and ``exact`` what it gives in 64 bits.  With ``own`` false ``run`` is the
plain form in elementary torch operations; with ``own`` true it makes the calls a user makes of this package.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One token of a decoder far into its context, frequencies scaled by parts: launch and host time.
        {"name": "rotary_token", "op": "rotary", "dir": "fwd", "dtype": "bf16", "tokens": 1, "hq": 32, "hk": 8, "d": 128, "rot": 128,
         "interleaved": False, "scaling": "parts", "positions": "far"},
        # A quarter-turned head in interleaved pairs, a token count that fits nothing.
        {"name": "rotary_part", "op": "rotary", "dir": "fwd", "dtype": "fp16", "tokens": 1999, "hq": 16, "hk": 16, "d": 80, "rot": 20,
         "interleaved": True, "scaling": "none", "positions": "packed"},
        # The gradient of a tensor-parallel rank's q and k, views of the packed projection, sequence of 4096.
        {"name": "rotary_shard", "op": "rotary", "dir": "bwd", "dtype": "bf16", "tokens": 4096, "hq": 8, "hk": 1, "d": 128, "rot": 128,
         "interleaved": False, "scaling": "bands", "positions": "sequence"},
        # A long packed context, whole heads, interleaved.
        {"name": "rotary_long", "op": "rotary", "dir": "fwd", "dtype": "bf16", "tokens": 65536, "hq": 32, "hk": 8, "d": 128, "rot": 128,
         "interleaved": True, "scaling": "ntk", "positions": "far"},
        # Router of a small mixture on a handful of tokens: losses, counts, and the gradient of the logits.
        {"name": "router_tiny", "op": "router", "tokens": 64, "experts": 8, "k": 2, "mask": False, "gates": True},
        # The mixture layer of the benchmark, a padded batch.
        {"name": "router_rank", "op": "router", "tokens": 8192, "experts": 8, "k": 2, "mask": True, "gates": True},
        # Many fine experts over a large batch.
        {"name": "router_fine", "op": "router", "tokens": 131072, "experts": 64, "k": 8, "mask": True, "gates": True},
        # A number of experts that is no power of two, balance and z loss alone.
        {"name": "router_odd", "op": "router", "tokens": 30011, "experts": 60, "k": 6, "mask": False, "gates": False},
        # Validation of a few rows over a whole vocabulary: the loss alone.
        {"name": "distill_rows", "op": "distill", "dir": "fwd", "dtype": "bf16", "rows": 16, "cols": 128256, "k": 64, "temperature": 1.0,
         "alpha": 1.0, "whole": False, "padded": False, "teacher": "fp32"},
        # fp32 logits of an odd vocabulary (rows off the 16-byte grid), the teacher's log-sum-exp at hand.
        {"name": "distill_odd", "op": "distill", "dir": "step", "dtype": "fp32", "rows": 1000, "cols": 50257, "k": 32, "temperature": 1.5,
         "alpha": 1.0, "whole": True, "padded": True, "teacher": "fp32"},
        # A rank's slice as the only one: forward and backward of one micro-batch, mixed with the labels' cross entropy.
        {"name": "distill_shard", "op": "distill", "dir": "step", "dtype": "bf16", "rows": 4096, "cols": 16032, "k": 64, "temperature": 2.0,
         "alpha": 0.5, "whole": False, "padded": True, "teacher": "bf16"},
        # The whole vocabulary on one GPU.
        {"name": "distill_full", "op": "distill", "dir": "step", "dtype": "bf16", "rows": 4096, "cols": 128256, "k": 128, "temperature": 1.0,
         "alpha": 0.5, "whole": False, "padded": False, "teacher": "fp32"},
    ]


def _log(rng, lo, hi):
    """A whole number between ``lo`` and ``hi``, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["rotary", "router", "distill"])
    if op == "rotary":
        hq, hk = rng.choice([(8, 1), (16, 16), (32, 8), (4, 2), (12, 4), (1, 1)])
        d = rng.choice([64, 64, 80, 96, 128, 128, 192, 256])
        return {"op": op, "dir": rng.choice(["fwd", "bwd"]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
                "tokens": _log(rng, 1, min(65536, 65536 * 40 * 64 // ((hq + hk) * d))), "hq": hq, "hk": hk, "d": d,
                "rot": rng.choice([d, d, d // 2, d // 4, 2 * rng.randint(1, d // 2)]), "interleaved": rng.random() < 0.5,
                "scaling": rng.choice(["none", "linear", "ntk", "parts", "bands"]),
                "positions": rng.choice(["sequence", "packed", "far"])}
    if op == "router":
        experts, k = rng.choice([(2, 1), (5, 3), (8, 1), (8, 2), (8, 2), (16, 4), (24, 2), (60, 6), (64, 1), (64, 8)])
        return {"op": op, "tokens": _log(rng, 1, 131072), "experts": experts, "k": k, "mask": rng.random() < 0.5,
                "gates": rng.random() < 0.7}
    cols = rng.choice([1000, 4001, 16032, 32000, 50257, 50304, 128256])
    return {"op": op, "dir": rng.choice(["fwd", "step", "step"]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "rows": _log(rng, 1, min(8192, 4096 * 64128 // cols)), "cols": cols, "k": rng.choice([1, 8, 20, 32, 64, 100, 128, 256]),
            "temperature": rng.choice([0.7, 1.0, 1.0, 1.5, 2.0, 4.0]), "alpha": rng.choice([0.3, 0.5, 0.9, 1.0, 1.0]),
            "whole": rng.random() < 0.4, "padded": rng.random() < 0.5, "teacher": rng.choice(["fp32", "bf16"])}


class _Draws:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return (t * std if std != 1.0 else t).to(dtype)

    def uniform(self, *shape):
        return torch.rand(shape, generator=self.gen, device="cuda")

    def ids(self, low, high, *shape):
        return torch.randint(low, high, shape, generator=self.gen, device="cuda")


THETA = 500000.0

SCALING = {"none": None, "linear": {"kind": "linear", "factor": 4.0}, "ntk": {"kind": "ntk", "factor": 8.0},
           "parts": {"kind": "parts", "factor": 16.0, "original_length": 4096, "beta_fast": 32.0, "beta_slow": 1.0},
           "bands": {"kind": "bands", "factor": 8.0, "original_length": 8192, "low": 1.0, "high": 4.0}}


def _frequencies(case):
    """The frequencies of a head's pairs and the factor on cos and sin, in Python's 64-bit floats."""
    dim, s = case["rot"], SCALING[case["scaling"]]
    f = [THETA ** (-2.0 * j / dim) for j in range(dim // 2)]
    if s is None:
        return f, 1.0
    n = s["factor"]
    if s["kind"] == "linear":
        return [x / n for x in f], 1.0
    if s["kind"] == "ntk":
        if dim == 2:
            return f, 1.0
        base = THETA * n ** (dim / (dim - 2.0))
        return [base ** (-2.0 * j / dim) for j in range(dim // 2)], 1.0
    length = s["original_length"]
    if s["kind"] == "parts":
        edge = lambda beta: dim * math.log(length / (beta * 2.0 * math.pi)) / (2.0 * math.log(THETA))
        lo, hi = max(math.floor(edge(s["beta_fast"])), 0), min(math.ceil(edge(s["beta_slow"])), dim - 1)
        span = float(hi - lo) if hi != lo else 0.001
        ramp = [min(max((j - lo) / span, 0.0), 1.0) for j in range(dim // 2)]
        return [x / n * r + x * (1.0 - r) for x, r in zip(f, ramp)], 0.1 * math.log(n) + 1.0
    out = []
    for x in f:
        wave = 2.0 * math.pi / x
        if wave < length / s["high"]:
            out.append(x)
        elif wave > length / s["low"]:
            out.append(x / n)
        else:
            t = (length / wave - s["low"]) / (s["high"] - s["low"])
            out.append((1.0 - t) * x / n + t * x)
    return out, 1.0


def _inputs(case, seed):
    r = _Draws(seed)
    s = {"case": case}
    if case["op"] == "rotary":
        dt = DTYPES[case["dtype"]]
        t, hq, hk, d = (case[x] for x in ("tokens", "hq", "hk", "d"))
        packed = r.normal(t, (hq + 2 * hk) * d, dtype=dt)      # q and k are views of the packed projection
        s["q"], s["k"] = packed[:, :hq * d].view(t, hq, d), packed[:, hq * d:(hq + hk) * d].view(t, hk, d)
        at = torch.arange(t, device="cuda")
        if case["positions"] == "packed":                     # documents behind one another, each from position 0
            at = at % max(1, t // 3 + 1)
        elif case["positions"] == "far":                      # a chunk of a context of a million
            at = at + int(r.ids(0, 1 << 20, 1))
        s["positions"] = None if case["positions"] == "sequence" else at.to(torch.int32)
        return s
    if case["op"] == "router":
        t, e, k = case["tokens"], case["experts"], case["k"]
        s["logits"] = r.normal(t, e, std=1.5) + r.normal(e)                    # some experts are liked more than others
        top, idx = torch.topk(s["logits"], k, dim=1)
        s["idx"], s["gates"] = idx.to(torch.int32).contiguous(), torch.softmax(top, 1).contiguous()
        s["dgates"] = r.normal(t, k, std=0.1) if case["gates"] else None
        s["mask"] = r.uniform(t) < 0.8 if case["mask"] else None
        return s
    dt = DTYPES[case["dtype"]]
    n, cols, k = case["rows"], case["cols"], case["k"]
    # distinct ids a row, the best first, a student that leans the teacher's way
    step = r.ids(1, cols // k + 1, n, 1)
    s["ids"] = (r.ids(0, cols, n, 1) + torch.arange(k, device="cuda") * step) % cols
    teacher = r.normal(n, k, std=2.0).sort(1, descending=True).values + 4.0
    s["logits"] = r.normal(n, cols, std=1.5, dtype=dt).scatter_add_(1, s["ids"], (0.7 * teacher).to(dt))
    s["teacher"] = teacher.to(DTYPES[case["teacher"]])
    if case["padded"]:                                        # lists of several lengths, some of them empty
        s["ids"].masked_fill_(torch.arange(k, device="cuda") >= r.ids(0, k + 1, n, 1), -1)
    s["lse"] = None
    if case["whole"]:                                         # the list holds nine tenths of what the teacher says
        s["lse"] = torch.logsumexp(s["teacher"].float() / case["temperature"], 1) + math.log(10.0 / 9.0)
    s["target"] = r.ids(0, cols, n) if case["alpha"] < 1.0 else None
    s["dout"] = r.uniform(n) / n
    return s


def prepare(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rotary":                                # a program makes its table of frequencies once
        if own:
            from dhellam_amd.operators.rope import rotary_table
            s["table"] = rotary_table(THETA, case["rot"], s["q"].device, case["interleaved"], SCALING[case["scaling"]])
        else:
            f, s["factor"] = _frequencies(case)
            s["freq"] = torch.tensor(f, dtype=torch.float64, device="cuda")
    return s


BALANCE, Z = 0.01, 0.001      # usual weights of the two losses


def _plain_rotary(s):
    case = s["case"]
    rot, back = case["rot"], case["dir"] == "bwd"
    t = case["tokens"]
    at = s["positions"].double() if s["positions"] is not None else torch.arange(t, device="cuda", dtype=torch.float64)
    angle = at[:, None] * s["freq"][None, :]
    cos, sin = (torch.cos(angle) * s["factor"]).float()[:, None, :], (torch.sin(angle) * s["factor"]).float()[:, None, :]
    if back:
        sin = -sin
    outs = []
    for x in (s["q"], s["k"]):
        y = x.float()
        if case["interleaved"]:
            a, b = y[..., 0:rot:2], y[..., 1:rot:2]
            turned = torch.stack((a * cos - b * sin, b * cos + a * sin), -1).flatten(-2)
        else:
            a, b = y[..., :rot // 2], y[..., rot // 2:rot]
            turned = torch.cat((a * cos - b * sin, b * cos + a * sin), -1)
        outs.append(torch.cat((turned, y[..., rot:]), -1).to(x.dtype))
    return outs


def _plain_router(s):
    x, idx, gates, dgates = s["logits"], s["idx"].long(), s["gates"], s["dgates"]
    t, e = x.shape
    k = idx.shape[1]
    m = s["mask"].float() if s["mask"] is not None else torch.ones(t, device=x.device)
    n = m.sum().clamp(min=1.0)
    top = x.max(1, keepdim=True).values
    ex = torch.exp(x - top)
    total = ex.sum(1, keepdim=True)
    p, lse = ex / total, (torch.log(total) + top)[:, 0]
    chosen = torch.zeros_like(x).scatter_add_(1, idx, torch.ones_like(gates))
    counts = (chosen * m[:, None]).sum(0)
    probs = (p * m[:, None]).sum(0)
    scale = BALANCE * e / (k * n * n)
    losses = torch.stack((scale * (counts * probs).sum(), Z / n * (m * lse * lse).sum()))
    d = m[:, None] * (scale * p * (counts - (counts * p).sum(1, keepdim=True)) + (2.0 * Z / n) * lse[:, None] * p)
    if dgates is not None:
        d = d.scatter_add(1, idx, gates * (dgates - (gates * dgates).sum(1, keepdim=True)))
    return [losses, counts.to(torch.int32), probs, d]


def _plain_distill(s):
    case = s["case"]
    tau, alpha = case["temperature"], case["alpha"]
    x, ids = s["logits"].float(), s["ids"]
    there = ids >= 0
    at = ids.clamp(min=0)
    teacher = torch.where(there, s["teacher"].float() / tau, torch.full((), -math.inf, device=x.device))
    if s["lse"] is not None:
        norm = s["lse"][:, None]
    else:
        best = teacher.max(1, keepdim=True).values.clamp(min=-1e30)
        norm = best + torch.log(torch.exp(teacher - best).sum(1, keepdim=True))
        norm = torch.where(there.any(1, keepdim=True), norm, torch.zeros_like(norm))
    logp = torch.where(there, teacher - norm, torch.zeros_like(teacher))
    p = torch.where(there, torch.exp(logp), torch.zeros_like(logp))
    top = x.max(1, keepdim=True).values
    ex = torch.exp((x - top) / tau)
    total = ex.sum(1, keepdim=True)
    logq = (x.gather(1, at) - top) / tau - torch.log(total)
    loss = alpha * tau * tau * (p * (logp - logq)).sum(1)
    if alpha < 1.0:
        ex1 = torch.exp(x - top)
        total1 = ex1.sum(1, keepdim=True)
        loss = loss + (1.0 - alpha) * (torch.log(total1) + top - x.gather(1, s["target"][:, None]))[:, 0]
    if case["dir"] == "fwd":
        return [loss]
    d = alpha * tau * p.sum(1, keepdim=True) * ex / total
    d = d.scatter_add_(1, at, -alpha * tau * p)
    if alpha < 1.0:
        d += (1.0 - alpha) * ex1 / total1
        d.scatter_add_(1, s["target"][:, None], torch.full_like(total1, alpha - 1.0))
    return [loss, (d * s["dout"][:, None]).to(s["logits"].dtype)]


_PLAIN = {"rotary": _plain_rotary, "router": _plain_router, "distill": _plain_distill}


def _own_rotary(s):
    from dhellam_amd.operators.rope import rotary_bwd, rotary_fwd
    turn = rotary_bwd if s["case"]["dir"] == "bwd" else rotary_fwd
    q, k, _ = turn(s["q"], s["k"], s["table"], s["positions"])
    return [q, k]


def _own_router(s):
    from dhellam_amd.operators.moe import balance_loss_fwd, route_bwd
    losses, balance, _ = balance_loss_fwd(s["logits"], s["idx"], s["mask"], BALANCE, Z)
    d, _ = route_bwd(s["logits"], s["idx"], s["gates"], s["dgates"], balance)
    return [losses, balance.counts, balance.prob_sum, d]


def _own_distill(s):
    from dhellam_amd.operators.loss import distill_bwd, distill_fwd
    case = s["case"]
    inputs = {"vocab_parallel_logits": s["logits"], "teacher_ids": s["ids"], "teacher_logits": s["teacher"], "teacher_lse": s["lse"],
              "target": s["target"]}
    out = distill_fwd(inputs, case["temperature"], case["alpha"])
    if case["dir"] == "fwd":
        return [out["loss"]]
    return [out["loss"], distill_bwd([inputs, out], s["dout"])]


_OWN = {"rotary": _own_rotary, "router": _own_router, "distill": _own_distill}


def run(state):
    return (_OWN if own else _PLAIN)[state["case"]["op"]](state)


def work(case):
    if case["op"] == "rotary":
        e, t, h = 4 if case["dtype"] == "fp32" else 2, case["tokens"], case["hq"] + case["hk"]
        at = 0 if case["positions"] == "sequence" else 4 * t
        return {"bytes": 2 * e * t * h * case["d"] + at, "flops": 3 * t * h * case["rot"] + 40 * t * case["rot"] // 2}
    if case["op"] == "router":
        t, e, k = case["tokens"], case["experts"], case["k"]
        # logits in, their gradient out; the choices, and the gates with their gradient where they take part
        return {"bytes": 8 * t * e + 4 * t * k * (3 if case["gates"] else 1) + (t if case["mask"] else 0) + 8 * e + 8,
                "flops": 15 * t * e + 6 * t * k}
    e, te = (4 if case[x] == "fp32" else 2 for x in ("dtype", "teacher"))
    n, cols, k = case["rows"], case["cols"], case["k"]
    passes, row = (2 if case["dir"] == "step" else 1), 4 + (4 if case["whole"] else 0) + (8 if case["alpha"] < 1.0 else 0)
    return {"bytes": passes * e * n * cols + n * (k * (8 + te) + row + (4 if passes == 2 else 0)),
            "flops": n * cols * (6 if case["alpha"] == 1.0 else 9) * passes + 20 * n * k}


def _exact_rotary(case, s):
    f, factor = _frequencies(case)
    f = torch.tensor(f, dtype=torch.float64, device="cuda")
    t, rot = case["tokens"], case["rot"]
    at = torch.arange(t, device="cuda") if s["positions"] is None else s["positions"]
    turn = torch.polar(torch.full((t, rot // 2), factor, dtype=torch.float64, device="cuda"), at.double()[:, None] * f)
    if case["dir"] == "bwd":
        turn = turn.conj()
    outs = []
    for x in (s["q"], s["k"]):
        y = x.double()
        z = y.clone()
        first, second = (slice(0, rot, 2), slice(1, rot, 2)) if case["interleaved"] else (slice(0, rot // 2), slice(rot // 2, rot))
        w = torch.complex(y[..., first].contiguous(), y[..., second].contiguous()) * turn[:, None, :]
        z[..., first], z[..., second] = w.real, w.imag
        outs.append(z)
    return outs


def _exact_router(s):
    """The derivative of the two losses and of the gates' share by 64-bit autograd; counts one expert at a time."""
    x = s["logits"].double().requires_grad_(True)
    t, e = x.shape
    idx, m = s["idx"].long(), torch.ones(t, dtype=torch.float64, device=x.device)
    if s["mask"] is not None:
        m = s["mask"].double()
    n, k = m.sum(), idx.shape[1]
    counts = torch.stack([((idx == i).double().sum(1) * m).sum() for i in range(e)])
    lse = torch.logsumexp(x, 1)
    probs = (torch.softmax(x, 1) * m[:, None]).sum(0)
    if float(n) > 0:
        losses = torch.stack((BALANCE * e / k * (counts / n * (probs / n)).sum(), Z * (lse ** 2 * m).sum() / n))
    else:
        losses = torch.zeros(2, dtype=torch.float64, device=x.device) * x.sum()
    total = losses.sum()
    if s["dgates"] is not None:
        # the gates that were given are the softmax of the chosen logits in 32 bits
        g, dg = s["gates"].double(), s["dgates"].double()
        chosen = x.gather(1, idx)
        jac = g * dg - g * (g * dg).sum(1, keepdim=True)
        total = total + (chosen * jac).sum()
    (d,) = torch.autograd.grad(total, x)
    return [losses.detach(), counts.to(torch.int32), probs.detach(), d]


def _exact_distill(case, s):
    """Rows a block at a time: distributions by log-softmax, gradients of the listed entries one column at a time."""
    tau, alpha, n, cols, k = case["temperature"], case["alpha"], case["rows"], case["cols"], case["k"]
    losses, grads = [], []
    step = max(1, (1 << 27) // cols)
    for lo in range(0, n, step):
        at = slice(lo, min(n, lo + step))
        x, ids, t = s["logits"][at].double(), s["ids"][at], s["teacher"][at].double() / tau
        there = ids >= 0
        t = t.masked_fill(~there, -math.inf)
        norm = s["lse"][at].double()[:, None] if s["lse"] is not None else torch.logsumexp(t, 1, keepdim=True)
        p = torch.exp(t - norm).masked_fill(~there, 0.0)
        soft = torch.log_softmax(x / tau, 1)
        col = ids.clamp(min=0)
        loss = alpha * tau ** 2 * ((t - norm).masked_fill(~there, 0.0) * p - soft.gather(1, col) * p).sum(1)
        g = torch.exp(soft) * p.sum(1, keepdim=True) * (alpha * tau)
        rows = torch.arange(x.shape[0], device=x.device)
        for j in range(k):
            g[rows, col[:, j]] -= alpha * tau * p[:, j]
        if alpha < 1.0:
            hard = torch.log_softmax(x, 1)
            loss = loss - (1.0 - alpha) * hard[rows, s["target"][at]]
            hard = torch.exp(hard)
            hard[rows, s["target"][at]] -= 1.0
            g += (1.0 - alpha) * hard
        losses.append(loss)
        if case["dir"] == "step":
            grads.append(g * s["dout"][at].double()[:, None])
    return [torch.cat(losses)] + ([torch.cat(grads)] if grads else [])


def exact(case, seed):
    s = _inputs(case, seed)
    if case["op"] == "rotary":
        return _exact_rotary(case, s)
    return _exact_router(s) if case["op"] == "router" else _exact_distill(case, s)
