"""Timed cases of what a training step in low precision adds to a decoder layer: the norm that writes its result in 8 bits with scales,
the quantisation to microscaled 8- and 4-bit floating point, the products of such operands, and the global norm of the gradients with
their clipping.

``listed()`` names a dozen cases, ``draw(rng)`` gives more of the same ranges, ``prepare`` makes a case's inputs, ``run`` takes ONE
pass over them, ``work`` says what a pass cannot do without and ``exact`` what it gives in 64 bits.  With ``own`` false ``run`` is the
plain form in elementary torch operations; with ``own`` true it makes the calls a user makes of this package.

The microscaled format, as both sides hold it: a row is cut into blocks of 32, a block has one power of two as its scale and its elements
in e4m3 (one a byte) or e2m1 (two a byte, the even column in the low half).  Rows are filled up to whole groups of 128 columns with zeros.
``scales[c, r // 4, i, r % 4]`` is the exponent code of row r, columns 128 c + 32 i and on: 2^(code - 127), 255 for a block that holds
anything not finite (its elements are then zeros).  Rows of the scales are filled up to a multiple of four, with zeros as well.
"""
import math

import torch

own = False

DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def listed():
    return [
        # One token through a decoder layer's second norm: launch and host time.
        {"name": "norm_token", "op": "norm", "dtype": "bf16", "rows": 1, "cols": 8192, "residual": True, "centered": False, "rule": "floor"},
        # fp32 activations of a width that is no multiple of a block, no residual, gamma around zero.
        {"name": "norm_odd", "op": "norm", "dtype": "fp32", "rows": 1999, "cols": 1000, "residual": False, "centered": True, "rule": "cover"},
        # The norm of a whole micro-batch behind the attention, residual added on the way.
        {"name": "norm_layer", "op": "norm", "dtype": "bf16", "rows": 8192, "cols": 8192, "residual": True, "centered": False, "rule": "floor"},
        # The gradient of a projection's output in both directions: its rows for the data gradient, its columns for the weight's.
        {"name": "quantise_grad", "op": "quantise", "dtype": "bf16", "rows": 4096, "cols": 7168, "along": "both", "rule": "floor"},
        # A packed batch whose tokens fill no block, fp16, the direction of the weight gradient alone.
        {"name": "quantise_odd", "op": "quantise", "dtype": "fp16", "rows": 1999, "cols": 1001, "along": "columns", "rule": "cover"},
        # One token through a tensor-parallel rank's first feed-forward weight: 8-bit activations, 4-bit weights.
        {"name": "linear_token", "op": "linear", "m": 1, "n": 7168, "k": 8192, "fa": "e4m3", "fb": "e2m1", "dtype": "bf16", "x": "mx"},
        # A few sequences' next tokens, quantised on the way, both in 4 bits.
        {"name": "linear_few", "op": "linear", "m": 24, "n": 8192, "k": 3584, "fa": "e2m1", "fb": "e2m1", "dtype": "bf16", "x": "bf16"},
        # Sizes that fit no tile, fp32 results.
        {"name": "linear_odd", "op": "linear", "m": 777, "n": 1001, "k": 2080, "fa": "e4m3", "fb": "e4m3", "dtype": "fp32", "x": "mx"},
        # The first feed-forward projection of a micro-batch, 8-bit activations quantised on the way, 4-bit weights.
        {"name": "linear_layer", "op": "linear", "m": 4096, "n": 7168, "k": 8192, "fa": "e4m3", "fb": "e2m1", "dtype": "bf16", "x": "bf16"},
        # The largest product, both in 4 bits.
        {"name": "linear_large", "op": "linear", "m": 8192, "n": 8192, "k": 8192, "fa": "e2m1", "fb": "e2m1", "dtype": "bf16", "x": "mx"},
        # Forward, data gradient and weight gradient of the attention's output projection, an odd number of tokens, fp32 main_grad.
        {"name": "linear_step", "op": "step", "tokens": 1999, "n": 8192, "k": 1024, "fx": "e4m3", "fw": "e4m3", "fg": "e4m3"},
        # The gradients of four layers of a rank and its slice of the vocabulary, bf16 to fp32 on the way, clipped.
        {"name": "clip_rank", "op": "clip", "layers": 4, "hidden": 8192, "qkv": 1280, "heads": 1024, "ffn": 3584, "vocab": 16032, "dtype": "bf16",
         "into": "fp32", "max_norm": 1.0, "scale": 0.5, "bad": "none"},
    ]


def _log(rng, lo, hi):
    """A whole number between ``lo`` and ``hi``, spread over its logarithm."""
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    op = rng.choice(["norm", "quantise", "linear", "linear", "step", "clip"])
    if op == "norm":
        cols = rng.choice([32, 100, 1000, 1024, 2047, 4096, 5120, 8192, 16384, _log(rng, 1, 16384)])
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "rows": _log(rng, 1, min(16384, (1 << 25) // cols)), "cols": cols,
                "residual": rng.random() < 0.6, "centered": rng.random() < 0.4, "rule": rng.choice(["floor", "cover"])}
    if op == "quantise":
        cols = rng.choice([32, 1000, 1001, 1024, 4096, 7168, 8192, _log(rng, 1, 16384)])
        return {"op": op, "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "rows": _log(rng, 1, min(16384, (1 << 25) // cols)), "cols": cols,
                "along": rng.choice(["rows", "columns", "both"]), "rule": rng.choice(["floor", "cover"])}
    if op == "linear":
        n, k = rng.choice([(1280, 8192), (8192, 1024), (7168, 8192), (8192, 3584), (1001, 2080), (_log(rng, 1, 8192), _log(rng, 1, 8192))])
        return {"op": op, "m": rng.choice([_log(rng, 1, 64), _log(rng, 64, 8192)]), "n": n, "k": k, "fa": rng.choice(["e4m3", "e2m1"]),
                "fb": rng.choice(["e4m3", "e2m1", "e2m1"]), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]), "x": rng.choice(["mx", "bf16"])}
    if op == "step":
        n, k = rng.choice([(1280, 8192), (8192, 1024), (1000, 520), (_log(rng, 32, 4096), _log(rng, 32, 4096))])
        f = rng.choice(["e4m3", "e2m1"])
        return {"op": op, "tokens": _log(rng, 16, 8192), "n": n, "k": k, "fx": f, "fw": rng.choice(["e4m3", "e2m1"]), "fg": rng.choice(["e4m3", f])}
    hidden = rng.choice([64, 250, 1000, 1024, 4096])
    return {"op": op, "layers": rng.randint(1, 8), "hidden": hidden, "qkv": hidden + 2 * rng.choice([8, 33, 128]), "heads": hidden,
            "ffn": _log(rng, 64, 3 * hidden), "vocab": _log(rng, 100, 32000), "dtype": rng.choice(["bf16", "bf16", "fp16", "fp32"]),
            "into": rng.choice(["fp32", "fp32", "same"]), "max_norm": rng.choice([0.5, 1.0, 1e6]), "scale": rng.choice([1.0, 0.125]),
            "bad": rng.choice(["none", "none", "none", "inf", "nan"])}


# ---- the plain form ---------------------------------------------------------------------------------------------------------------
TOP = {"e4m3": 448.0, "e2m1": 6.0}
TOP_EXPONENT = {"e4m3": 8, "e2m1": 2}
TOP_FRACTION = {"e4m3": 0x600000, "e2m1": 0x400000}


def _up(n, to):
    return -(-n // to) * to


def _e2m1_codes(v):
    """Codes 0..15 of values within +-6, to the nearest, ties to the even code."""
    a = v.abs()
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step
    low = torch.where(a < 2, a * 2, torch.where(a < 4, a + 2, a / 2 + 4))
    return low.to(torch.uint8) + 8 * torch.signbit(v).to(torch.uint8)


def _quantise(x, form, rule):
    """Codes and scales of the rows of a matrix, in 32 bits."""
    rows, cols = x.shape
    kp = _up(cols, 128)
    v = torch.zeros(rows, kp, device=x.device)
    v[:, :cols] = x
    v = v.view(rows, kp // 32, 32)
    top = v.view(torch.int32).bitwise_and(0x7FFFFFFF).amax(2)
    code = (top >> 23) - TOP_EXPONENT[form]
    if rule == "cover":
        code = code + ((top & 0x7FFFFF) > TOP_FRACTION[form]).int()
    code = code.clamp(min=0)
    fine = top < 0x7F800000
    v = v * ((254 - code) << 23).view(torch.float32).unsqueeze(2)
    v = torch.where(fine.unsqueeze(2), v, torch.zeros((), device=x.device)).clamp(-TOP[form], TOP[form]).view(rows, kp)
    code = torch.where(fine, code, torch.full((), 255, device=x.device, dtype=code.dtype)).to(torch.uint8)
    if form == "e4m3":
        codes = v.to(torch.float8_e4m3fn).view(torch.uint8)
    else:
        c = _e2m1_codes(v).view(rows, kp // 2, 2)
        codes = c[:, :, 0] + 16 * c[:, :, 1]
    scales = torch.zeros(_up(rows, 4), kp // 32, dtype=torch.uint8, device=x.device)
    scales[:rows] = code
    return codes, scales.view(-1, 4, kp // 128, 4).permute(2, 0, 3, 1).contiguous()


def _by_rows(scales, rows):
    """The scales' codes as a matrix of a row's blocks."""
    return scales.permute(1, 3, 0, 2).reshape(4 * scales.shape[1], -1)[:rows]


def _values(codes, scales, rows, form, dtype=torch.float32):
    """What codes and scales stand for, filled up to whole groups of 128 columns."""
    if form == "e4m3":
        v = codes.view(torch.float8_e4m3fn).to(dtype)
    else:
        table = torch.tensor([0, 0.5, 1, 1.5, 2, 3, 4, 6, -0.0, -0.5, -1, -1.5, -2, -3, -4, -6], dtype=dtype, device=codes.device)
        v = table[torch.stack([codes & 15, codes >> 4], 2).view(rows, -1).int()]
    code = _by_rows(scales, rows).int()
    bits = torch.where(code == 0, 0x400000, torch.where(code == 255, 0x7FC00000, code << 23)).int()      # 2^-127 is no normal number
    return (v.view(rows, -1, 32) * bits.view(torch.float32).to(dtype).unsqueeze(2)).view(rows, -1)


def _floats(codes, scales):
    """8-bit codes and scales as the floating point numbers that they are."""
    return [codes.view(torch.float8_e4m3fn), scales.view(torch.float8_e8m0fnu)]


# ---- inputs -----------------------------------------------------------------------------------------------------------------------
class _Draws:
    """Tensors on the GPU from one seed."""

    def __init__(self, seed):
        self.gen = torch.Generator(device="cuda").manual_seed(seed)

    def normal(self, *shape, std=1.0, dtype=torch.float32):
        t = torch.randn(shape, generator=self.gen, device="cuda", dtype=torch.float32)
        return (t * std if std != 1.0 else t).to(dtype)

    def activations(self, rows, cols, std=1.0, dtype=torch.float32):
        """Normal values whose rows and some columns differ in size, as activations and gradients do."""
        t = self.normal(rows, cols, std=std)
        t *= torch.exp(self.normal(rows, 1, std=0.7))
        t *= torch.exp(self.normal(1, cols, std=0.5))
        return t.to(dtype)


def _weight(r, rows, cols, form):
    return _quantise(r.normal(rows, cols, std=0.02), form, "cover")


def _shapes(case):
    h = case["hidden"]
    layer = [(h,), (case["qkv"], h), (h, case["heads"]), (h,), (2 * case["ffn"], h), (h, case["ffn"])]
    return layer * case["layers"] + [(h,), (case["vocab"], h)]


def prepare(case, seed):
    r = _Draws(seed)
    s = {"case": case}
    if case["op"] == "norm":
        dt = DTYPES[case["dtype"]]
        s["x"] = r.activations(case["rows"], case["cols"], dtype=dt)
        s["residual"] = r.activations(case["rows"], case["cols"], std=2.0, dtype=dt) if case["residual"] else None
        s["gamma"] = r.normal(case["cols"], std=0.1).add_(0.0 if case["centered"] else 1.0).to(dt)
    elif case["op"] == "quantise":
        s["x"] = r.activations(case["rows"], case["cols"], std=1e-3, dtype=DTYPES[case["dtype"]])
    elif case["op"] == "linear":
        x = r.activations(case["m"], case["k"], dtype=torch.bfloat16)
        s["a"] = _quantise(x.float(), case["fa"], "floor") if case["x"] == "mx" else x
        s["b"] = _weight(r, case["n"], case["k"], case["fb"])
    elif case["op"] == "step":
        t, n, k = case["tokens"], case["n"], case["k"]
        s["x"], s["dy"] = r.activations(t, k, dtype=torch.bfloat16), r.activations(t, n, std=1e-2, dtype=torch.bfloat16)
        w = r.normal(n, k, std=0.02)
        s["w"], s["wt"] = _quantise(w, case["fw"], "cover"), _quantise(w.t().contiguous(), case["fw"], "cover")
        s["main_grad"] = r.normal(n, k, std=0.1)
    else:
        dt = DTYPES[case["dtype"]]
        s["grads"] = [r.normal(*shape, std=10.0 ** -(2 + i % 3), dtype=dt) for i, shape in enumerate(_shapes(case))]
        if case["bad"] != "none":
            s["grads"][1][0, seed % case["hidden"]] = math.inf if case["bad"] == "inf" else math.nan
        s["out"] = [torch.empty_like(g, dtype=torch.float32 if case["into"] == "fp32" else dt) for g in s["grads"]]
    return s


# ---- one pass ---------------------------------------------------------------------------------------------------------------------
EPS = 1e-5


def _own_run(s):
    from dhellam_amd.operators.grads import clip_grads, grad_norm
    from dhellam_amd.operators.layernorm import pyrmsnorm_mx_fwd
    from dhellam_amd.operators.mx import MXTensor, mx_gemm_nt, mx_quantise
    case = s["case"]
    if case["op"] == "norm":
        q, rsigma, total, _ = pyrmsnorm_mx_fwd(s["x"], s["gamma"], EPS, case["centered"], residual=s["residual"], scale_rule=case["rule"])
        return _floats(q.codes, q.scales) + [rsigma] + ([total] if case["residual"] else [])
    if case["op"] == "quantise":
        q, _ = mx_quantise(s["x"], "e4m3", case["along"], case["rule"])
        return [t for one in (q if case["along"] == "both" else (q,)) for t in _floats(one.codes, one.scales)]
    if case["op"] == "linear":
        b = MXTensor(*s["b"], case["n"], case["k"], case["fb"])
        a = MXTensor(*s["a"], case["m"], case["k"], case["fa"]) if case["x"] == "mx" else mx_quantise(s["a"], case["fa"])[0]
        return mx_gemm_nt(a, b, out_dtype=DTYPES[case["dtype"]])
    if case["op"] == "step":
        t, n, k = case["tokens"], case["n"], case["k"]
        (x, xt), _ = mx_quantise(s["x"], case["fx"], "both")
        y = mx_gemm_nt(x, MXTensor(*s["w"], n, k, case["fw"]))
        (g, gt), _ = mx_quantise(s["dy"], case["fg"], "both")
        dx = mx_gemm_nt(g, MXTensor(*s["wt"], k, n, case["fw"]))
        return [y, dx, mx_gemm_nt(gt, xt, out=s["main_grad"], accumulate=True)]
    sum_sq, _ = grad_norm(s["grads"])
    found, _ = clip_grads(s["grads"], sum_sq, case["max_norm"], scale=case["scale"], out=s["out"])
    return [found] + s["out"]


def run(s):
    if own:
        return _own_run(s)
    case = s["case"]
    if case["op"] == "norm":
        dt = s["x"].dtype
        total = (s["x"].float() + s["residual"].float()).to(dt) if case["residual"] else s["x"]
        v = total.float()
        rsigma = torch.rsqrt(v.square().mean(1) + EPS)
        y = v * rsigma.unsqueeze(1) * (s["gamma"].float() + (1.0 if case["centered"] else 0.0))
        return _floats(*_quantise(y, "e4m3", case["rule"])) + [rsigma] + ([total] if case["residual"] else [])
    if case["op"] == "quantise":
        x = s["x"].float()
        out = _floats(*_quantise(x, "e4m3", case["rule"])) if case["along"] != "columns" else []
        return out + (_floats(*_quantise(x.t().contiguous(), "e4m3", case["rule"])) if case["along"] != "rows" else [])
    if case["op"] == "linear":
        a = s["a"] if case["x"] == "mx" else _quantise(s["a"].float(), case["fa"], "floor")
        return (_values(*a, case["m"], case["fa"]) @ _values(*s["b"], case["n"], case["fb"]).t()).to(DTYPES[case["dtype"]])
    if case["op"] == "step":
        t, n, k = case["tokens"], case["n"], case["k"]
        x, dy = s["x"].float(), s["dy"].float()
        y = _values(*_quantise(x, case["fx"], "floor"), t, case["fx"]) @ _values(*s["w"], n, case["fw"]).t()
        dx = _values(*_quantise(dy, case["fg"], "floor"), t, case["fg"]) @ _values(*s["wt"], k, case["fw"]).t()
        xt = _values(*_quantise(x.t().contiguous(), case["fx"], "floor"), k, case["fx"])
        gt = _values(*_quantise(dy.t().contiguous(), case["fg"], "floor"), n, case["fg"])
        s["main_grad"] += gt @ xt.t()
        return [y.to(torch.bfloat16), dx.to(torch.bfloat16), s["main_grad"]]
    norm = case["scale"] * torch.stack([g.double().square().sum() for g in s["grads"]]).sum().sqrt()
    fine = torch.isfinite(norm)
    factor = torch.where(fine, case["scale"] * (case["max_norm"] / (norm + 1e-6)).clamp(max=1.0), torch.zeros_like(norm))
    out = [torch.where(fine, g.float() * factor.float(), torch.zeros((), device="cuda")).to(o.dtype) for g, o in zip(s["grads"], s["out"])]
    return [torch.stack([norm, factor]).float()] + out


# ---- what a pass cannot do without ------------------------------------------------------------------------------------------------
def _mx_bytes(rows, cols, form):
    kp = _up(cols, 128)
    return rows * kp * (1.0 if form == "e4m3" else 0.5) + rows * kp / 32


def work(case):
    size = {"bf16": 2, "fp16": 2, "fp32": 4}
    if case["op"] == "norm":
        r, c, es = case["rows"], case["cols"], size[case["dtype"]]
        return {"bytes": r * c * es * (3 if case["residual"] else 1) + c * es + 4 * r + _mx_bytes(r, c, "e4m3"), "flops": 6 * r * c}
    if case["op"] == "quantise":
        r, c = case["rows"], case["cols"]
        out = (_mx_bytes(r, c, "e4m3") if case["along"] != "columns" else 0) + (_mx_bytes(c, r, "e4m3") if case["along"] != "rows" else 0)
        return {"bytes": r * c * size[case["dtype"]] + out, "flops": 3 * r * c}
    if case["op"] == "linear":
        m, n, k = case["m"], case["n"], case["k"]
        a = _mx_bytes(m, k, case["fa"]) if case["x"] == "mx" else 2 * m * k
        return {"bytes": a + _mx_bytes(n, k, case["fb"]) + m * n * size[case["dtype"]], "flops": 2 * m * n * k}
    if case["op"] == "step":
        t, n, k = case["tokens"], case["n"], case["k"]
        return {"bytes": 2 * (2 * t * k + 2 * t * n) + _mx_bytes(n, k, case["fw"]) + _mx_bytes(k, n, case["fw"]) + 8 * n * k, "flops": 6 * t * n * k}
    count, es = sum(math.prod(x) for x in _shapes(case)), size[case["dtype"]]
    # every gradient before the first is written: read again unless it is still on the chip, which is not counted here
    return {"bytes": count * (es + (4 if case["into"] == "fp32" else es)), "flops": 3 * count}


# ---- the same in 64 bits ----------------------------------------------------------------------------------------------------------
def _grid(form):
    """The values from 0 up that a format has, by their definition."""
    bits, bias, codes = (3, 7, 127) if form == "e4m3" else (1, 1, 8)
    one = 1 << bits
    return [(c % one / one if c < one else (1 + c % one / one) * 2.0 ** (c // one - 1)) * 2.0 ** (1 - bias) for c in range(codes)]


def _nearest(v, form):
    """The nearest values of the format, ties to the even code: the half-way points decide."""
    g = torch.tensor(_grid(form), dtype=torch.float64, device=v.device)
    half = (g[1:] + g[:-1]) / 2
    a = v.abs().contiguous()
    i = torch.searchsorted(half, a)                                    # ties fall to the lower one
    i += ((i < len(half)) & (half[i.clamp(max=len(half) - 1)] == a) & (i % 2 == 1)).long()
    return torch.where(v < 0, -g[i], g[i])


def _power64(exponent):
    """2 to whole numbers, exactly (a power function may be off in the last bit, and a half-way point then is none)."""
    return ((exponent.long() + 1023) << 52).view(torch.float64)


def _parts64(x, form, rule):
    """Elements and scales of the rows of a matrix, in 64 bits, a block in a row of its own."""
    rows, cols = x.shape
    x = torch.nn.functional.pad(x, (0, _up(cols, 128) - cols)).reshape(-1, 32)
    top = x.abs().amax(1)
    exponent = torch.frexp(top).exponent.long() - 1 - TOP_EXPONENT[form]
    exponent = torch.where(top > 0, exponent, torch.full_like(exponent, -127)).clamp(min=-127)
    if rule == "cover":
        exponent += (top > TOP[form] * _power64(exponent)).long()
    scale = _power64(exponent)
    return _nearest((x / scale.unsqueeze(1)).clamp(-TOP[form], TOP[form]), form), scale


def _held64(x, form, rule):
    """The same as a matrix of what it stands for."""
    e, scale = _parts64(x, form, rule)
    return (e * scale.unsqueeze(1)).view(x.shape[0], -1)


def _laid_out64(x, rule):
    """Elements and scales as ``run`` gives them."""
    rows = x.shape[0]
    e, scale = _parts64(x, "e4m3", rule)
    laid = torch.full((_up(x.shape[1], 128) // 128, _up(rows, 4) // 4, 4, 4), 2.0 ** -127, dtype=torch.float64, device=x.device)
    r = torch.arange(rows, device=x.device)
    laid[:, r // 4, :, r % 4] = scale.view(rows, -1, 4)
    return [e.view(rows, -1), laid]


def _decoded64(pair, rows, form):
    """The values of given codes and scales, by the definition of the format."""
    codes, scales = pair
    g = torch.tensor(_grid(form), dtype=torch.float64, device=codes.device)
    g = torch.cat([g, g.new_zeros(1), -g, g.new_zeros(1)]) if form == "e4m3" else torch.cat([g, -g])
    c = codes.long() if form == "e4m3" else torch.stack([codes.long() % 16, codes.long() // 16], 2).view(rows, -1)
    r = torch.arange(rows, device=codes.device)
    power = _power64(scales[:, r // 4, :, r % 4].long() - 127)
    return g[c] * power.reshape(rows, -1).repeat_interleave(32, 1)


def exact(case, seed):
    s = prepare(case, seed)
    if case["op"] == "norm":
        x = s["x"].double()
        total = (x + s["residual"].double()) if case["residual"] else x
        held = total.to(s["x"].dtype).double()                         # what is normalised is the sum as it is stored
        r = 1.0 / torch.sqrt((held * held).sum(1) / case["cols"] + EPS)
        y = held * r[:, None] * (s["gamma"].double() + float(case["centered"]))
        return _laid_out64(y, case["rule"]) + [r] + ([total] if case["residual"] else [])
    if case["op"] == "quantise":
        x = s["x"].double()
        return (_laid_out64(x, case["rule"]) if case["along"] != "columns" else []) + (_laid_out64(x.t(), case["rule"]) if case["along"] != "rows" else [])
    if case["op"] == "linear":
        a = _decoded64(s["a"], case["m"], case["fa"]) if case["x"] == "mx" else _held64(s["a"].double(), case["fa"], "floor")
        return a @ _decoded64(s["b"], case["n"], case["fb"]).t()
    if case["op"] == "step":
        t, n, k = case["tokens"], case["n"], case["k"]
        x, dy = s["x"].double(), s["dy"].double()
        y = _held64(x, case["fx"], "floor") @ _decoded64(s["w"], n, case["fw"]).t()
        dx = _held64(dy, case["fg"], "floor") @ _decoded64(s["wt"], k, case["fw"]).t()
        return [y, dx, s["main_grad"].double() + _held64(dy.t(), case["fg"], "floor") @ _held64(x.t(), case["fx"], "floor").t()]
    norm = case["scale"] * math.sqrt(sum(float((g.double() ** 2).sum()) for g in s["grads"]))
    if not math.isfinite(norm):
        return [torch.tensor([norm, 0.0], dtype=torch.float64)] + [torch.zeros_like(g, dtype=torch.float64) for g in s["grads"]]
    factor = case["scale"] * min(1.0, case["max_norm"] / (norm + 1e-6))
    return [torch.tensor([norm, factor], dtype=torch.float64)] + [g.double() * factor for g in s["grads"]]
