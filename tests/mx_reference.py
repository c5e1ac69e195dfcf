"""Microscaled floating point in 64 bits, written from its definition: what the GPU tests of its operators compare with."""
import torch

TOP = {"e4m3": 448.0, "e2m1": 6.0}
EMAX = {"e4m3": 8, "e2m1": 2}


def up(n, to):
    return -(-n // to) * to


def grid(form):
    """The non-negative values of a format by code."""
    mant, bias, codes = (3, 7, 127) if form == "e4m3" else (1, 1, 8)
    one = 1 << mant
    return torch.tensor([(c / one if c < one else (1 + c % one / one) * 2.0 ** (c // one - 1)) * 2.0 ** (1 - bias) for c in range(codes)],
                        dtype=torch.float64)


def power(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def scale_codes(x, form, rule):
    """int64 [rows, kp / 32] of a matrix."""
    rows, cols = x.shape
    v = torch.nn.functional.pad(x.double(), (0, up(cols, 128) - cols)).reshape(rows, -1, 32)
    top = v.abs().amax(2)
    fine = torch.isfinite(v).all(2)
    top = torch.where(fine, top, 1.0)
    e = torch.where(top > 0, torch.frexp(top).exponent.long() - 1 - EMAX[form], -127).clamp(min=-127)
    if rule == "cover":
        e = e + (top > TOP[form] * power(e)).long()
    return torch.where(fine, e + 127, 255)


def element_codes(x, codes, form):
    """uint8 codes [rows, kp], one an element, of a matrix under given scale codes."""
    rows, cols = x.shape
    g = grid(form).to(x.device)
    v = torch.nn.functional.pad(x.double(), (0, up(cols, 128) - cols)).reshape(rows, -1, 32)
    fine = (codes < 255).unsqueeze(2)
    a = torch.where(fine, v.abs() / power(torch.where(codes < 255, codes, 127) - 127).unsqueeze(2), 0.0)
    half = (g[1:] + g[:-1]) / 2
    i = torch.searchsorted(half, a.contiguous())
    i = i + ((i < len(half)) & (half[i.clamp(max=len(half) - 1)] == a) & (i % 2 == 1)).long()
    sign = torch.signbit(v) & fine
    return (i + sign * (128 if form == "e4m3" else 8)).to(torch.uint8).reshape(rows, -1)


def pack(elements, form):
    return elements if form == "e4m3" else elements[:, 0::2] + 16 * elements[:, 1::2]


def lay_out(codes, rows):
    """Scale codes [rows, kp / 32] as the operators hold them."""
    full = torch.zeros(up(rows, 4), codes.shape[1], dtype=torch.uint8, device=codes.device)
    full[:rows] = codes.to(torch.uint8)
    return full.reshape(-1, 4, codes.shape[1] // 4, 4).permute(2, 0, 3, 1).contiguous()


def quantise(x, form, rule="floor"):
    """codes, scales as ``MXTensor`` holds them."""
    s = scale_codes(x, form, rule)
    return pack(element_codes(x, s, form), form), lay_out(s, x.shape[0])


def values(q):
    """fp64 [rows, kp] of an ``MXTensor``."""
    g = grid(q.format).to(q.codes.device)
    g = torch.cat([g, g.new_full((1,), float("nan")), -g, g.new_full((1,), float("nan"))]) if q.format == "e4m3" else torch.cat([g, -g])
    e = q.codes.long() if q.format == "e4m3" else torch.stack([q.codes.long() % 16, q.codes.long() // 16], 2).reshape(q.rows, -1)
    s = q.scales.permute(1, 3, 0, 2).reshape(4 * q.scales.shape[1], -1)[:q.rows].long()
    p = torch.where(s == 255, torch.full((), float("nan"), dtype=torch.float64, device=s.device), power(s - 127))
    return g[e] * p.repeat_interleave(32, 1)
