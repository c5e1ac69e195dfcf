"""Rotary position embedding on q and k: ``rope_*`` turn the halves of whole heads, ``rotary_*`` take a table of
``rotary_table`` and turn a part of the head, in halves or interleaved pairs, with frequencies scaled for long contexts.

The reference has no RoPE; these wrappers follow its operator convention and sit
where a Llama layer needs them: after the q/k/v split and before the attention
call (dhellam/core/dstb.py:122-126), and on dq/dk before the dq|dk|dv concat in
backward (:376-382).
"""
from __future__ import annotations

import math
from dataclasses import dataclass
from typing import Optional

import torch

from .. import _host
from ._util import issue

_inv_freq_cache: dict = {}


def rope_inv_freq(theta: float, d: int, device) -> torch.Tensor:
    """fp32 [d/2] table theta^(-2j/d), evaluated in double and rounded once."""
    key = (theta, d, device)
    t = _inv_freq_cache.get(key)
    if t is None:
        vals = [float(theta) ** (-2.0 * j / d) for j in range(d // 2)]
        t = torch.tensor(vals, dtype=torch.float64).to(torch.float32).to(device)
        _inv_freq_cache[key] = t
    return t


def _rope(q, k, positions, theta, seq_len, backward, stream, profiling, inplace):
    inv = rope_inv_freq(theta, q.shape[-1], q.device)
    (qo, ko), ms = issue(_host.rope, stream, profiling, q, k, inv, positions, int(seq_len or 0), backward, inplace)
    return (q, k, ms) if inplace else (qo, ko, ms)


def rope_fwd(q, k, positions=None, theta=10000.0, seq_len=None, stream=None, profiling=False, inplace=False):
    """q [tokens, hq, d], k [tokens, hk, d] (views with a token stride are fine).
    positions: int32 [tokens], or None for pos = t % seq_len (t if seq_len is None).
    Returns (q_rot, k_rot, ms)."""
    return _rope(q, k, positions, theta, seq_len, False, stream, profiling, inplace)


def rope_bwd(dq, dk, positions=None, theta=10000.0, seq_len=None, stream=None, profiling=False, inplace=False):
    """Gradient of rope_fwd: the inverse rotation applied to dq, dk."""
    return _rope(dq, dk, positions, theta, seq_len, True, stream, profiling, inplace)


# ---------------------------------------------------------------------------------------
# the general form
# ---------------------------------------------------------------------------------------
_SCALING_KEYS = {"linear": {"factor"}, "ntk": {"factor"},
                 "parts": {"factor", "original_length", "beta_fast", "beta_slow", "attention_factor"},
                 "bands": {"factor", "original_length", "low", "high"}}


def rotary_frequencies(theta: float, dim: int, scaling: Optional[dict] = None):
    """(frequencies of the ``dim / 2`` pairs in radians a position, factor on cos and sin), 64-bit Python floats.

    theta^(-2j / dim), changed by ``scaling`` = {"kind": ..., "factor": s, ...} for contexts s times as long:

    * ``linear``: all divided by s (position interpolation, Chen et al. 2023)
    * ``ntk``: theta multiplied by s^(dim / (dim - 2)), so that the slowest pair is divided by s and the fastest stays (the static
      "NTK-aware" rule)
    * ``parts`` (``original_length``, ``beta_fast`` = 32, ``beta_slow`` = 1, ``attention_factor`` = 0.1 ln s + 1): pairs that turn more
      than ``beta_fast`` times over the original length stay, pairs that turn less than ``beta_slow`` times are divided by s, a line in
      the pair's index between, its ends rounded outwards to pairs; cos and sin are multiplied by the attention factor (YaRN, Peng et al.
      2023; a configuration's "yarn")
    * ``bands`` (``original_length``, ``low`` = 1, ``high`` = 4): wavelengths below original_length / high stay, above original_length / low
      they are divided by s, between them a line in original_length / wavelength (Llama 3.1's rule; a configuration's "llama3", ``low`` and
      ``high`` its low and high frequency factors)
    """
    if not (isinstance(dim, int) and dim >= 2 and dim % 2 == 0):
        raise ValueError(f"rotary: the turned part of a head is an even number of elements, not {dim!r}")
    if not (math.isfinite(theta) and theta > 0):
        raise ValueError(f"rotary: theta must be positive, not {theta!r}")
    f = [float(theta) ** (-2.0 * j / dim) for j in range(dim // 2)]
    if scaling is None:
        return f, 1.0
    kind = scaling.get("kind")
    if kind not in _SCALING_KEYS:
        raise ValueError(f"rotary: unknown scaling {kind!r}, known are {sorted(_SCALING_KEYS)}")
    unknown = set(scaling) - _SCALING_KEYS[kind] - {"kind"}
    if unknown:
        raise ValueError(f"rotary: scaling {kind!r} does not take {sorted(unknown)}")
    s = float(scaling.get("factor", 0.0))
    if not (math.isfinite(s) and s > 0):
        raise ValueError("rotary: scaling needs a positive factor")
    if kind == "linear":
        return [x / s for x in f], 1.0
    if kind == "ntk":
        if dim == 2:                          # one pair, the fastest
            return f, 1.0
        base = float(theta) * s ** (dim / (dim - 2.0))
        return [base ** (-2.0 * j / dim) for j in range(dim // 2)], 1.0
    length = float(scaling.get("original_length", 0))
    if not (math.isfinite(length) and length > 0):
        raise ValueError(f"rotary: scaling {kind!r} needs the original_length")
    if kind == "parts":
        fast, slow = float(scaling.get("beta_fast", 32.0)), float(scaling.get("beta_slow", 1.0))
        if not (0 < slow <= fast) or theta <= 1:
            raise ValueError("rotary: scaling 'parts' needs 0 < beta_slow <= beta_fast and theta above 1")
        # the index of the pair that turns beta times over the original length
        edge = lambda beta: dim * math.log(length / (beta * 2.0 * math.pi)) / (2.0 * math.log(theta))
        lo, hi = math.floor(edge(fast)), math.ceil(edge(slow))
        if hi >= 0 and lo <= dim - 1:         # (a line that ends before the first pair, or begins behind the last, stays where it is)
            lo, hi = max(lo, 0), min(hi, dim - 1)
        span = float(hi - lo) if hi != lo else 0.001
        ramp = [min(max((j - lo) / span, 0.0), 1.0) for j in range(dim // 2)]
        factor = scaling.get("attention_factor")
        return ([x / s * r + x * (1.0 - r) for x, r in zip(f, ramp)],
                float(factor) if factor is not None else 0.1 * math.log(s) + 1.0 if s > 1 else 1.0)
    low, high = float(scaling.get("low", 1.0)), float(scaling.get("high", 4.0))
    if not 0 < low < high:
        raise ValueError("rotary: scaling 'bands' needs 0 < low < high")
    out = []
    for x in f:
        turns = length * x / (2.0 * math.pi)          # original_length / wavelength
        if turns > high:
            out.append(x)
        elif turns < low:
            out.append(x / s)
        else:
            t = (turns - low) / (high - low)
            out.append((1.0 - t) * x / s + t * x)
    return out, 1.0


@dataclass(frozen=True)
class RotaryTable:
    """What ``rotary_fwd`` turns by; made once by ``rotary_table``."""
    steps: torch.Tensor        # int64 [dim / 2]: a position's turn of each pair in units of 2^-64 turns, modulo one turn
    dim: int                   # turned elements at the front of a head
    interleaved: bool          # pairs (2j, 2j + 1); else (j, j + dim / 2)
    factor: float              # on cos and sin


def rotary_table(theta: float, dim: int, device, interleaved: bool = False, scaling: Optional[dict] = None) -> RotaryTable:
    """The table for heads whose first ``dim`` elements are turned (``rotary_frequencies`` says what ``scaling`` takes)."""
    f, factor = rotary_frequencies(theta, dim, scaling)
    steps = []
    for x in f:
        u = round(math.fmod(x / (2.0 * math.pi), 1.0) * 2.0 ** 64) % (1 << 64)
        steps.append(u - (1 << 64) if u >= 1 << 63 else u)
    return RotaryTable(torch.tensor(steps, dtype=torch.int64).to(device), dim, bool(interleaved), factor)


_table_cache: dict = {}


def cached_rotary_table(theta, dim, device, interleaved=False, scaling=None) -> RotaryTable:
    """``rotary_table``, made once for equal arguments (what a layer's configuration holds)."""
    key = (theta, dim, device, interleaved, tuple(sorted(scaling.items())) if scaling is not None else None)
    t = _table_cache.get(key)
    if t is None:
        t = _table_cache[key] = rotary_table(theta, dim, device, interleaved, scaling)
    return t


def _rotary(q, k, table, positions, seq_len, backward, stream, profiling, inplace):
    (qo, ko), ms = issue(_host.rotary, stream, profiling, q, k, table.steps, table.dim, table.interleaved, table.factor, positions,
                         int(seq_len or 0), backward, inplace)
    return (q, k, ms) if inplace else (qo, ko, ms)


def rotary_fwd(q, k, table, positions=None, seq_len=None, stream=None, profiling=False, inplace=False):
    """q [tokens, hq, d], k [tokens, hk, d] or None, any token and head strides, d >= table.dim; the elements behind the turned part
    are passed through (a part that does not start the head is a view: ``rotary_fwd(q[..., at:], k[..., at:], ..., inplace=True)``).
    positions: int32 or int64 [tokens], or None for pos = t % seq_len (t if seq_len is None).  The angle is position times
    frequency with all its whole turns taken off exactly, at any position.  Returns (q_rot, k_rot, ms)."""
    return _rotary(q, k, table, positions, seq_len, False, stream, profiling, inplace)


def rotary_bwd(dq, dk, table, positions=None, seq_len=None, stream=None, profiling=False, inplace=False):
    """Gradient of rotary_fwd: the inverse rotation (times the same factor) applied to dq, dk."""
    return _rotary(dq, dk, table, positions, seq_len, True, stream, profiling, inplace)
