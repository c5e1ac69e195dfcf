"""Frequencies and tables of the general rotary positions (no GPU)."""
import math
from decimal import Decimal, getcontext

import pytest
import torch

from dhellam_amd.operators.rope import rotary_frequencies, rotary_table

PI = Decimal("3.14159265358979323846264338327950288419716939937510582097494459")


def test_a_table_holds_the_turns_of_a_position():
    """A step is theta^(-2j / dim) / (2 pi) turns: 2^-53 of it from the 64-bit power and two more roundings."""
    getcontext().prec = 50
    theta, dim = 500000.0, 128
    t = rotary_table(theta, dim, "cpu")
    assert t.steps.dtype == torch.int64 and t.steps.shape == (dim // 2,) and not t.interleaved and t.factor == 1.0
    for j, u in enumerate(t.steps.tolist()):
        want = (Decimal(theta).ln() * (Decimal(-2 * j) / Decimal(dim))).exp() / (2 * PI)
        assert abs(Decimal(u) / 2 ** 64 - want) <= want * Decimal(2.0 ** -50) + Decimal(2.0 ** -64)


def test_steps_past_half_a_turn_are_negative_numbers():
    t = rotary_table(10000.0, 4, "cpu", scaling={"kind": "linear", "factor": 0.25})      # 4 radians a position
    assert t.steps[0].item() < 0
    assert abs(t.steps[0].item() % 2 ** 64 / 2 ** 64 - 4 / (2 * math.pi)) < 1e-15


@pytest.mark.parametrize("dim", [2, 20, 64, 128])
def test_scaled_frequencies(dim):
    theta, s = 10000.0, 8.0
    plain, one = rotary_frequencies(theta, dim)
    assert one == 1.0 and plain[0] == 1.0 and len(plain) == dim // 2
    assert rotary_frequencies(theta, dim, {"kind": "linear", "factor": s})[0] == [x / s for x in plain]
    ntk, _ = rotary_frequencies(theta, dim, {"kind": "ntk", "factor": s})
    assert ntk[0] == 1.0
    if dim > 2:
        assert math.isclose(ntk[-1], plain[-1] / s, rel_tol=1e-12)                        # the slowest pair is interpolated, the fastest stays
    length = 4096
    bands, one = rotary_frequencies(theta, dim, {"kind": "bands", "factor": s, "original_length": length})
    parts, m = rotary_frequencies(theta, dim, {"kind": "parts", "factor": s, "original_length": length})
    assert one == 1.0 and math.isclose(m, 0.1 * math.log(s) + 1)
    for got in (bands, parts):
        assert all(x / s * (1 - 1e-12) <= y <= x * (1 + 1e-12) for x, y in zip(plain, got))
        ratio = [y / x for x, y in zip(plain, got)]
        assert ratio == sorted(ratio, reverse=True) or all(a >= b - 1e-12 for a, b in zip(ratio, ratio[1:]))
    for x, y in zip(plain, bands):
        turns = length * x / (2 * math.pi)
        if turns > 4:
            assert y == x
        if turns < 1:
            assert y == x / s
    for x, y in zip(plain, parts):                      # a pair's index is rounded outwards: two more pairs on either side of the line
        step = theta ** (2.0 / dim)
        if length * x / (2 * math.pi) > 32 * step ** 2:
            assert math.isclose(y, x, rel_tol=1e-12)
        if length * x / (2 * math.pi) < step ** -2:
            assert math.isclose(y, x / s, rel_tol=1e-12)
    assert rotary_frequencies(theta, dim, {"kind": "parts", "factor": s, "original_length": length, "attention_factor": 1.5})[1] == 1.5


@pytest.mark.parametrize("args", [
    (10000.0, 3), (10000.0, 0), (10000.0, 2.0), (0.0, 4), (math.nan, 4), (10000.0, 4, {}), (10000.0, 4, {"kind": "other", "factor": 2.0}),
    (10000.0, 4, {"kind": "linear"}), (10000.0, 4, {"kind": "linear", "factor": -1.0}), (10000.0, 4, {"kind": "linear", "factor": 2.0, "low": 1}),
    (10000.0, 4, {"kind": "bands", "factor": 2.0}), (10000.0, 4, {"kind": "bands", "factor": 2.0, "original_length": 64, "low": 4.0, "high": 4.0}),
    (10000.0, 4, {"kind": "parts", "factor": 2.0, "original_length": 64, "beta_fast": 1.0, "beta_slow": 2.0}),
    (1.0, 4, {"kind": "parts", "factor": 2.0, "original_length": 64})])
def test_refused_frequencies(args):
    with pytest.raises(ValueError):
        rotary_frequencies(*args)


@pytest.mark.parametrize("dim", [0, -2, 7])
def test_a_layer_whose_turned_part_is_no_part_of_a_head_is_refused(dim):
    """0 is not "all": a share of the head that was rounded to nothing is an error of the configuration."""
    from dhellam_amd.core.dstb import LayerConfig, _turn
    cfg = LayerConfig(hidden_size=256, num_attention_heads=4, num_query_groups=4, ffn_hidden_size=192, seq_length=64, rotary_dim=dim)
    assert cfg.general_rotary
    with pytest.raises(ValueError, match="even number"):
        _turn(cfg, torch.zeros(64, 4, 64), torch.zeros(64, 4, 64), None, None)


@pytest.mark.parametrize("theta,dim,length", [(10.0, 64, 100000), (10.0, 2, 1 << 20), (10000.0, 64, 4), (10000.0, 128, 0.5), (10.0, 64, 1), (2.0, 8, 300)])
def test_parts_whose_line_lies_outside_the_pairs(theta, dim, length):
    """All pairs turn more than 32 times over the original length and stay, or all less than once and are divided (the line's end is
    rounded up to a pair: one that turns theta^(-2 / dim) of once may stay); nothing in between turns round."""
    s = 8.0
    plain, _ = rotary_frequencies(theta, dim)
    got, _ = rotary_frequencies(theta, dim, {"kind": "parts", "factor": s, "original_length": length})
    step = theta ** (2.0 / dim)
    seen = set()
    for x, y in zip(plain, got):
        turns = length * x / (2 * math.pi)
        if turns > 32:
            assert math.isclose(y, x, rel_tol=1e-12)
            seen.add("stays")
        elif turns < 1 / step:
            assert math.isclose(y, x / s, rel_tol=1e-12)
            seen.add("divided")
        else:
            assert x / s * (1 - 1e-12) <= y <= x * (1 + 1e-12)
    assert seen
