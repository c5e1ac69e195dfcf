"""Clipping by norms and factors at the ends of fp32's range."""
import math

import pytest
import torch

from dhellam_amd.operators.grads import clip_grads, grad_norm

pytestmark = pytest.mark.gpu


def grads(dtype, size):
    g = torch.Generator(device="cuda").manual_seed(5)
    return [(torch.rand(n, generator=g, device="cuda") * size).to(dtype) for n in (33001, 7)]


def close(out, g, factor):
    """The factor is rounded to 24 bits, the product to 24 bits, the result to its type."""
    half = torch.finfo(out.dtype).eps / 2
    want = g.double() * factor
    tiny = torch.finfo(out.dtype).smallest_normal * 2 * half
    assert ((out.double() - want).abs() <= (half + 2.0 ** -23) * (1 + half) * want.abs() + tiny).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_a_norm_past_fp32_counts_as_not_finite(dtype):
    """Every gradient is finite and so is their norm in 64 bits, but not what is reported of it: the factor agrees with that."""
    gs = grads(dtype, 3e38)
    sum_sq, _ = grad_norm(gs)
    assert 3.5e38 < math.sqrt(sum_sq.item()) < math.inf
    for max_norm, scale in ((1.0, 1.0), (math.inf, 1.0)):
        into = [torch.full_like(g, 7.0, dtype=torch.float32) for g in gs]
        found, _ = clip_grads(gs, sum_sq, max_norm, scale, out=into)
        assert found.tolist() == [math.inf, 0.0] and all((o == 0).all() for o in into)
    # a scale that brings the norm back into fp32's range
    found, _ = clip_grads(gs, sum_sq, math.inf, 0.0009765625, out=into)
    assert math.isfinite(found[0].item()) and found[1].item() == 0.0009765625
    for o, g in zip(into, gs):
        close(o, g, 0.0009765625)
    clip_grads(gs, sum_sq, 1.0)
    assert all((g == 0).all() for g in gs)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("max_norm,scale", [(1.0, 1.0), (1e-3, 1.0), (2e-6, 1.0), (math.inf, 1e-39), (math.inf, -3e-43), (1e-3, 0.5)])
def test_a_factor_below_the_normal_numbers(dtype, max_norm, scale):
    gs = grads(dtype, 1e36)
    sum_sq, _ = grad_norm(gs)
    norm = abs(scale) * math.sqrt(sum(float(g.double().square().sum()) for g in gs))
    factor = scale * min(1.0, max_norm / (norm + 1e-6))
    for kind in (torch.float32, dtype):
        into = [torch.full_like(g, 7.0, dtype=kind) for g in gs]
        found, _ = clip_grads(gs, sum_sq, max_norm, scale, out=into)
        assert abs(found[0].item() - norm) <= 2.0 ** -23 * norm and abs(found[1].item() - factor) <= 2.0 ** -23 * abs(factor) + 2.0 ** -150
        assert found[1].item() != 0
        for o, g in zip(into, gs):
            close(o, g, factor)


def test_a_factor_below_every_number():
    gs = grads(torch.float32, 1e36)
    into = [torch.full_like(g, 7.0) for g in gs]
    found, _ = clip_grads(gs, grad_norm(gs)[0], 1e-9, out=into)
    assert found[1].item() == 0 and all((o == 0).all() for o in into)
