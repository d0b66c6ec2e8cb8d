"""Gradients where a score has reached its end."""

import pytest
import torch

import keep_amd

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("renormalize", [False, True])
def test_slope_of_saturated_sigmoid_scores(dev, renormalize):
    """s (1 - s) keeps its bits where s rounds to 1: each factor within 2^-20 of itself (exp, a sum, a reciprocal), the
    weights' gradient as without saturation."""
    z = torch.linspace(8, 40, 64, device=dev).view(8, 8).requires_grad_(True)
    dw = torch.randn(8, 3, device=dev, generator=torch.Generator(device=dev).manual_seed(0))
    r = keep_amd.route_experts(z, 3, score_func="sigmoid", renormalize=renormalize)
    got, = torch.autograd.grad(r.weight, z, dw)
    at = r.idx.long()
    zc, g = z.detach().double().gather(1, at), dw.double()
    s, rest = 1 / (1 + torch.exp(-zc)), 1 / (1 + torch.exp(zc))
    p, size = g, g.abs()
    if renormalize:
        total = s.sum(1, keepdim=True)
        p = (g - (g * s).sum(1, keepdim=True) / total) / total
        size = (g.abs() + (g.abs() * s).sum(1, keepdim=True) / total) / total
    want = torch.zeros_like(z, dtype=torch.float64).scatter_(1, at, p * s * rest)
    bound = torch.zeros_like(want).scatter_(1, at, size * s * rest * 2.0 ** -17)
    assert ((got.double() - want).abs() <= bound).all()
