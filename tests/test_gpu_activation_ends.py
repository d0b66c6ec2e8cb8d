"""Gradients of activations whose kept values have passed their type's largest."""

import pytest
import torch

import keep_amd

pytestmark = pytest.mark.gpu
F32, F16 = torch.float32, torch.float16


@pytest.mark.parametrize("act", ["relu", "silu", "gelu", "gelu_tanh"])
def test_float_output_whose_kept_values_pass_float16(dev, act):
    """u is kept in float16 for the gradient; past its largest value the slopes are 1 and 0."""
    for M in (3, 40):
        x = torch.full((M, 8), 100.0, device=dev, dtype=F16)
        x[1::2] = -100.0
        w = torch.full((8, 8), 100.0, device=dev, dtype=F16)  # u = +-80000
        leaves = [x.requires_grad_(True), w.requires_grad_(True)]
        out = keep_amd.linear(*leaves, activation=act, out_dtype=F32)
        assert torch.equal(out[0], torch.full((8,), 80000.0, device=dev)) and (out[1] == 0).all()
        dx, dw = torch.autograd.grad(out, leaves, torch.ones_like(out))
        assert (dx[0::2] == 800.0).all() and (dx[1::2] == 0).all()
        assert (dw == 100.0 * ((M + 1) // 2)).all()


def test_infinite_values_before_the_activation(dev):
    """Slopes of +inf and -inf are 1 and 0, of NaN NaN."""
    x = torch.tensor([[float("inf")], [-float("inf")], [float("nan")], [1.0]], device=dev)
    one = torch.ones(1, 1, device=dev)
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        leaf = x.clone().requires_grad_(True)
        y = keep_amd.linear(leaf, one, activation=act)
        slope, = torch.autograd.grad(y, leaf, torch.ones_like(y))
        assert slope[0] == 1 and slope[1] == 0 and slope[2].isnan() and slope[3] > 0
