"""Layers on dense experts and adapters, captured and replayed on changing inputs."""

import pytest
import torch

import keep_amd
from tests.test_gpu_dense import _replays

pytestmark = pytest.mark.gpu


def _normal(dev, g, *s, std=1.0):
    return torch.randn(*s, device=dev, generator=g) * std


@pytest.mark.parametrize("T", [3, 200])
def test_switch_linear_with_a_bias(dev, T):
    """Forward and every gradient, routes without an expert among them."""
    def inputs(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        idx = torch.randint(-1, 6, (T, 2), device=dev, generator=g, dtype=torch.int32)
        idx[0] = 0
        return [_normal(dev, g, T, 64), _normal(dev, g, 5, 48, 64), _normal(dev, g, 5, 48), idx,
                _normal(dev, g, T, 2, 48)]
    x, w, b, idx, dy = buffers = inputs(0)

    def step():
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        out = keep_amd.SwitchLinear(leaves[1], leaves[2])(leaves[0], idx)
        grads = torch.autograd.grad(out, leaves, dy)
        return [t.detach().nan_to_num(7.0) for t in (out, *grads)]

    _replays(step, buffers, [inputs(s) for s in range(1, 5)])


@pytest.mark.parametrize("T", [1, 5, 200])
def test_adapters_of_routed_experts_in_the_layer(dev, T):
    E, H, I, n, r = 4, 64, 48, 3, 8

    def inputs(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        return [_normal(dev, g, T, H), _normal(dev, g, T, E),
                torch.randint(-1, n, (T,), device=dev, generator=g, dtype=torch.int32),
                _normal(dev, g, E, I, H, std=0.125), _normal(dev, g, E, H, I, std=0.14),
                _normal(dev, g, n, E, r, H, std=0.1), _normal(dev, g, n, E, I, r, std=0.3)]
    x, logits, ad, wi, wo, a, b = buffers = inputs(0)
    scales = torch.rand(n, device=dev)

    def step():
        fa, fb = a.detach().requires_grad_(True), b.detach().requires_grad_(True)
        glu = keep_amd.QuantizedVQSwitchGLU(
            gate_proj=keep_amd.SwitchLinear(wi, adapters=keep_amd.LoraAdapters(fa, fb, scales)),
            up_proj=keep_amd.SwitchLinear(wi), down_proj=keep_amd.SwitchLinear(wo))
        out = keep_amd.RoutedVQMoE(glu, top_k=2)(x, logits, adapter_indices=ad)[0]
        return [out.detach(), *torch.autograd.grad(out, (fa, fb), x)]

    _replays(step, buffers, [inputs(s) for s in range(1, 5)])
