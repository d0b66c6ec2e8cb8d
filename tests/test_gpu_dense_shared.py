"""A dense shared expert's sums enter the layer's combine in float32 where nothing is recorded."""

import pytest
import torch

import keep_amd
from tests.bounded import Bounded

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("T", [1, 5, 70])
@pytest.mark.parametrize("dtype", [BF16, F16])
@pytest.mark.parametrize("limit", [0.0, 1.5])
def test_rounded_once(dev, T, dtype, limit):
    g = torch.Generator(device=dev).manual_seed(T)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(dtype)
    E, H, I, k = 4, 96, 48, 2
    up, down = keep_amd.SwitchLinear(normal(E, I, H, std=H ** -0.5)), keep_amd.SwitchLinear(normal(E, H, I, std=I ** -0.5))
    glu = keep_amd.QuantizedVQSwitchGLU(gate_proj=up, up_proj=up, down_proj=down)
    w = [normal(I, H, std=H ** -0.5), normal(I, H, std=H ** -0.5), normal(H, I, std=I ** -0.5)]
    shared = keep_amd.DenseGLU(**{n: keep_amd.DenseLinear(t) for n, t in zip(("gate_proj", "up_proj", "down_proj"), w)})
    moe = keep_amd.RoutedVQMoE(glu, top_k=k, shared_experts=shared, swiglu_limit=limit, out_dtype=F32)
    x, z, res = normal(T, H), torch.randn(T, E, device=dev, generator=g), torch.randn(T, H, device=dev, generator=g)
    if limit:
        hidden = keep_amd.LimitedSwiGLU(limit)(keep_amd.linear(x, w[1]), keep_amd.linear(x, w[0]))
    else:
        hidden = keep_amd.linear(x, w[0], activation="silu") * keep_amd.linear(x, w[1])
    want = Bounded(hidden) @ Bounded(w[2]).T  # float32 sums of the hidden rows as they are held
    sh = moe.shared(x)
    assert sh.dtype == F32
    want.check(sh)
    out, r = moe(x, z, residual=res)
    routed = moe.experts(x, r.idx, r.weight, out_dtype=F32)
    (Bounded(res) + (Bounded(routed) + want)).round(F32).check(out)
    # recorded: the same within the weights' dtype, with gradients
    leaf = w[2].clone().requires_grad_(True)
    shared.down_proj.weight = leaf
    trained = moe.shared(x)
    want.round(dtype).check(trained.detach())
    assert torch.autograd.grad(trained.sum(), leaf)[0].shape == leaf.shape
    with torch.no_grad():
        want.check(moe.shared(x))
