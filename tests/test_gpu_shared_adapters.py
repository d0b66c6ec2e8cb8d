"""Adapters of a layer's shared expert, beside those of its routed experts or alone."""

import pytest
import torch

import keep_amd

pytestmark = pytest.mark.gpu
E, H, I, N, R = 4, 512, 256, 3, 8


def _glu(dev, experts, seed, kind, adapters):
    import numpy as np
    from keep_amd import synth
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*s, std):
        return (torch.randn(*s, device=dev, generator=g) * std).half()

    def one(n, m, s):
        ad = keep_amd.LoraAdapters(normal(N, experts, R, m, std=m ** -0.5), normal(N, experts, n, R, std=0.5)) \
            if adapters else None
        if kind == "dense":
            return keep_amd.SwitchLinear(normal(experts, n, m, std=m ** -0.5), adapters=ad)
        c, sc = synth.projection_np(experts, n, m, seed=s)[:2]
        return keep_amd.QuantizedVQSwitchLinear(
            input_dims=m, output_dims=n, num_experts=experts, codes=torch.from_numpy(c.view(np.int16)).to(dev),
            scales=torch.from_numpy(sc).to(dev), group_size=m // sc.shape[-1], code_bits=16, adapters=ad)
    return keep_amd.QuantizedVQSwitchGLU(gate_proj=one(I, H, seed), up_proj=one(I, H, seed + 1),
                                         down_proj=one(H, I, seed + 2))


@pytest.mark.parametrize("T", [1, 3, 90])
@pytest.mark.parametrize("kind", ["dense", "codes"])
@pytest.mark.parametrize("routed", [False, True])
def test_a_shared_experts_adapters_are_added(dev, T, kind, routed):
    glu, shared = _glu(dev, E, 1, kind, routed), _glu(dev, 1, 7, kind, True)
    moe = keep_amd.RoutedVQMoE(glu, top_k=2, shared_experts=shared)
    g = torch.Generator(device=dev).manual_seed(T)
    x = (torch.randn(T, H, device=dev, generator=g) * 0.1).half()
    logits = torch.randn(T, E, device=dev, generator=g)
    ad = torch.randint(-1, N, (T,), device=dev, generator=g)
    ad[0] = 1
    out, r = moe(x, logits, adapter_indices=ad)
    idx = torch.zeros(T, 1, dtype=torch.int32, device=dev)
    own = shared(x, idx, ad).reshape(T, H).float()
    part = moe.experts(x, r.idx, r.weight, out_dtype=torch.float32, adapter_indices=ad if routed else None)
    assert torch.equal(out, keep_amd.combine_add(part, own, None, torch.float32))
    assert not torch.equal(own[0], moe.shared(x)[0])
    # a token without an adapter: the layer's own output, up to the kernels that serve it without adapters
    plain, _ = moe(x, logits)
    if kind == "dense":
        assert torch.equal(out[ad < 0], plain[ad < 0])


def test_no_adapters_anywhere(dev):
    moe = keep_amd.RoutedVQMoE(_glu(dev, E, 1, "dense", False), top_k=2, shared_experts=_glu(dev, 1, 7, "dense", False))
    with pytest.raises(ValueError, match="projection with adapters"):
        moe(torch.zeros(2, H, device=dev).half(), torch.zeros(2, E, device=dev), adapter_indices=[0, 1])
