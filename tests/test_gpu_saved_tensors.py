"""Backward passes on saved tensors that a hook gives back in another layout than it took them (offloading, compression): the
gradients of the plain call, to the bit."""

import pytest
import torch

import keep_amd

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _spread(t):
    """The same values, every second one of a larger tensor of NaN (whole numbers: of -1)."""
    if t.ndim == 0 or t.numel() == 0:
        return t
    big = torch.full((*t.shape, 2), float("nan") if t.is_floating_point() else -1, dtype=t.dtype, device=t.device)
    big[..., 0] = t
    return big[..., 0]


def _pitched(t):
    """The same values in rows that lie further apart, behind an odd start."""
    if t.ndim == 0 or t.numel() == 0:
        return t
    big = torch.full((*t.shape[:-1], t.shape[-1] + 24), float("nan") if t.is_floating_point() else -1, dtype=t.dtype,
                     device=t.device)
    big[..., 1:t.shape[-1] + 1] = t
    return big[..., 1:t.shape[-1] + 1]


HOOKS = {
    "offloaded": lambda: torch.autograd.graph.save_on_cpu(),
    "offloaded to pinned memory": lambda: torch.autograd.graph.save_on_cpu(pin_memory=True),
    "spread": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), _spread),
    "pitched": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.clone(), _pitched),
    "compact": lambda: torch.autograd.graph.saved_tensors_hooks(lambda t: t.contiguous().clone(), lambda t: t),
}


def _both(call, leaves, douts):
    """The gradients of ``call`` as it is, and under each hook."""
    outs = call()
    want = torch.autograd.grad(outs, leaves, douts)
    for name, hook in HOOKS.items():
        with hook():
            outs = call()
        torch.cuda.synchronize()
        for g, w in zip(torch.autograd.grad(outs, leaves, douts), want):
            assert torch.equal(g, w), name
    assert all(torch.isfinite(w).all() for w in want)


def _normal(dev, *shape, dtype=F32, seed=0):
    return torch.randn(*shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("M, N, K", [(20, 33, 10), (5, 16, 17), (300, 72, 333), (40, 24, 96)])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("act", [None, "silu"])
def test_linear(dev, M, N, K, dtype, act):
    x, w = _normal(dev, M, K, dtype=dtype), _normal(dev, N, K, dtype=dtype, seed=1)
    wide_x, wide_w = (torch.full((len(t), K + 30), float("nan"), device=dev, dtype=dtype) for t in (x, w))
    piece = 16 // x.element_size()
    wide_x[:, piece:piece + K], wide_w[:, :K] = x, w
    for x, w in ((x, w), (wide_x[:, piece:piece + K], w), (x, wide_w[:, :K])):
        leaves = [x.detach().requires_grad_(True), w.detach().requires_grad_(True),
                  _normal(dev, N, seed=2).requires_grad_(True)]
        for od in {dtype, F32}:
            _both(lambda: keep_amd.linear(*leaves, activation=act, out_dtype=od), leaves,
                  _normal(dev, M, N, dtype=od, seed=3))


@pytest.mark.parametrize("n", [7, 96, 333])
def test_rmsnorm(dev, n):
    leaves = [_normal(dev, 9, n, dtype=BF16).requires_grad_(True), _normal(dev, n, seed=1).requires_grad_(True),
              _normal(dev, 9, n, dtype=BF16, seed=2).requires_grad_(True)]
    douts = [_normal(dev, 9, n, dtype=BF16, seed=3), _normal(dev, 9, n, dtype=BF16, seed=4)]
    _both(lambda: keep_amd.rmsnorm(leaves[0], leaves[1], residual=leaves[2]), leaves, douts)
    _both(lambda: keep_amd.rmsnorm(*leaves[:2]), leaves[:2], douts[0])


def test_route_experts(dev):
    z = _normal(dev, 11, 40).requires_grad_(True)
    _both(lambda: keep_amd.route_experts(z, 3).weight, [z], _normal(dev, 11, 3, seed=1))


def test_routed_products_and_their_combine(dev):
    x, w = _normal(dev, 13, 72, dtype=BF16).requires_grad_(True), _normal(dev, 5, 40, 72, dtype=BF16, seed=1).requires_grad_(True)
    idx = torch.randint(0, 5, (13, 2), device=dev, dtype=torch.int32, generator=torch.Generator(device=dev).manual_seed(2))
    weight = _normal(dev, 13, 2, seed=3).requires_grad_(True)
    _both(lambda: keep_amd.gather_mm(x, w, idx), [x, w], _normal(dev, 13, 2, 40, dtype=BF16, seed=4))
    y = _normal(dev, 13, 2, 40, dtype=BF16, seed=5).requires_grad_(True)
    _both(lambda: keep_amd.route_combine(y, weight), [y, weight], _normal(dev, 13, 40, seed=6))


def test_adapters(dev):
    x = _normal(dev, 13, 72, dtype=BF16).requires_grad_(True)
    a, b = (_normal(dev, *s, dtype=BF16, seed=i).requires_grad_(True) for i, s in enumerate([(3, 8, 72), (3, 40, 8)], 1))
    idx = torch.tensor([0, 2, -1, 1, 1, 0, 2, 2, 2, -1, 0, 1, 1], device=dev)
    _both(lambda: keep_amd.gather_lora(x, a, b, idx), [x, a, b], _normal(dev, 13, 40, dtype=BF16, seed=6))
