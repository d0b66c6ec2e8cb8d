"""Bias gradients of dense expert layers."""

import pytest
import torch


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_routes_without_an_expert_give_no_bias_gradient(monkeypatch, dtype):
    """On the CPU, the product in torch."""
    from keep_amd import nn

    def product(x, w, idx):
        y = torch.einsum("tk,tjnk->tjn", x.float(), w[idx.long().clamp(0, 2)].float()).to(x.dtype)
        return torch.where(((idx >= 0) & (idx < 3))[..., None], y, float("nan"))
    monkeypatch.setattr(nn, "gather_mm", product)
    g = torch.Generator().manual_seed(0)
    x = torch.randint(-4, 5, (5, 8), generator=g).to(dtype)
    w = torch.randint(-2, 3, (3, 6, 8), generator=g).to(dtype)
    bias = torch.randint(-2, 3, (3, 6), generator=g).to(dtype).requires_grad_(True)
    idx = torch.tensor([[0, 1], [-1, 2], [3, 0], [-2 ** 31, 2 ** 31 - 1], [2, 2]])
    dy = torch.randint(-3, 4, (5, 2, 6), generator=g).to(dtype)  # whole numbers: exact sums
    y = nn.SwitchLinear(w, bias)(x, idx)
    valid = (idx >= 0) & (idx < 3)
    assert torch.isnan(y[~valid]).all()
    assert torch.equal(y[valid], product(x, w, idx)[valid] + bias.detach()[idx[valid]])
    want = torch.zeros(3, 6, dtype=torch.float64).index_add_(0, idx[valid], dy[valid].double())
    assert torch.equal(torch.autograd.grad(y, bias, dy)[0].double(), want)
