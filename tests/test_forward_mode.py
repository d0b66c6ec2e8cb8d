"""Forward-mode differentiation: the operators have no rule for it, and say so."""

import pytest
import torch
from torch.autograd import forward_ad

import keep_amd
from keep_amd import _grad


def test_a_tangent_counts_as_a_gradient_asked_for():
    x = torch.ones(3)
    assert not _grad.wanted(x, None)
    with forward_ad.dual_level():
        d = forward_ad.make_dual(x, torch.ones(3))
        assert _grad.wanted(None, d) and not _grad.wanted(x)
        with torch.no_grad():
            assert _grad.wanted(d)
    assert not _grad.wanted(x)


@pytest.mark.gpu
@pytest.mark.parametrize("which", ["x", "w", "a", "base", "scales", "y", "weight", "routed", "residual"])
def test_tangents_are_refused(dev, which):
    """There is no forward-mode rule: an operator says so, and does not drop the tangent."""
    t = {"x": torch.randn(4, 16, device=dev), "w": torch.randn(3, 8, 16, device=dev), "a": torch.randn(3, 2, 16, device=dev),
         "b": torch.randn(3, 8, 2, device=dev), "base": torch.randn(4, 8, device=dev), "scales": torch.rand(3, device=dev),
         "y": torch.randn(4, 2, 8, device=dev), "weight": torch.rand(4, 2, device=dev),
         "routed": torch.randn(4, 8, device=dev), "residual": torch.randn(4, 8, device=dev)}
    idx = torch.tensor([[0, 1], [1, 2], [2, 0], [1, 1]], device=dev)
    calls = {"x": [lambda: keep_amd.gather_mm(t["x"], t["w"], idx),
                   lambda: keep_amd.gather_lora(t["x"], t["a"], t["b"], idx[:, 0], base=t["base"], scales=t["scales"])],
             "y": [lambda: keep_amd.route_combine(t["y"], t["weight"])],
             "routed": [lambda: keep_amd.combine_add(t["routed"], None, t["residual"])]}
    calls["w"] = calls["x"][:1]
    calls["a"] = calls["base"] = calls["scales"] = calls["x"][1:]
    calls["weight"], calls["residual"] = calls["y"], calls["routed"]
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        for call in calls[which]:
            with pytest.raises((NotImplementedError, ValueError)):
                call()
            with torch.no_grad(), pytest.raises((NotImplementedError, ValueError)):
                call()
