"""Scales of adapters beside routed experts."""

import pytest
import torch

import keep_amd


def test_scales_of_routed_adapters_take_no_gradient():
    """As those of a dense projection's: refused, where the layer's own copy would leave them out."""
    ad = keep_amd.LoraAdapters(torch.zeros(2, 3, 4, 16), torch.zeros(2, 3, 8, 4), torch.ones(2, requires_grad=True))
    with pytest.raises(ValueError, match="scales take no gradient"):
        ad.add(torch.zeros(2, 1, 8), torch.zeros(2, 16), torch.zeros(2, dtype=torch.int32),
               torch.zeros(2, 1, dtype=torch.int32))
