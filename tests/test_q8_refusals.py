"""8-bit operands that require a gradient are refused, on the CPU: before any launch."""

import pytest
import torch

import keep_amd
from keep_amd import _lib, ops


@pytest.mark.parametrize("leaf", ["x", "weight"])
def test_operands_that_require_a_gradient(monkeypatch, leaf):
    monkeypatch.setattr(ops, "_dense_device", lambda *ts: torch.device("cpu"))
    monkeypatch.setattr(_lib, "call", lambda name, *a: pytest.fail(f"{name} was launched"))
    args = {"x": torch.zeros(2, 16).to(torch.float8_e4m3fn), "weight": torch.zeros(8, 16).to(torch.float8_e4m3fn)}
    args[leaf].requires_grad_(True)
    with pytest.raises(ValueError, match="no gradients"):
        keep_amd.linear_q8(args["x"], torch.zeros(2, 1), args["weight"], torch.zeros(1, 1))
