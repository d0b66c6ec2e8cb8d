"""Gradients of adapters whose output is float32 over 16-bit rows."""

import pytest
import torch

import keep_amd
from tests import test_gpu_lora as lora

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", [(1, 0, 2, 16, 64, 48), (50, 0, 3, 16, 64, 80), (9, 0, 2, 5, 33, 17),
                                   (300, 2, 6, 8, 72, 40)])
@pytest.mark.parametrize("size", [1.0, 2.0 ** 40, 2.0 ** -40])
def test_gradients_of_a_float_output_keep_their_bits(dev, monkeypatch, dtype, shape, size):
    """A loss's scale beyond 16 bits, and values between two 16-bit ones: float32 gradients enter the products whole."""
    monkeypatch.setattr(lora, "_low", lambda t, _: t)  # float32 rows throughout
    c = lora._case(dev, dtype, *shape, seed=7)
    c["base"] = c["base"].float()
    g = torch.Generator(device=dev).manual_seed(8)
    c["dy"] = torch.randn(c["dy"].shape, device=dev, generator=g) * size
    c["scales"] = c["scales"] / size  # brings dx and dA back; dB = dy^T t has them cancel in t
    want = lora._expected(c)
    leaves = [c[n].requires_grad_(True) for n in ("x", "a", "b", "base")]
    dx, da, db, dbase = torch.autograd.grad(lora._call(c), leaves, c["dy"])
    assert torch.equal(dbase, c["dy"])
    for got, w, name in zip((dx, da, db), want[1:], ("dx", "da", "db")):
        assert got.dtype == dtype
        w.check(got, name)


def test_gradients_of_a_float_output_in_a_graph(dev):
    cases = [lora._case(dev, torch.bfloat16, 300, 2, 5, 16, 64, 48, seed=s) for s in range(3)]
    for o in cases:
        o["base"], o["dy"] = o["base"].float(), o["dy"].float() * 1.001
    names = ("x", "a", "b", "idx", "base", "scales", "dy")
    c = {n: cases[0][n].clone() for n in names}

    def step():
        leaf = {n: c[n].detach().requires_grad_(True) for n in ("x", "a", "b")}
        out = lora._call({**c, **leaf})
        return [out.detach(), *torch.autograd.grad(out, list(leaf.values()), c["dy"])]

    lora._replays(step, [c[n] for n in names], [[o[n] for n in names] for o in cases])


def test_a_float_output_and_no_adapter(dev):
    """Rows without an adapter take no part, whatever the gradient holds there."""
    c = lora._case(dev, torch.float16, 20, 0, 2, 8, 64, 48, seed=9)
    c["idx"][4] = -1
    x = c["x"].clone().requires_grad_(True)
    dy = c["dy"].float()
    dy[4] = float("inf")
    dx = torch.autograd.grad(keep_amd.gather_lora(x, c["a"], c["b"], c["idx"], base=c["base"].float()), x, dy)[0]
    assert (dx[4] == 0).all() and torch.isfinite(dx).all()
