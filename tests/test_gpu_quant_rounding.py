"""``rmsnorm_quant``'s codes are the rounded quotients of the normed values and their scale: values one float32 step about the
middles between two codes."""

import numpy as np
import pytest
import torch

import keep_amd

pytestmark = pytest.mark.gpu


def _middles():
    codes = torch.arange(0, 127, dtype=torch.uint8).view(torch.float8_e4m3fn).double()
    return ((codes[1:] + codes[:-1]) / 2).numpy()


@pytest.mark.parametrize("pow2", [False, True])
def test_codes_beside_the_middles(dev, pow2):
    """Rows of +-1 have a mean square of 1 and r = 1: the normed values are the weight, to the bit."""
    rng = np.random.default_rng(0)
    n, block = 16384, 128
    tops = rng.uniform(0.5, 400.0, n // block).astype(np.float32)
    w = np.empty((n // block, block), np.float32)
    for b, top in enumerate(tops):
        s = np.float32(top / np.float32(448))
        near = (rng.choice(_middles(), block) * np.float64(s)).astype(np.float32)
        near = np.nextafter(near, np.where(rng.random(block) < 0.5, np.float32(np.inf), np.float32(0)), dtype=np.float32)
        w[b] = np.where(rng.random(block) < 0.3, near, np.nextafter(near, np.float32(0), dtype=np.float32))
        w[b] = np.minimum(w[b], top)
        w[b, 0] = top
    w *= rng.choice(np.float32([-1, 1]), w.shape)
    weight = torch.from_numpy(w.reshape(-1))
    x = torch.where(torch.rand(3, n, generator=torch.Generator().manual_seed(1)) < 0.5, 1.0, -1.0)
    q, scales = keep_amd.rmsnorm_quant(x.to(dev), weight.to(dev), 0.0, quant_block=block, pow2_scales=pow2)
    y = x * weight
    s = y.view(3, -1, block).abs().amax(2) / np.float32(448)
    if pow2:
        s = torch.exp2(torch.ceil(torch.log2(s.double()))).float()
    assert torch.equal(scales.cpu(), s)
    want = (y.view(3, -1, block) / s[..., None]).clamp(-448, 448).view(3, n).to(torch.float8_e4m3fn)
    assert torch.equal(q.cpu().view(torch.uint8), want.view(torch.uint8))


def test_infinite_and_nan_rows(dev):
    x = torch.ones(3, 64, device=dev)
    w = torch.linspace(1, 2, 64, device=dev)
    w[5], w[40] = float("inf"), float("nan")
    q, s = keep_amd.rmsnorm_quant(x, w, 0.0, quant_block=16)
    q, s = q.float().cpu(), s.cpu()
    assert (s[:, 0] == float("inf")).all() and s[:, 2].isnan().all() and torch.isfinite(s[:, [1, 3]]).all()
    assert q[:, 5].isnan().all() and (q[:, [0, 1, 2, 15]] == 0).all()  # finite values beside an infinite one
    assert q[:, 32:48].isnan().all() and torch.isfinite(q[:, 16:32]).all() and torch.isfinite(q[:, 48:]).all()
