"""How many bits the adapters hold between their products."""

import pytest
import torch

from tests import test_gpu_lora as lora
from tests.bounded import Bounded

pytestmark = pytest.mark.gpu


def _held(t, dtype):
    """The low-rank rows as the sum of 16-bit terms of a row scaled to [1, 4): three bf16 terms are off by at most
    (2^-8)^3 of a value, two of fp16 by (2^-11)^2 and half of its smallest subnormal, 2^-25 of the row's largest."""
    if dtype == torch.float32:
        return t
    mag = t.v.abs() + t.e
    off = 2.0 ** -24 * mag if dtype == torch.bfloat16 else 2.0 ** -22 * mag + 2.0 ** -25 * mag.amax(-1, keepdim=True)
    return Bounded(t.v, t.e + off)


@pytest.fixture
def held(monkeypatch):
    monkeypatch.setattr(lora, "_low", _held)


SHAPES = [
    (1, 0, 2, 16, 512, 256),
    (5, 0, 3, 7, 72, 41),          # nothing aligned
    (70, 0, 3, 32, 264, 200),      # tiles of more than 16 rows
    (40, 0, 4, 64, 128, 600),
    (33, 0, 2, 128, 256, 72),
    (300, 3, 12, 16, 96, 64),      # planned, several routes a row
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_low_rank_rows_keep_their_bits(dev, held, dtype, shape):
    """In the rows' type, forward and gradients."""
    lora._check(lora._case(dev, dtype, *shape, seed=3))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape", SHAPES)
def test_low_rank_rows_keep_their_bits_in_a_float_output(dev, held, dtype, shape):
    c = lora._case(dev, dtype, *shape, seed=4)
    c["base"] = c["base"].float()
    lora._expected(c)[0].check(lora._call(c))


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_low_rank_rows_of_any_size(dev, held, dtype):
    """Rows whose values span many powers of two, and rows near both ends of float32's range."""
    c = lora._case(dev, dtype, 48, 0, 2, 16, 256, 128, seed=5)
    c["base"] = torch.zeros_like(c["base"]).float()
    c["scales"] = torch.tensor([2.0 ** 100, 2.0 ** -100], device=dev)
    c["a"] = (c["a"].float() * torch.logspace(0, -3, 16, device=dev)[:, None]).to(dtype)
    lora._expected(c)[0].check(lora._call(c))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_infinities_of_a_factor_reach_the_outputs(dev, dtype):
    c = lora._case(dev, dtype, 40, 0, 2, 16, 64, 48, seed=6)
    c["b"][0, 3, 5], c["b"][1, 7, 2] = float("inf"), -float("inf")
    got = lora._call(c)
    plain = lora._call({**c, "b": c["b"].nan_to_num(posinf=0.0, neginf=0.0)})
    t = (c["x"].double() @ c["a"].double().mT).permute(1, 0, 2)  # [rows, adapters, rank]
    for row in range(40):
        want = plain[row].clone()
        e = int(c["idx"][row])
        if e == 0:
            want[3] = t[row, 0, 5].sign() * float("inf")
        elif e == 1:
            want[7] = -t[row, 1, 2].sign() * float("inf")
        assert torch.equal(got[row], want)
