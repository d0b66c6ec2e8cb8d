"""Equal keys at the boundary of a biased choice, with other keys behind them that float32 does not tell apart: the choice is
64 bits' (``route_experts``)."""

import pytest
import torch

import keep_amd
from tests.test_gpu_route_experts import _check

pytestmark = pytest.mark.gpu
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")
# logits whose scores float32 does not tell apart beside the bias, and the bias
CLOSE = {"sigmoid": (20.0, 0.0), "softmax": (0.0, 0.5), "sqrtsoftplus": (-40.0, 1.0)}


def test_a_larger_key_behind_an_equal_pair(dev):
    zero = torch.zeros(3, device=dev)
    for last in (20.125, 21.0):
        z = torch.tensor([[20.0, 20.0, last]], device=dev)
        for k in (1, 2):
            assert int(_check(z, k, score_func="sigmoid", bias=zero).idx[0, 0]) == 2
    z = torch.tensor([[25.0, 20.0, 20.0, 20.0, 20.0, 21.0, 20.0]], device=dev)
    assert _check(z, 2, score_func="sigmoid", bias=torch.zeros(7, device=dev)).idx.tolist() == [[0, 5]]
    masked = torch.tensor([[-INF, -INF, 0.0, 30.0]], device=dev)
    r = _check(masked, 2, score_func="softmax", bias=torch.full((4,), 0.5, device=dev))
    assert r.idx.tolist() == [[3, 2]]


@pytest.mark.parametrize("func", sorted(CLOSE))
@pytest.mark.parametrize("groups, topk_groups", [(1, 1), (8, 3), (8, 8)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16])
def test_runs_of_equal_keys_among_close_ones(dev, func, groups, topk_groups, dtype):
    """Four logits among many experts, so that every boundary cuts a run of equal keys; float32 sees one key."""
    base, b = CLOSE[func]
    g = torch.Generator(device=dev).manual_seed(groups + topk_groups)
    for E in (8, 40, 256):
        if topk_groups * (E // groups) < 7:
            continue
        z = base + 0.25 * torch.randint(0, 4, (60, E), device=dev, generator=g).float()
        rare = torch.rand(60, E, device=dev, generator=g)
        z = torch.where(rare < 0.9, torch.full_like(z, base), z)  # mostly one value: the larger ones lie behind it
        if func == "softmax":
            z[:, 3] = 30.0  # the others' scores vanish beside the bias
        z = z.to(dtype)
        bias = torch.full((E,), b, device=dev)
        for k in (1, 2, 5, 7):
            _check(z, k, score_func=func, groups=groups, topk_groups=topk_groups, bias=bias)


@pytest.mark.parametrize("func", sorted(CLOSE))
def test_masked_logits_under_a_constant_bias(dev, func):
    g = torch.Generator(device=dev).manual_seed(7)
    z = torch.randn(40, 64, device=dev, generator=g)
    z[torch.rand(40, 64, device=dev, generator=g) < 0.9] = -INF
    z[:, 60] = 30.0
    for groups, topk_groups in ((1, 1), (8, 4)):
        for k in (2, 4, 8):
            _check(z, k, score_func=func, groups=groups, topk_groups=topk_groups, bias=torch.full((64,), 0.5, device=dev))


def test_every_expert_equal(dev):
    for func in sorted(CLOSE):
        r = _check(torch.full((20, 96), 0.25, device=dev), 6, score_func=func, bias=torch.zeros(96, device=dev))
        assert (r.idx == torch.arange(6, device=dev, dtype=torch.int32)).all()
