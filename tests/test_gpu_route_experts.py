"""The choice of experts among groups (``route_experts``) against float64: the same experts everywhere, weights and gradients
within derived bounds.

A score's error in float32: 2^-20 of it, for the softmax 2^-17 (its exponent loses up to 104 2^-24). Weights divide by a sum
of k such scores."""

import pytest
import torch

import keep_amd
from tests.test_gpu_dense import _replays

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
UNSURE = {"softmax": 2.0 ** -17, "sigmoid": 2.0 ** -20, "sqrtsoftplus": 2.0 ** -20}


def _scores(z, func):
    if func == "softmax":
        p = torch.softmax(z, 1)
        return torch.where((z == -float("inf")).all(1, keepdim=True), 0.0, p)
    if func == "sigmoid":
        return 1 / (1 + torch.exp(-z))
    return torch.sqrt(torch.clamp(z, min=0) + torch.log1p(torch.exp(-z.abs())))


def _order(keys):
    """Descending, NaN as -inf, the lower index first among equals."""
    keys = torch.where(torch.isnan(keys), -float("inf"), keys)
    return torch.sort(keys, dim=1, descending=True, stable=True).indices


def _expected(z, k, bias=None, score_func="softmax", groups=1, topk_groups=None, renormalize=True, route_scale=1.0):
    """On the host, in 64 bits."""
    z = z.detach().double().cpu()
    T, E = z.shape
    s = _scores(z, score_func)
    keys = s if bias is None else s + bias.double().cpu()
    order = _order(keys if bias is not None else z)
    tg = topk_groups or groups
    if tg < groups:
        parts = torch.where(torch.isnan(keys), -float("inf"), keys).view(T, groups, -1)
        value = torch.sort(parts, dim=2, descending=True).values[:, :, :2].sum(2)
        kept = torch.zeros(T, groups, dtype=torch.bool).scatter_(1, _order(value)[:, :tg], True)
        kept = kept.repeat_interleave(E // groups, 1).gather(1, order)
        order = order.gather(1, torch.sort((~kept).to(torch.int32), dim=1, stable=True).indices)
    idx = order[:, :k]
    w = s.gather(1, idx)
    if renormalize:
        w = w / (w.sum(1, keepdim=True) + 1e-20)
    return idx.to(torch.int32), w * route_scale, s


def _check(z, k, **kw):
    func = kw.get("score_func", "softmax")
    r = keep_amd.route_experts(z, k, count_load=True, **kw)
    idx, w, _ = _expected(z, k, **kw)
    assert r.idx.dtype == torch.int32 and torch.equal(r.idx.cpu(), idx)
    assert torch.equal(r.load.cpu(), torch.bincount(idx.reshape(-1).long(), minlength=z.shape[1]).to(torch.int32))
    err = (2 * UNSURE[func] + (k + 4) * 2.0 ** -24) * w.abs() + 2.0 ** -126
    assert ((r.weight.double().cpu() - w).abs() <= err).all()
    return r


def _logits(dev, T, E, dtype=F32, seed=0, std=2.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(T, E, device=dev, generator=g) * std).to(dtype)


CASES = [  # T, E, k, groups, topk_groups
    (1, 1, 1, 1, 1), (1, 384, 6, 1, 1), (5, 8, 8, 1, 1), (3, 7, 3, 1, 1), (257, 256, 8, 8, 4), (64, 384, 6, 8, 3),
    (9, 60, 5, 6, 2), (33, 512, 32, 1, 1), (10, 1024, 8, 1, 1), (4, 1020, 4, 5, 2), (6, 990, 7, 33, 9), (12, 64, 4, 64, 5),
    (11, 128, 2, 64, 40), (7, 12, 1, 12, 1), (100, 96, 8, 4, 4), (5, 160, 6, 8, 8), (2, 1023, 3, 11, 3),
]


@pytest.mark.parametrize("T, E, k, groups, topk_groups", CASES)
@pytest.mark.parametrize("func", sorted(UNSURE))
@pytest.mark.parametrize("biased", [False, True])
def test_choice(dev, T, E, k, groups, topk_groups, func, biased):
    for dtype in (F32, BF16, F16):
        z = _logits(dev, T, E, dtype, seed=E + T)
        bias = torch.randn(E, device=dev) * 0.1 if biased else None
        _check(z, k, bias=bias, score_func=func, groups=groups, topk_groups=topk_groups)
        _check(z, k, bias=bias, score_func=func, groups=groups, topk_groups=topk_groups, renormalize=False,
               route_scale=2.5)


@pytest.mark.parametrize("func", sorted(UNSURE))
@pytest.mark.parametrize("groups, topk_groups", [(1, 1), (8, 3), (5, 2)])
def test_equal_keys_take_the_lower_index(dev, func, groups, topk_groups):
    z = torch.randint(-2, 3, (200, 40), device=dev).float() + 0.3  # five values among forty experts, no two pairs' sums alike
    _check(z, 6, score_func=func, groups=groups, topk_groups=topk_groups)
    _check(z, 6, score_func=func, groups=groups, topk_groups=topk_groups, bias=torch.zeros(40, device=dev))
    _check(z, 6, score_func=func, groups=groups, topk_groups=topk_groups, 
           bias=torch.tensor([0.0, 0.25, 0.6], device=dev).repeat(14)[:40])


@pytest.mark.parametrize("func", sorted(UNSURE))
@pytest.mark.parametrize("groups, topk_groups", [(1, 1), (8, 4), (6, 1)])
def test_keys_closer_than_float32_tells_apart(dev, func, groups, topk_groups):
    """The bias takes each score back to one value as far as float32 can: keys differ by its rounding alone."""
    E = 96
    z = _logits(dev, 1, E, seed=3)
    s = _scores(z.double(), func)[0]
    bias = (0.7 - s).float()
    _check(z, 8, score_func=func, groups=groups, topk_groups=topk_groups, bias=bias)
    many = z + torch.randn(300, E, device=dev, generator=torch.Generator(device=dev).manual_seed(5)) * 1e-6
    _check(many, 8, score_func=func, groups=groups, topk_groups=topk_groups, bias=bias)


@pytest.mark.parametrize("func", sorted(UNSURE))
@pytest.mark.parametrize("groups, topk_groups", [(1, 1), (4, 2)])
def test_masked_logits(dev, func, groups, topk_groups):
    """Experts behind logits of -inf or the lowest value, down to rows that have nothing left."""
    low = torch.finfo(F32).min
    for mask in (-float("inf"), low):
        z = _logits(dev, 6, 32)
        z[0, :] = mask
        z[1, 1:] = mask
        z[2, ::2] = mask
        z[3, 4:] = mask
        for bias in (None, torch.randn(32, device=dev, generator=torch.Generator(device=dev).manual_seed(1)) * 0.1):
            r = _check(z, 5, score_func=func, groups=groups, topk_groups=topk_groups, bias=bias)
            assert torch.isfinite(r.weight).all()
        leaf = z.clone().requires_grad_(True)
        w = keep_amd.route_experts(leaf, 5, score_func=func, groups=groups, topk_groups=topk_groups).weight
        assert torch.isfinite(torch.autograd.grad(w.square().sum(), leaf)[0]).all()


def test_nan_and_infinite_logits(dev):
    z = _logits(dev, 3, 16)
    z[1, 4] = float("nan")
    z[2, 6] = float("inf")
    for func in sorted(UNSURE):
        r = keep_amd.route_experts(z, 4, score_func=func)
        assert (r.idx[1] != 4).all() and int(r.idx[2, 0]) == 6
        for row in range(3):
            assert len(set(r.idx[row].tolist())) == 4 and ((r.idx[row] >= 0) & (r.idx[row] < 16)).all()
        biased = keep_amd.route_experts(z, 4, score_func=func, bias=torch.zeros(16, device=dev), groups=4, topk_groups=2)
        assert ((biased.idx >= 0) & (biased.idx < 16)).all()
        assert torch.equal(r.idx[0], keep_amd.route_experts(z[:1], 4, score_func=func).idx[0])


def test_absent_experts_of_a_biased_choice(dev):
    """Experts that the bias rules out (the residency cache's -1e30)."""
    z = _logits(dev, 50, 64)
    bias = torch.zeros(64, device=dev)
    bias[::3] = keep_amd.router.OFF
    r = _check(z, 6, score_func="sigmoid", bias=bias)
    assert (r.idx % 3 != 0).all()
    _check(z, 6, score_func="sigmoid", bias=bias, groups=8, topk_groups=4)


def test_one_group_is_the_dual_router(dev):
    z = _logits(dev, 40, 384)
    for func in sorted(UNSURE):
        a, b = keep_amd.route_experts(z, 6, score_func=func), keep_amd.router_dual_topk(z, 6, score_func=func)
        assert torch.equal(a.idx, b.idx)
        assert ((a.weight - b.weight).abs() <= 4 * UNSURE[func] * b.weight).all()


def _expected_grad(z, dw, idx, func, renormalize, scale):
    """dz and its bound: each score within UNSURE of itself, times what it enters."""
    leaf = z.detach().double().cpu().requires_grad_(True)
    s = _scores(leaf, func).gather(1, idx.long().cpu())
    w = s / (s.sum(1, keepdim=True) + 1e-20) if renormalize else s
    dz, = torch.autograd.grad(w * scale, leaf, dw.double().cpu())
    with torch.no_grad():
        full = _scores(leaf, func)
        g = dw.double().cpu().abs() * abs(scale)
        if renormalize:
            total = s.sum(1, keepdim=True) + 1e-20
            g = (g + (g * s).sum(1, keepdim=True) / total) / total
        part = torch.zeros_like(full).scatter_(1, idx.long().cpu(), g * s)
        if func == "softmax":
            part = part + full * (g * s).sum(1, keepdim=True)
        u = 8 * UNSURE[func] + 40 * 2.0 ** -24
    return dz, part * u + 2.0 ** -120


@pytest.mark.parametrize("T, E, k, groups, topk_groups", CASES)
@pytest.mark.parametrize("func", sorted(UNSURE))
@pytest.mark.parametrize("renormalize", [False, True])
def test_gradient(dev, T, E, k, groups, topk_groups, func, renormalize):
    for dtype in (F32, BF16):
        z = _logits(dev, T, E, dtype, seed=k).requires_grad_(True)
        dw = torch.randn(T, k, device=dev, generator=torch.Generator(device=dev).manual_seed(2))
        r = keep_amd.route_experts(z, k, score_func=func, groups=groups, topk_groups=topk_groups, renormalize=renormalize,
                                   route_scale=1.5, count_load=True)
        assert not r.idx.requires_grad and not r.load.requires_grad
        plain = keep_amd.route_experts(z.detach(), k, score_func=func, groups=groups, topk_groups=topk_groups,
                                       renormalize=renormalize, route_scale=1.5)
        assert torch.equal(plain.idx, r.idx) and torch.equal(plain.weight, r.weight.detach())
        got, = torch.autograd.grad(r.weight, z, dw)
        assert got.dtype == dtype
        want, err = _expected_grad(z, dw, r.idx, func, renormalize, 1.5)
        f = torch.finfo(dtype)
        err = err + (want.abs() + err) * f.eps / 2 + f.tiny * f.eps
        assert ((got.double().cpu() - want).abs() <= err).all()


def test_gradient_against_differences(dev):
    z = _logits(dev, 4, 24, seed=9).requires_grad_(True)
    dw = torch.randn(4, 3, device=dev)
    for func in sorted(UNSURE):
        r = keep_amd.route_experts(z, 3, score_func=func, groups=4, topk_groups=2)
        got, = torch.autograd.grad(r.weight, z, dw)
        along = torch.randn(4, 24, device=dev, dtype=torch.float64)

        def loss(t):
            s = _scores(z.detach().double() + t * along, func).gather(1, r.idx.long())
            return (s / s.sum(1, keepdim=True) * dw.double()).sum()
        slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
        # 96 terms of magnitude 1, each within the scores' 2^-17 and the difference's 1e-9
        assert abs(slope - (got.double() * along).sum()) <= 96 * 2.0 ** -16


def test_layouts_streams_and_empty(dev):
    z = _logits(dev, 30, 64)
    want = keep_amd.route_experts(z, 4)
    wide = torch.randn(30, 100, device=dev)
    wide[:, 20:84] = z
    assert torch.equal(keep_amd.route_experts(wide[:, 20:84], 4).idx, want.idx)
    assert torch.equal(keep_amd.route_experts(z.t().contiguous().t(), 4).weight, want.weight)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = keep_amd.route_experts(z, 4, count_load=True)
    s.synchronize()
    assert torch.equal(got.idx, want.idx)
    leaf = z[:0].clone().requires_grad_(True)
    none = keep_amd.route_experts(leaf, 4, count_load=True)
    assert none.idx.shape == (0, 4) and (none.load == 0).all()
    assert torch.autograd.grad(none.weight.sum(), leaf)[0].shape == (0, 64)


def test_graphs(dev):
    cases = [(_logits(dev, 50, 256, seed=s), torch.randn(256, device=dev) * 0.1, torch.randn(50, 8, device=dev))
             for s in range(4)]
    c = [t.clone() for t in cases[0]]

    def step():
        leaf = c[0].detach().requires_grad_(True)
        r = keep_amd.route_experts(leaf, 8, bias=c[1], score_func="sigmoid", groups=8, topk_groups=4, count_load=True)
        return [r.idx, r.weight.detach(), r.load, *torch.autograd.grad(r.weight, leaf, c[2])]
    _replays(step, c, cases)
