"""The norm with the residual's addition (``rmsnorm``, ``rmsnorm_quant``) and its gradients against float64.

Bounds: a row's sums run over at most 32 values in a thread, six steps of a wave and eight waves, 46 roundings; with the
products' and the division's 64 of 2^-24 each, half of it behind the square root of a sum of one sign (``ROW``). The weight's
gradient adds rows in an order of the kernel's choice: T 2^-24 of the terms' magnitudes (``Bounded.sum``)."""

import pytest
import torch

import keep_amd
from tests.bounded import Bounded
from tests.test_gpu_dense import _replays

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
ROW = 64 * 2.0 ** -24
EPS = 1e-6


def _case(dev, T, n, dtype, res, wdt, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dt, std=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(dt)
    return {"x": normal(T, n, dt=dtype), "res": None if res is None else normal(T, n, dt=res, std=3.0),
            "w": None if wdt is None else (1 + normal(n, dt=F32, std=0.3)).to(wdt), "dy": normal(T, n, dt=dtype),
            "dh": None if res is None else normal(T, n, dt=res)}


def _stream(c):
    """The stream within its bound, and (from the kernel's own) what it normalises."""
    return None if c["res"] is None else (Bounded(c["res"]) + Bounded(c["x"])).round(c["res"].dtype)


def _normed(c, h):
    """Unrounded y, its bound, and the row's 1 / rms in 64 bits."""
    h = h.double()
    r = 1 / torch.sqrt((h * h).sum(-1, keepdim=True) / h.shape[-1] + EPS)
    y = h * r * (1 if c["w"] is None else c["w"].double())
    return Bounded(y, y.abs() * (ROW / 2 + 8 * 2.0 ** -24)), r


def _expected_grads(c, h, r):
    h, dy = h.double(), c["dy"].double()
    n = h.shape[-1]
    w = torch.ones(n, device=h.device, dtype=torch.float64) if c["w"] is None else c["w"].double()
    g = dy * w
    mean, size = (g * h).sum(-1, keepdim=True) / n, (g * h).abs().sum(-1, keepdim=True) / n
    d = r * (g - h * r * r * mean)
    e = r * (g.abs() * ROW + h.abs() * r * r * (mean.abs() * 2 * ROW + size * 2 * ROW))
    d = Bounded(d, e)
    if c["res"] is not None:
        d = d + Bounded(c["dh"])
    terms = dy * h * r
    dw = Bounded(terms, terms.abs() * ROW).sum(0)
    return d, dw


def _check(c):
    x, res, w = c["x"], c["res"], c["w"]
    out = keep_amd.rmsnorm(x, w, EPS, residual=res)
    y, h = (out, x) if res is None else out
    assert y.dtype == x.dtype and (res is None or h.dtype == res.dtype)
    if res is not None:
        _stream(c).check(h, "h")
    unrounded, r = _normed(c, h)
    unrounded.round(x.dtype).check(y, "y")
    names = [k for k in ("x", "res", "w") if c[k] is not None]
    leaves = [c[k].detach().requires_grad_(True) for k in names]
    a = dict(zip(names, leaves))
    out = keep_amd.rmsnorm(a["x"], a.get("w"), EPS, residual=a.get("res"))
    outs = (out,) if res is None else out
    assert torch.equal(outs[0], y) and (res is None or torch.equal(outs[1], h))
    grads = dict(zip(names, torch.autograd.grad(outs, leaves, [c["dy"], c["dh"]][:len(outs)])))
    d, dw = _expected_grads(c, h, r)
    d.round(x.dtype).check(grads["x"], "dx")
    if res is not None:
        d.round(res.dtype).check(grads["res"], "dres")
    if w is not None:
        dw.round(w.dtype).check(grads["w"], "dw")
    for k, g in grads.items():
        assert g.dtype == c[k].dtype and g.shape == c[k].shape


SHAPES = [(1, 1), (1, 7168), (3, 8), (5, 13), (2, 64), (9, 511), (4, 513), (7, 1000), (65, 1024), (33, 2880), (130, 2048),
          (3, 2049), (17, 4096), (5, 4100), (1031, 72), (6, 7168), (3, 8191), (2, 8200), (3, 16384), (2, 16383), (2100, 520)]


@pytest.mark.parametrize("T, n", SHAPES)
@pytest.mark.parametrize("dtype, res, wdt", [(BF16, BF16, BF16), (F16, F32, F16), (F32, F32, F32), (BF16, None, F32),
                                             (F16, F16, None), (BF16, F32, BF16)])
def test_norm_and_gradients(dev, T, n, dtype, res, wdt):
    _check(_case(dev, T, n, dtype, res, wdt, seed=T + n))


@pytest.mark.parametrize("T, n", SHAPES)
@pytest.mark.parametrize("dtype, res, block, pow2", [(BF16, BF16, 128, False), (F16, F32, 16, True), (F32, None, 512, False),
                                                     (BF16, None, 64, True)])
def test_quant(dev, T, n, dtype, res, block, pow2):
    c = _case(dev, T, n, dtype, res, dtype, seed=n)
    if T > 1:
        c["x"][-1] = 0  # a row of zeros under zeros: its scales are the bound's
        if res is not None:
            c["res"][-1] = 0
    got = keep_amd.rmsnorm_quant(c["x"], c["w"], EPS, residual=c["res"], quant_block=block, pow2_scales=pow2)
    q, scales = got[:2]
    h = c["x"] if res is None else got[2]
    if res is not None:
        assert torch.equal(h, keep_amd.rmsnorm(c["x"], c["w"], EPS, residual=c["res"])[1])
    blocks = (n + block - 1) // block
    assert q.dtype == torch.float8_e4m3fn and q.shape == (T, n) and scales.shape == (T, blocks)
    y, _ = _normed(c, h)
    pad = torch.zeros(T, blocks * block, device=dev, dtype=torch.float64)
    pad[:, :n] = y.v.abs()
    top = pad.view(T, blocks, block).amax(2).clamp(min=1e-4)
    err = ROW / 2 + 10 * 2.0 ** -24
    s = scales.double()
    if pow2:
        mantissa, _ = torch.frexp(s)
        assert (mantissa == 0.5).all()
        assert (s >= top / 448 * (1 - err)).all() and (s < 2 * top / 448 * (1 + err)).all()
    else:
        assert ((s - top / 448).abs() <= err * top / 448).all()
    each = s.repeat_interleave(block, 1)[:, :n]
    # half a step of e4m3 (2^-4 of the value, or half of the smallest subnormal 2^-9), y's own bound, the division's rounding
    bound = y.e + (y.v.abs() + y.e) * 2.0 ** -4 + each * 2.0 ** -10 + y.v.abs() * 2.0 ** -23
    off = (q.double() * each - y.v).abs() - bound
    assert (off <= 0).all(), off.max()
    if T > 1:
        assert (q[-1].float() == 0).all()


def test_rows_of_infinities_and_nan(dev):
    x = torch.randn(4, 256, device=dev)
    x[1, 3], x[2, 7] = float("inf"), float("nan")
    y = keep_amd.rmsnorm(x)
    q, s = keep_amd.rmsnorm_quant(x, quant_block=64)
    for row in (0, 3):
        assert torch.isfinite(y[row]).all() and torch.isfinite(q[row].float()).all()
    assert torch.isnan(y[1, 3]) and (y[1, :3] == 0).all()  # inf / inf, and finite / inf
    assert torch.isnan(y[2]).all() and torch.isnan(q[2].float()).all() and torch.isnan(s[2]).all()
    assert torch.isnan(q[1, 3].float()) and (q[1, 64:].float() == 0).all()


def test_extreme_rows(dev):
    """Rows whose squares are subnormal or near the largest: eps keeps the first finite."""
    for scale in (1e-30, 1e-18, 1e15):
        x = torch.randn(3, 512, device=dev) * scale
        want = x.double() / torch.sqrt((x.double() ** 2).mean(-1, keepdim=True) + EPS)
        got = keep_amd.rmsnorm(x)
        assert ((got.double() - want).abs() <= want.abs() * 2 * ROW + 2.0 ** -126).all()


@pytest.mark.parametrize("used", ["y", "h"])
def test_only_one_output_used(dev, used):
    c = _case(dev, 5, 96, BF16, BF16, BF16)
    leaves = [c[k].requires_grad_(True) for k in ("x", "res", "w")]
    y, h = keep_amd.rmsnorm(c["x"], c["w"], EPS, residual=c["res"])
    if used == "h":
        dx, dr, dw = torch.autograd.grad(h, leaves, c["dh"])
        assert torch.equal(dx, c["dh"]) and torch.equal(dr, c["dh"]) and (dw == 0).all()
    else:
        got = torch.autograd.grad(y, leaves, c["dy"])
        c["dh"] = torch.zeros_like(c["dh"])
        d, dw = _expected_grads(c, h.detach(), _normed(c, h.detach())[1])
        d.round(BF16).check(got[0])
        d.round(BF16).check(got[1])
        dw.round(BF16).check(got[2])


@pytest.mark.parametrize("needs", [(1, 0, 0), (0, 1, 0), (0, 0, 1)])
@pytest.mark.parametrize("res", [BF16, F32])
def test_one_gradient_alone(dev, needs, res):
    c = _case(dev, 37, 264, BF16, res, F32)
    leaves = [c[k].requires_grad_(bool(n)) for k, n in zip(("x", "res", "w"), needs)]
    y, h = keep_amd.rmsnorm(c["x"], c["w"], EPS, residual=c["res"])
    leaf = next(t for t in leaves if t.requires_grad)
    got, = torch.autograd.grad((y, h) if h.requires_grad else y, leaf, (c["dy"], c["dh"]) if h.requires_grad else c["dy"])
    c = {k: v.detach() for k, v in c.items()}
    d, dw = _expected_grads(c, h.detach(), _normed(c, h.detach())[1])
    (dw if needs[2] else d).round(leaf.dtype).check(got)


def test_gradient_against_differences(dev):
    c = _case(dev, 3, 40, F32, F32, F32, seed=4)
    names = ("x", "res", "w")
    leaves = [c[k].requires_grad_(True) for k in names]
    grads = torch.autograd.grad(keep_amd.rmsnorm(c["x"], c["w"], EPS, residual=c["res"]), leaves, (c["dy"], c["dh"]))
    g = torch.Generator(device=dev).manual_seed(1)

    def loss(t, along):
        x, res, w = (c[k].detach().double() + t * a for k, a in zip(names, along))
        h = res + x
        y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + EPS) * w
        return (y * c["dy"].double()).sum() + (h * c["dh"].double()).sum()
    for i in range(3):
        along = [torch.randn(t.shape, device=dev, generator=g, dtype=torch.float64) * (i == j) for j, t in enumerate(leaves)]
        slope = (loss(1e-5, along) - loss(-1e-5, along)) / 2e-5
        got = sum((a * gr.double()).sum() for a, gr in zip(along, grads))
        # float32 gradients and float32's rounding of h (2^-24 of it), about 120 terms of magnitude 1
        assert abs(slope - got) <= 120 * 2.0 ** -20


def test_layouts_streams_and_empty(dev):
    c = _case(dev, 6, 200, BF16, BF16, BF16)
    want = keep_amd.rmsnorm(c["x"], c["w"], EPS, residual=c["res"])
    wide = torch.randn(6, 300, device=dev).to(BF16)
    wide[:, 40:240] = c["x"]
    strided = keep_amd.rmsnorm(wide[:, 40:240], c["w"], EPS, residual=c["res"].view(2, 3, 200).view(6, 200))
    assert all(torch.equal(a, b) for a, b in zip(want, strided))
    odd = torch.empty(6 * 200 + 1, device=dev, dtype=BF16)[1:].view(6, 200).copy_(c["x"])
    assert odd.data_ptr() % 4 == 2
    assert torch.equal(keep_amd.rmsnorm(odd, c["w"], EPS, residual=c["res"])[0], want[0])
    three = keep_amd.rmsnorm(c["x"].view(2, 3, 200), c["w"], EPS, residual=c["res"].view(2, 3, 200))
    assert three[0].shape == (2, 3, 200) and torch.equal(three[0].view(6, 200), want[0])
    assert torch.equal(keep_amd.rmsnorm(c["x"][0], c["w"], EPS), keep_amd.rmsnorm(c["x"], c["w"], EPS)[0])
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = keep_amd.rmsnorm(c["x"], c["w"], EPS, residual=c["res"])
    s.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    w = c["w"].requires_grad_(True)
    none = keep_amd.rmsnorm(c["x"][:0], w, EPS, residual=c["res"][:0])
    assert none[0].shape == (0, 200) and (torch.autograd.grad(none[0].sum(), w)[0] == 0).all()
    assert keep_amd.rmsnorm_quant(c["x"][:0])[1].shape == (0, 2)


def test_graphs(dev):
    cases = [_case(dev, 70, 1032, BF16, F32, BF16, seed=s) for s in range(4)]
    names = ("x", "res", "w", "dy", "dh")
    c = [cases[0][k].clone() for k in names]
    _replays(lambda: list(keep_amd.rmsnorm_quant(c[0], c[2], EPS, residual=c[1])), c, [[k[n] for n in names] for k in cases])

    def step():
        leaves = [t.detach().requires_grad_(True) for t in c[:3]]
        y, h = keep_amd.rmsnorm(leaves[0], leaves[2], EPS, residual=leaves[1])
        return [y.detach(), h.detach(), *torch.autograd.grad((y, h), leaves, (c[3], c[4]))]
    _replays(step, c, [[k[n] for n in names] for k in cases])


def test_results_do_not_change_from_call_to_call(dev):
    c = _case(dev, 3000, 264, BF16, BF16, F32)
    leaves = [c[k].requires_grad_(True) for k in ("x", "res", "w")]

    def grads():
        return torch.autograd.grad(keep_amd.rmsnorm(c["x"], c["w"], EPS, residual=c["res"]), leaves, (c["dy"], c["dh"]))
    first = grads()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, grads()))
