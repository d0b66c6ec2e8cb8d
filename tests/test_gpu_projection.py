"""Dense projections with their epilogue (``linear``, ``linear_q8``) and their gradients against float64 with derived bounds.

The activations' own errors: the sigmoid's exponent rounds by |u| 2^-24, v_exp_f32, the sum and v_rcp_f32 by a step each; the
error function's complement by 16 steps, its argument's rounding times 2 x^2; all of it under ``_act``'s (u^2 + 24) 2^-23 of the
value. Slopes of act are at most 1.13, their own slopes at most 0.8 (gelu; silu 0.5)."""

import math

import pytest
import torch

import keep_amd
from tests.bounded import U, Bounded
from tests.test_gpu_dense import _replays

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
C = math.sqrt(2 / math.pi)


def _value(u, act):
    if act == "relu":
        return u.clamp(min=0)
    if act == "silu":
        return u / (1 + torch.exp(-u))
    if act == "gelu":
        return 0.5 * u * torch.special.erfc(-u * math.sqrt(0.5))
    if act == "gelu_tanh":
        return u / (1 + torch.exp(-2 * C * (u + 0.044715 * u ** 3)))
    return u


def _slope(u, act):
    u = u.detach().requires_grad_(True)
    with torch.enable_grad():
        v = _value(u, act)
        return torch.autograd.grad(v.sum(), u)[0].detach() if act else torch.ones_like(u)


def _act(u, act):
    if act is None:
        return u
    v = _value(u.v, act)
    return Bounded(v, 1.13 * u.e + (v.abs() + u.e) * ((u.v.abs() + u.e) ** 2 + 24) * U)


def _case(dev, dtype, M, N, K, bias=None, residual=None, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, dt=dtype, std=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(dt)
    return {"x": normal(M, K), "w": normal(N, K, std=K ** -0.5), "b": None if bias is None else normal(N, dt=bias),
            "r": None if residual is None else normal(M, N, dt=residual), "dy": normal(M, N)}


def _call(c, act, od=None):
    return keep_amd.linear(c["x"], c["w"], c["b"], activation=act, residual=c["r"], out_dtype=od)


def _expected(c, act, od, grads=True):
    x, w = Bounded(c["x"]), Bounded(c["w"])
    dtype, M = c["x"].dtype, c["x"].shape[0]
    u = x @ w.T
    if c["b"] is not None:
        u = u + Bounded(c["b"].expand(M, -1))
    out = _act(u, act)
    if c["r"] is not None:
        out = Bounded(c["r"]) + out
    out = out.round(od)
    if not grads:
        return out, None
    dy = c["dy"].double()
    if act is None:
        du = Bounded(dy)
    else:
        kept = u.round(dtype)  # what the gradient sees
        s = _slope(u.v, act)
        if act == "relu":
            e = (kept.v.abs() <= kept.e).double()
        else:
            e = 0.8 * kept.e + ((u.v.abs() + u.e) ** 2 + 24) * U * (s.abs() + u.v.abs().clamp(max=1.0))
        du = Bounded(dy * s, dy.abs() * (e + U * s.abs()))
    low = du.round(dtype) if act is not None else du
    got = {"x": (low @ w).round(dtype), "w": (low.T @ x).round(dtype)}
    if c["b"] is not None:
        got["b"] = du.sum(0).round(c["b"].dtype)
    if c["r"] is not None:
        got["r"] = Bounded(c["dy"]).round(c["r"].dtype)
    return out, got


def _check(c, act, od=None, grads=True):
    dtype = c["x"].dtype
    od = od or (dtype if c["r"] is None else c["r"].dtype)
    out = _call(c, act, od)
    assert out.dtype == od
    grads = grads and od == dtype
    want, gw = _expected(c, act, od, grads)
    want.check(out, "out")
    if not grads:
        return
    names = [n for n in ("x", "w", "b", "r") if c[n] is not None]
    leaves = {n: c[n].detach().requires_grad_(True) for n in names}
    rec = _call({**c, **leaves}, act, od)
    assert torch.equal(rec, out)
    for n, g in zip(names, torch.autograd.grad(rec, list(leaves.values()), c["dy"])):
        assert g.dtype == c[n].dtype and g.shape == c[n].shape
        gw[n].check(g, "d" + n)


SHAPES = [  # M, N, K
    (1, 1, 1), (1, 384, 4096), (2, 33, 40), (3, 20, 17), (7, 130, 200), (16, 256, 1000), (17, 64, 64), (5, 1440, 2880),
    (33, 129, 513), (64, 384, 512), (65, 100, 36), (100, 513, 72), (129, 260, 264), (200, 31, 2048), (333, 144, 288),
    (512, 8, 8), (300, 640, 8), (260, 264, 1032), (1500, 136, 100), (700, 300, 333),
]


@pytest.mark.parametrize("M, N, K", SHAPES)
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_linear(dev, dtype, M, N, K):
    _check(_case(dev, dtype, M, N, K, seed=M), None)
    _check(_case(dev, dtype, M, N, K, bias=dtype, residual=dtype, seed=N), "silu")


@pytest.mark.parametrize("act", [None, "relu", "silu", "gelu", "gelu_tanh"])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
def test_epilogues(dev, act, dtype):
    for M in (3, 90, 300):
        _check(_case(dev, dtype, M, 72, 80, bias=F32), act)
        _check(_case(dev, dtype, M, 71, 80, residual=dtype, seed=1), act)
        _check(_case(dev, dtype, M, 72, 80, bias=dtype, residual=F32, seed=2), act)
        _check(_case(dev, dtype, M, 72, 80, bias=dtype, seed=3), act, od=F32)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M, N, K", [(4100, 4352, 200), (4096, 4096, 64), (3900, 4097, 136), (3840, 200, 4232)])
def test_large_tiles(dev, dtype, M, N, K):
    """Tiles of 256 x 256, whole and cut, in each of the three products."""
    _check(_case(dev, dtype, M, N, K), None)


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("M, N, K", [(20, 16, 8192), (130, 130, 5000), (40, 300, 16392), (9000, 40, 24)])
def test_slices_of_the_summed_index(dev, dtype, M, N, K):
    _check(_case(dev, dtype, M, N, K, bias=dtype, residual=dtype), "gelu")


def test_float_output_of_16_bit_rows_keeps_its_gradients_bits(dev):
    c = _case(dev, BF16, 70, 40, 96, bias=F32)
    leaves = [c[n].requires_grad_(True) for n in ("x", "w", "b")]
    out = keep_amd.linear(*leaves, out_dtype=F32)
    dy = torch.randn(70, 40, device=dev) * 1e-30  # below bfloat16's products, and with float32's bits
    dx, dw, db = torch.autograd.grad(out, leaves, dy)
    x, w, d = Bounded(c["x"]), Bounded(c["w"]), Bounded(dy)
    (d @ w).round(BF16).check(dx)
    (d.T @ x).round(BF16).check(dw)
    d.sum(0).round(F32).check(db)


def test_extreme_values_of_the_activations(dev):
    x = torch.tensor([[-3e38], [-1e20], [-100.0], [-20.0], [0.0], [20.0], [100.0], [1e20], [3e38]], device=dev)
    one = torch.ones(1, 1, device=dev)
    for act in ("relu", "silu", "gelu", "gelu_tanh"):
        leaf = x.clone().requires_grad_(True)
        y = keep_amd.linear(leaf, one, activation=act)
        slope, = torch.autograd.grad(y.sum(), leaf)
        assert torch.isfinite(y).all() and torch.isfinite(slope).all()
        assert torch.equal(y[5:], x[5:]) and (y[:3].abs() <= 1e-30).all() and y[4] == 0
        assert (slope[5:] == 1).all() and (slope[:3].abs() <= 1e-30).all()


def test_infinities_and_nan_stay_in_their_rows(dev):
    for M in (5, 200):
        c = _case(dev, BF16, M, 144, 264)
        c["x"][1, 3], c["x"][3, 0] = float("inf"), float("nan")
        out = _call(c, "silu")
        clean = torch.ones(M, dtype=torch.bool, device=dev)
        clean[1] = clean[3] = False
        assert torch.isfinite(out[clean]).all() and torch.isnan(out[3]).all() and not torch.isfinite(out[1]).any(0).all()


def test_one_gradient_alone(dev):
    c = _case(dev, BF16, 150, 72, 88, bias=F32, residual=F32)
    for n in ("x", "w", "b", "r"):
        leaf = c[n].detach().requires_grad_(True)
        got, = torch.autograd.grad(keep_amd.linear(**{k: v for k, v in zip(("x", "weight", "bias"), (
            {**c, n: leaf}[m] for m in ("x", "w", "b")))}, residual={**c, n: leaf}["r"], activation="silu", out_dtype=BF16),
            leaf, c["dy"])
        _expected(c, "silu", BF16)[1][n].check(got, n)


def test_gradient_against_differences(dev):
    g = torch.Generator(device=dev).manual_seed(3)
    for act in ("silu", "gelu", "gelu_tanh"):
        c = _case(dev, F32, 5, 6, 8, bias=F32, residual=F32)
        names = ("x", "w", "b", "r")
        leaves = [c[n].requires_grad_(True) for n in names]
        grads = torch.autograd.grad(_call(c, act), leaves, c["dy"])
        for i in range(4):
            along = [torch.randn(t.shape, device=dev, generator=g, dtype=torch.float64) * (i == j)
                     for j, t in enumerate(leaves)]

            def loss(t):
                x, w, b, r = (c[n].detach().double() + t * a for n, a in zip(names, along))
                return ((_value(x @ w.T + b, act) + r) * c["dy"].double()).sum()
            slope = (loss(1e-5) - loss(-1e-5)) / 2e-5
            got = sum((a * gr.double()).sum() for a, gr in zip(along, grads))
            assert abs(slope - got) <= 300 * 2.0 ** -19  # at most 300 terms of magnitude 1 to 4, in float32


def test_layouts(dev):
    """Views with a pitch are read where they lie; other strides and odd addresses are copied."""
    c = _case(dev, BF16, 40, 72, 96, bias=BF16, residual=BF16)
    want = _call(c, "silu")
    wide = torch.full((40, 160), float("nan"), device=dev, dtype=BF16)
    wide[:, 32:128] = c["x"]
    wview = torch.full((72, 112), float("nan"), device=dev, dtype=BF16)
    wview[:, :96] = c["w"]
    odd = torch.empty(40 * 96 + 1, device=dev, dtype=BF16)[1:].view(40, 96).copy_(c["x"])
    for x in (wide[:, 32:128], c["x"].t().contiguous().t(), odd, c["x"].view(8, 5, 96)):
        for w in (c["w"], wview[:, :96], c["w"].t().contiguous().t()):
            got = keep_amd.linear(x, w, c["b"], activation="silu", residual=c["r"].view(*x.shape[:-1], 72))
            assert torch.equal(got.view(40, 72), want)
    row = keep_amd.linear(c["x"][0], c["w"])
    assert row.shape == (72,) and torch.equal(row, keep_amd.linear(c["x"][:1], c["w"])[0])
    same = keep_amd.linear(c["x"][:1].expand(40, 96), c["w"])
    assert torch.equal(same[0], same[39])
    odd_k = torch.full((40, 100), float("nan"), device=dev, dtype=BF16)
    odd_k[:, :93] = c["x"][:, :93]
    assert torch.isfinite(keep_amd.linear(odd_k[:, :93], c["w"][:, :93])).all()


def test_streams_and_empty(dev):
    c = _case(dev, BF16, 200, 72, 96)
    want = _call(c, None)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = _call(c, None)
    s.synchronize()
    assert torch.equal(got, want)
    leaves = [c["x"][:0].clone().requires_grad_(True), c["w"].requires_grad_(True), torch.zeros(72, device=dev, requires_grad=True)]
    none = keep_amd.linear(*leaves, activation="silu")
    assert none.shape == (0, 72)
    dx, dw, db = torch.autograd.grad(none.sum(), leaves)
    assert dx.shape == (0, 96) and (dw == 0).all() and (db == 0).all()


@pytest.mark.parametrize("M", [4, 300])
def test_graphs(dev, M):
    names = ("x", "w", "b", "r", "dy")
    cases = [_case(dev, BF16, M, 72, 1000, bias=F32, residual=BF16, seed=s) for s in range(4)]
    c = [cases[0][n].clone() for n in names]

    def step():
        leaves = [t.detach().requires_grad_(True) for t in c[:4]]
        out = keep_amd.linear(*leaves[:3], activation="silu", residual=leaves[3])
        return [out.detach(), *torch.autograd.grad(out, leaves, c[4])]
    _replays(step, c, [[k[n] for n in names] for k in cases])


# --------------------------------------------------------------------------- 8 bits


def _q8(dev, M, N, K, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    kb, nb = (K + 127) // 128, (N + 127) // 128
    x = torch.randn(M, K, device=dev, generator=g).clamp(-3.5, 3.5).mul(100).to(torch.float8_e4m3fn)
    w = torch.randn(N, K, device=dev, generator=g).clamp(-3.5, 3.5).mul(100).to(torch.float8_e4m3fn)
    xs = (torch.rand(M, kb, device=dev, generator=g) + 0.5) / 100
    ws = (torch.rand(nb, kb, device=dev, generator=g) + 0.5) / 100 * K ** -0.5
    return x, xs, w, ws


def _q8_expected(x, xs, w, ws):
    """A block's products are exact values of 8 bits summed in float32, times two scales, the blocks added."""
    (M, K), N = x.shape, w.shape[0]
    out = Bounded(torch.zeros(M, N, device=x.device, dtype=torch.float64))
    for b in range(xs.shape[1]):
        at = slice(128 * b, min(K, 128 * b + 128))
        part = Bounded(x[:, at].float()) @ Bounded(w[:, at].float()).T
        rows = ws[:, b].repeat_interleave(128)[:N]
        scale = xs[:, b, None].double() * rows[None].double()
        out = out + Bounded(part.v * scale, (part.e + 2 * U * part.v.abs()) * scale)
    return out


@pytest.mark.parametrize("M, N, K", [(1, 16, 16), (1, 384, 4096), (3, 130, 144), (16, 257, 1024), (17, 100, 2880), (64, 384, 7168),
                                     (70, 33, 272), (129, 260, 400), (333, 640, 128), (300, 136, 1040), (3840, 4100, 144)])
def test_q8(dev, M, N, K):
    x, xs, w, ws = _q8(dev, M, N, K)
    want = _q8_expected(x, xs, w, ws)
    got = keep_amd.linear_q8(x, xs, w, ws)
    assert got.dtype == BF16
    want.round(BF16).check(got)
    b, r = torch.randn(N, device=dev), torch.randn(M, N, device=dev)
    both = Bounded(r) + _act(want + Bounded(b.expand(M, -1)), "silu")
    both.round(F32).check(keep_amd.linear_q8(x, xs, w, ws, b, activation="silu", residual=r))


def test_q8_odd_widths_and_views(dev):
    x, xs, w, ws = _q8(dev, 40, 48, 100)
    _q8_expected(x, xs, w, ws).round(F16).check(keep_amd.linear_q8(x, xs, w, ws, out_dtype=F16))
    wide = torch.zeros(40, 160, device=dev).to(torch.float8_e4m3fn)
    x, xs, w, ws = _q8(dev, 40, 48, 112)
    wide[:, 32:144] = x
    assert torch.equal(keep_amd.linear_q8(wide[:, 32:144], xs, w, ws), keep_amd.linear_q8(x, xs, w, ws))
    three = keep_amd.linear_q8(x.view(4, 10, 112), xs.view(4, 10, 1), w, ws)
    assert three.shape == (4, 10, 48)
    assert keep_amd.linear_q8(x[:0], xs[:0], w, ws).shape == (0, 48)


def test_q8_of_normed_rows(dev):
    """The norm's 8-bit rows through the 8-bit product, against the rows' values."""
    x = torch.randn(50, 512, device=dev).to(BF16)
    _, _, w, ws = _q8(dev, 1, 200, 512)
    q, s = keep_amd.rmsnorm_quant(x)
    _q8_expected(q, s, w, ws).round(BF16).check(keep_amd.linear_q8(q, s, w, ws))


def test_q8_graphs(dev):
    cases = [_q8(dev, 200, 72, 1024, seed=s) for s in range(3)]
    c = [t.clone() for t in cases[0]]
    _replays(lambda: [keep_amd.linear_q8(*c)], c, cases)
