"""Low-rank adapters of many requests (``gather_lora``, ``LoraAdapters``) against float64 with derived bounds."""

import pytest
import torch

import keep_amd
from tests.bounded import Bounded
from tests.test_gpu_dense import _replays

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _case(dev, dtype, T, k, n, r, K, N, seed=0, runs=False):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std=1.0):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(dtype)
    shape = (T, k) if k else (T,)
    idx = torch.randint(-1, n, shape, device=dev, generator=g, dtype=torch.int32)
    if runs:
        idx = torch.sort(idx, dim=0).values
    return {"x": normal(T, K), "a": normal(n, r, K, std=K ** -0.5), "b": normal(n, N, r, std=r ** -0.5), "idx": idx,
            "base": normal(*shape, N), "scales": torch.rand(n, device=dev, generator=g) + 0.5, "dy": normal(*shape, N)}


def _low(t, dtype):
    """The low-rank rows as they enter the second product: 16-bit values of rows scaled to [1, 2) at most, so smaller
    ones are off by at most fp16's smallest subnormal's half of twice the row's largest."""
    if dtype == torch.float32:
        return t
    top = (t.v.abs() + t.e).amax(-1, keepdim=True)
    return t.round(dtype, floor=2.0 ** -24 * top)


def _expected(c):
    x, a, b, idx = c["x"], c["a"], c["b"], c["idx"]
    dtype, n = x.dtype, a.shape[0]
    k = idx.shape[1] if idx.ndim == 2 else 1
    T, (K, N) = x.shape[0], (x.shape[1], b.shape[1])
    flat, token = idx.reshape(-1).long(), torch.arange(T, device=x.device).repeat_interleave(k)
    zero = lambda *s: Bounded(torch.zeros(*s, device=x.device, dtype=torch.float64))  # noqa: E731
    out, dxr = zero(T * k, N), zero(T * k, K)
    da, db = zero(*a.shape), zero(*b.shape)
    dy = c["dy"].reshape(T * k, N)
    for e in range(n):
        at = (flat == e).nonzero()[:, 0]
        if not at.numel():
            continue
        xe, ae, be, de = Bounded(x[token[at]]), Bounded(a[e]), Bounded(b[e]), Bounded(dy[at])
        s = c["scales"][e] if c["scales"] is not None else torch.ones((), device=x.device)
        t = (xe @ ae.T).times(s)
        dt = (de @ be).times(s)
        for to, what in ((out, _low(t, dtype) @ be.T), (dxr, _low(dt, dtype) @ ae)):
            to.v[at], to.e[at] = what.v, what.e
        for to, what in ((da, dt.T @ xe), (db, de.T @ t)):
            to.v[e], to.e[e] = what.v, what.e
    if c["base"] is not None:
        out = out + Bounded(c["base"].reshape(T * k, N))
    od = c["base"].dtype if c["base"] is not None else dtype
    dx = Bounded(dxr.v.view(T, k, K), dxr.e.view(T, k, K)).sum(1)
    shape = (*idx.shape, N)
    out = out.round(od)
    return (Bounded(out.v.view(shape), out.e.view(shape)), dx.round(dtype), da.round(dtype), db.round(dtype))


def _call(c):
    return keep_amd.gather_lora(c["x"], c["a"], c["b"], c["idx"], base=c["base"], scales=c["scales"])


def _check(c):
    want = _expected(c)
    plain = _call(c)
    want[0].check(plain, "out")
    leaves = [c[n].requires_grad_(True) for n in ("x", "a", "b")]
    out = _call(c)
    assert torch.equal(out, plain)
    for g, w, name in zip(torch.autograd.grad(out, leaves, c["dy"]), want[1:], ("dx", "da", "db")):
        assert g.dtype == c["x"].dtype
        w.check(g, name)


SHAPES = [
    (1, 0, 1, 1, 1, 1),
    (1, 0, 4, 16, 128, 96),       # a token
    (5, 0, 3, 8, 64, 80),
    (7, 0, 2, 3, 33, 17),         # nothing aligned
    (64, 0, 40, 16, 256, 200),    # a request per row
    (150, 0, 3, 24, 136, 72),     # windows, more than 16 rows of an adapter
    (300, 0, 5, 64, 96, 520),     # blocks of 16 positions
    (200, 0, 2, 100, 72, 64),
    (33, 0, 4, 128, 520, 40),
    (40, 3, 12, 16, 64, 48),      # an adapter per route
    (300, 4, 24, 8, 72, 40),      # planned
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gather_lora_and_its_gradients(dev, dtype, shape):
    _check(_case(dev, dtype, *shape))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gather_lora_runs_of_rows(dev, dtype):
    _check(_case(dev, dtype, 700, 0, 4, 16, 256, 128, runs=True))


@pytest.mark.parametrize("dtype", DTYPES)
def test_gather_lora_without_base_or_scales(dev, dtype):
    c = _case(dev, dtype, 50, 0, 3, 16, 64, 80)
    _check({**c, "base": None, "scales": None})


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_gather_lora_float_base(dev, dtype):
    """A float32 base keeps its bits; the rows' gradients take the output's gradient in their own type."""
    c = _case(dev, dtype, 50, 0, 3, 16, 64, 80)
    c["base"] = c["base"].float() + 2.0 ** -20
    want = _expected(c)
    got = _call(c)
    assert got.dtype == torch.float32
    want[0].check(got)
    base = c["base"].requires_grad_(True)
    x = c["x"].requires_grad_(True)
    dx, dbase = torch.autograd.grad(_call(c), (x, base), c["dy"].float())
    assert torch.equal(dbase, c["dy"].float())  # dy is exact in 16 bits here
    want[1].check(dx)


def test_gather_lora_large_rows_stay_in_fp16(dev):
    """Low-rank rows beyond fp16's largest value (65504) whose second product brings them back."""
    c = _case(dev, torch.float16, 40, 0, 2, 16, 4096, 64)
    c["a"] = (c["a"].float() * 4096).half()  # t near 4096 * 64 = 2^18
    c["x"] = (c["x"].float() * 64).half()
    c["b"] = (c["b"].float() * 2.0 ** -12).half()
    want = _expected(c)
    assert want[0].v.abs().max() < 60000
    want[0].check(_call(c))


@pytest.mark.parametrize("k", [0, 3])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gather_lora_no_adapter_and_out_of_range(dev, dtype, k):
    c = _case(dev, dtype, 24, k, 4, 8, 64, 48)
    idx = c["idx"]
    idx[5], idx[7], idx[9] = -1, -(2 ** 31), 4
    idx[11] = 2 ** 31 - 1
    got = _call(c)
    assert torch.equal(got[[5, 7]], c["base"][[5, 7]])
    assert torch.isnan(got[[9, 11]]).all()
    keep = torch.ones(24, dtype=torch.bool, device=dev)
    keep[[9, 11]] = False
    want = _expected(c)[0]
    Bounded(want.v[keep], want.e[keep]).check(got[keep])
    none = keep_amd.gather_lora(c["x"], c["a"], c["b"], torch.full_like(idx, -1))
    assert (none == 0).all()
    # rows without an adapter: no gradient of x, no share in the factors'
    x = c["x"].clone().requires_grad_(True)
    c2 = {**c, "x": x, "idx": torch.full_like(idx, -1)}
    a = c["a"].clone().requires_grad_(True)
    dx, da = torch.autograd.grad(_call({**c2, "a": a}), (x, a), c["dy"])
    assert (dx == 0).all() and (da == 0).all()
    # NaN in an adapter nobody asks for, and in the base of one row
    b = c["b"].clone()
    b[3] = float("nan")
    base = c["base"].clone()
    base[2] = float("nan")
    safe = idx.clamp(-1, 2)
    got = keep_amd.gather_lora(c["x"], c["a"], b, safe, base=base, scales=c["scales"])
    assert torch.isnan(got[2]).all() and torch.isfinite(got[torch.arange(24, device=dev) != 2]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gather_lora_empty_calls(dev, dtype):
    c = _case(dev, dtype, 4, 0, 3, 8, 32, 16)
    for idx in (torch.zeros(0, device=dev, dtype=torch.int32), torch.zeros(0, 2, device=dev, dtype=torch.int32)):
        x = c["x"][:0].clone().requires_grad_(True)
        a, b = (c[n].clone().requires_grad_(True) for n in "ab")
        out = keep_amd.gather_lora(x, a, b, idx)
        assert out.shape == (*idx.shape, 16)
        dx, da, db = torch.autograd.grad(out, (x, a, b), torch.zeros_like(out))
        assert dx.shape == x.shape and (da == 0).all() and (db == 0).all()


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_gather_lora_strides_and_more_adapters_than_a_plan_holds(dev, dtype):
    c = _case(dev, dtype, 530, 2, 1100, 4, 40, 24)
    want = _expected(c)
    want[0].check(_call(c))
    v = dict(c)
    v["x"] = torch.cat([c["x"], c["x"]], 1)[:, :40]
    v["a"] = c["a"].transpose(1, 2).contiguous().transpose(1, 2)
    v["b"] = torch.stack([c["b"], c["b"]], -1)[..., 0]
    v["base"] = torch.cat([c["base"], c["base"]], 2)[:, :, :24]
    assert torch.equal(_call(v), _call(c))
    x = c["x"].clone().requires_grad_(True)
    want[1].check(torch.autograd.grad(_call({**c, "x": x}), x, c["dy"])[0])
    with pytest.raises(ValueError, match="at most 1024"):
        _call({**c, "a": c["a"].clone().requires_grad_(True)})


def test_gather_lora_gradients_against_differences(dev):
    c = _case(dev, torch.float32, 60, 2, 4, 8, 32, 24)
    leaves = {n: c[n].requires_grad_(True) for n in ("x", "a", "b", "base")}
    grads = dict(zip(leaves, torch.autograd.grad(_call(c), list(leaves.values()), c["dy"])))
    for name, t in leaves.items():
        step = torch.randn(t.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(2))
        with torch.no_grad():
            up, down = (_call({**c, name: t + s * step}).double() for s in (1, -1))
        got = ((up - down) * c["dy"]).sum() / 2
        want = (grads[name].double() * step).sum()
        # linear in each operand; float32 rows of up to 32 + 8 + 1 chained terms near 1
        scale = ((up.abs() + down.abs()) * c["dy"].abs()).sum() + (grads[name].double().abs() * step.abs()).sum()
        assert abs(got - want) <= 48 * 2.0 ** -23 * 8 * scale


def test_gather_lora_beyond_32_bit_offsets(dev):
    """The last rows of base and out lie past 2^31 values."""
    T, N = 270_000, 8192
    base = torch.zeros(T, N, device=dev, dtype=torch.bfloat16)
    c = _case(dev, torch.bfloat16, 20, 0, 3, 16, 64, N)
    base[-20:] = c["base"]
    x = torch.zeros(T, 64, device=dev, dtype=torch.bfloat16)
    x[-20:] = c["x"]
    idx = torch.full((T,), -1, device=dev, dtype=torch.int32)
    idx[-20:] = c["idx"]
    got = keep_amd.gather_lora(x, c["a"], c["b"], idx, base=base, scales=c["scales"])
    _expected(c)[0].check(got[-20:])
    assert (got[:1000] == 0).all()


@pytest.mark.parametrize("T, k", [(3, 0), (300, 2)])
def test_gather_lora_in_graphs(dev, T, k):
    cases = [_case(dev, torch.bfloat16, T, k, 5, 16, 64, 48, seed=s) for s in range(4)]
    names = ("x", "a", "b", "idx", "base", "scales", "dy")
    c = {n: cases[0][n].clone() for n in names}
    values = [[o[n] for n in names] for o in cases]
    _replays(lambda: [_call(c)], [c[n] for n in names], values)

    def step():
        leaf = {n: c[n].detach().requires_grad_(True) for n in ("x", "a", "b")}
        out = _call({**c, **leaf})
        return [out.detach(), *torch.autograd.grad(out, list(leaf.values()), c["dy"])]

    _replays(step, [c[n] for n in names], values)


# --------------------------------------------------------------------------- layers


def test_adapters_of_a_code_projection(dev):
    """A dense VQ projection with an input RHT: the adapters see the untransformed rows."""
    g = torch.Generator(device=dev).manual_seed(4)
    w = torch.randn(96, 512, device=dev, generator=g) * 512 ** -0.5
    signs = (torch.randint(0, 2, (512,), device=dev, generator=g) * 2 - 1).float()
    plain = keep_amd.QuantizedVQLinear.from_weights(w, group_size=512, rht_signs=signs)
    c = _case(dev, torch.bfloat16, 9, 0, 4, 16, 512, 96)
    ad = keep_amd.LoraAdapters(c["a"], c["b"], c["scales"])
    layer = keep_amd.QuantizedVQLinear(input_dims=512, output_dims=96, codes=plain.codes, scales=plain.scales,
                                       codebook=plain.codebook, group_size=plain.group_size, code_bits=plain.code_bits,
                                       rht_signs=signs, adapters=ad)
    base = plain(c["x"])
    assert torch.equal(layer(c["x"]), base)
    got = layer(c["x"].view(3, 3, 512), c["idx"].view(3, 3))
    assert torch.equal(got.view(9, 96), _call({**c, "base": base}))
    row = layer(c["x"][2], c["idx"][2])
    assert torch.equal(row, _call({**{n: v[2:3] if n in ("x", "idx") else v for n, v in c.items()},
                                   "base": plain(c["x"][2])[None]})[0])
    # the adapters train on it, its input does not
    a = c["a"].clone().requires_grad_(True)
    train = keep_amd.QuantizedVQLinear(input_dims=512, output_dims=96, codes=plain.codes, scales=plain.scales,
                                       codebook=plain.codebook, group_size=plain.group_size, code_bits=plain.code_bits,
                                       rht_signs=signs, adapters=keep_amd.LoraAdapters(a, c["b"], c["scales"]))
    da = torch.autograd.grad(train(c["x"], c["idx"]), a, c["dy"])[0]
    _expected({**c, "base": base})[2].check(da)
    with pytest.raises(ValueError, match="no gradient"):
        train(c["x"].clone().requires_grad_(True), c["idx"])


@pytest.mark.parametrize("T", [2, 200])
def test_adapters_of_routed_experts(dev, T):
    """Adapters on all three projections of a dense-expert layer, forward and gradients, against the operators composed
    by hand; a token without an adapter gets the layer's own output."""
    E, H, I, k, n, r = 4, 64, 48, 2, 3, 8
    g = torch.Generator(device=dev).manual_seed(T)

    def normal(*s, std=1.0):
        return torch.randn(*s, device=dev, generator=g) * std
    ws = {"gate": normal(E, I, H, std=0.125), "up": normal(E, I, H, std=0.125), "down": normal(E, H, I, std=0.14)}
    fa = {p: normal(n, E, r, w.shape[2], std=0.1).requires_grad_(True) for p, w in ws.items()}
    fb = {p: normal(n, E, w.shape[1], r, std=0.3).requires_grad_(True) for p, w in ws.items()}
    sc = torch.rand(n, device=dev, generator=g) + 0.5

    def glu(with_adapters):
        return keep_amd.QuantizedVQSwitchGLU(**{
            p + "_proj": keep_amd.SwitchLinear(w, adapters=keep_amd.LoraAdapters(fa[p], fb[p], sc)
                                               if with_adapters else None) for p, w in ws.items()})
    moe, bare = (keep_amd.RoutedVQMoE(glu(f), top_k=k) for f in (True, False))
    x, logits = normal(T, H), normal(T, E)
    ad = torch.randint(-1, n, (T,), device=dev, generator=g, dtype=torch.int32)
    ad[0] = -1
    out, route = moe(x, logits, adapter_indices=ad)
    plain, _ = bare(x, logits)
    assert torch.equal(moe(x, logits)[0], plain)
    assert torch.equal(out[ad < 0], plain[ad < 0])
    leaves = [*fa.values(), *fb.values()]
    dout = normal(T, H)
    grads = torch.autograd.grad(out, leaves, dout)
    dl = {id(t): t.detach().double().requires_grad_(True) for t in leaves}

    def proj(p, v, t, e):
        y = v @ ws[p][e].double().T
        a = int(ad[t])
        if a < 0:
            return y
        return y + sc[a].double() * (v @ dl[id(fa[p])][a, e].T) @ dl[id(fb[p])][a, e].T
    rows = []
    for t in range(T):
        v, acc = x[t].double(), 0
        for j in range(k):
            e = int(route.idx[t, j])
            h = torch.nn.functional.silu(proj("gate", v, t, e)) * proj("up", v, t, e)
            acc = acc + route.weight[t, j].double() * proj("down", h, t, e)
        rows.append(acc)
    ref = torch.stack(rows)
    want = torch.autograd.grad(ref, [dl[id(t)] for t in leaves], dout.double())
    for a, b in zip((out, *grads), (ref, *want)):
        # about eight chained operations of up to T + 64 float32 terms
        tol = 8 * (T + 64) * 2.0 ** -24 * max(1.0, b.abs().max().item()) * 8
        assert (a.double() - b).abs().max().item() <= tol


def test_adapters_on_code_experts_in_the_layer(dev):
    from keep_amd import synth
    import numpy as np
    E, H, I, k, T = 4, 512, 256, 2, 3
    fa = torch.randn(2, E, 4, H, device=dev).half() * 0.05
    fb = torch.randn(2, E, I, 4, device=dev).half() * 0.3

    def codes(n, m, seed, adapters=None):
        c, s = synth.projection_np(E, n, m, seed=seed)[:2]
        return keep_amd.QuantizedVQSwitchLinear(
            input_dims=m, output_dims=n, num_experts=E, codes=torch.from_numpy(c.view(np.int16)).to(dev),
            scales=torch.from_numpy(s).to(dev), group_size=m // s.shape[-1], code_bits=16, adapters=adapters)
    glu = keep_amd.QuantizedVQSwitchGLU(gate_proj=codes(I, H, 1, keep_amd.LoraAdapters(fa, fb)), up_proj=codes(I, H, 2),
                                        down_proj=codes(H, I, 3))
    moe = keep_amd.RoutedVQMoE(glu, top_k=k)
    x, logits = torch.randn(T, H, device=dev).half(), torch.randn(T, E, device=dev)
    ad = torch.tensor([1, -1, 0], device=dev)
    out, r = moe(x, logits, adapter_indices=ad)
    g, u, d = glu.gate_proj, glu.up_proj, glu.down_proj
    gate = g(x, r.idx)
    flat = torch.where(ad[:, None] < 0, -1, ad[:, None] * E + r.idx)
    gate = keep_amd.gather_lora(x, fa.flatten(0, 1), fb.flatten(0, 1), flat, base=gate)
    y = d(torch.nn.functional.silu(gate) * u(x, r.idx), r.idx)
    assert torch.equal(out, keep_amd.route_combine(y, r.weight))
