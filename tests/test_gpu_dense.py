"""Routed products with dense expert weights (``gather_mm``), the routed combine with its gradients, and the layers on
them, against float64 with derived bounds."""

import pytest
import torch

import keep_amd
from keep_amd import ops
from tests.bounded import Bounded

pytestmark = pytest.mark.gpu
DTYPES = [torch.float32, torch.float16, torch.bfloat16]


def _case(dev, dtype, T, E, k, N, K, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(T, K, device=dev, generator=g).to(dtype)
    w = (torch.randn(E, N, K, device=dev, generator=g) * K ** -0.5).to(dtype)
    idx = torch.randint(0, E, (T, k), device=dev, generator=g, dtype=torch.int32)
    dy = torch.randn(T, k, N, device=dev, generator=g).to(dtype)
    return x, w, idx, dy


def _expected(x, w, idx, dy):
    """Output and gradients, expert by expert."""
    T, k = idx.shape
    E, N, K = w.shape
    token, expert = torch.arange(T, device=x.device).repeat_interleave(k), idx.reshape(-1).long()
    out, dxr = (Bounded(torch.zeros(T * k, n, device=x.device, dtype=torch.float64)) for n in (N, K))
    dw = Bounded(torch.zeros(E, N, K, device=x.device, dtype=torch.float64))
    dyr = dy.reshape(T * k, N)
    for e in range(E):
        at = (expert == e).nonzero()[:, 0]
        if not at.numel():
            continue
        xe, we, de = Bounded(x[token[at]]), Bounded(w[e]), Bounded(dyr[at])
        for to, what in ((out, xe @ we.T), (dxr, de @ we)):
            to.v[at], to.e[at] = what.v, what.e
        g = de.T @ xe
        dw.v[e], dw.e[e] = g.v, g.e
    dx = Bounded(dxr.v.view(T, k, K), dxr.e.view(T, k, K)).sum(1)
    return (Bounded(out.v.view(T, k, N), out.e.view(T, k, N)).round(x.dtype), dx.round(x.dtype), dw.round(w.dtype))


SHAPES = [
    (1, 1, 1, 1, 1),          # one of everything
    (1, 8, 2, 48, 64),        # a token
    (3, 5, 2, 33, 40),        # an odd number of outputs
    (7, 4, 3, 20, 17),        # rows at odd addresses
    (40, 3, 3, 64, 136),      # windows with more than 16 routes of an expert
    (130, 6, 2, 72, 128),     # a plan, ragged tiles
    (257, 2, 1, 40, 100),
    (300, 24, 4, 160, 264),
    (1100, 3, 1, 130, 72),    # hundreds of rows per expert
    (700, 2, 2, 264, 520),
    (500, 5, 2, 136, 200),    # the product through LDS, tiles of 128 routes
    (900, 3, 2, 512, 320),
    (61, 5, 8, 1024, 64),
    (2000, 40, 1, 64, 1032),
    (400, 3, 2, 8, 8),        # less than one step of the summed index
    (17000, 9, 1, 40, 72),    # a plan over several workgroups
]


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("shape", SHAPES)
def test_gather_mm_and_its_gradients(dev, dtype, shape):
    x, w, idx, dy = _case(dev, dtype, *shape)
    want = _expected(x, w, idx, dy)
    plain = keep_amd.gather_mm(x, w, idx)
    want[0].check(plain, "out")
    x.requires_grad_(True), w.requires_grad_(True)
    out = keep_amd.gather_mm(x, w, idx)
    assert torch.equal(out, plain)
    dx, dw = torch.autograd.grad(out, (x, w), dy)
    assert dx.dtype == dw.dtype == dtype
    want[1].check(dx, "dx")
    want[2].check(dw, "dw")


@pytest.mark.parametrize("R, E, tile", [(1, 1, 16), (4096, 3, 64), (4097, 1024, 64), (20000, 7, 256), (70001, 384, 16),
                                        (33000, 1, 128)])
def test_plan_over_several_workgroups(dev, R, E, tile):
    """The single workgroup's plan, array by array, routes out of range included."""
    from keep_amd import _lib
    g = torch.Generator(device=dev).manual_seed(R)
    rhs = torch.randint(-1, E + 1, (R,), device=dev, generator=g, dtype=torch.int32)
    want = ops.route_plan(rhs, E, tile)
    got = [torch.full_like(t, -7) for t in want]
    need = _lib.load().keep_route_plan_blocks_workspace_bytes(R, E)
    ws = torch.empty(need, dtype=torch.uint8, device=dev)
    order, inverse, counts, offsets, te, to, tc, nt = got
    _lib.call("keep_route_plan_blocks", rhs.data_ptr(), R, E, tile, *(t.data_ptr() for t in (order, inverse, counts,
              offsets, te, to, tc)), te.numel(), nt.data_ptr(), ws.data_ptr(), need, ops._stream(dev))
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", DTYPES)
def test_gather_mm_more_experts_than_a_plan_holds(dev, dtype):
    x, w, idx, dy = _case(dev, dtype, 300, 1030, 1, 24, 16)
    want = _expected(x, w, idx, dy)
    want[0].check(keep_amd.gather_mm(x, w, idx))
    x.requires_grad_(True)
    out = keep_amd.gather_mm(x, w, idx)
    want[1].check(torch.autograd.grad(out, x, dy)[0])
    with pytest.raises(ValueError, match="at most 1024"):
        keep_amd.gather_mm(x, w.requires_grad_(True), idx)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T", [5, 200])
def test_gather_mm_layouts(dev, dtype, T):
    """Transposed and strided weights, strided rows, and the per-route layout."""
    x, w, idx, dy = _case(dev, dtype, T, 6, 2, 40, 64)
    want = _expected(x, w, idx, dy)
    wt = w.transpose(1, 2).contiguous().transpose(1, 2)  # [E, K, N] memory
    assert not wt.is_contiguous()
    wide = torch.zeros(T, 80, device=dev, dtype=dtype)
    wide[:, 3:67] = x
    odd = torch.zeros(6, 40, 70, device=dev, dtype=dtype)
    odd[:, :, 5:69] = w
    for xv, wv in ((x, wt), (wide[:, 3:67], w), (x, odd[:, :, 5:69]), (wide[:, 3:67], wt)):
        a, b = xv.detach().requires_grad_(True), wv.detach().requires_grad_(True)
        out = keep_amd.gather_mm(a, b, idx)
        want[0].check(out, "out")
        dx, dw = torch.autograd.grad(out, (a, b), dy)
        want[1].check(dx, "dx")
        want[2].check(dw, "dw")
    lhs = torch.arange(T, device=dev).repeat_interleave(2)
    flat = keep_amd.gather_mm(x, w, idx.reshape(-1), lhs_indices=lhs)
    assert torch.equal(flat.view(T, 2, 40), keep_amd.gather_mm(x, w, idx))
    again = keep_amd.gather_mm(x, w, idx.reshape(-1).flip(0), lhs_indices=lhs.flip(0))
    want[0].check(again.flip(0).view(T, 2, 40))


@pytest.mark.parametrize("T", [4, 150])
@pytest.mark.parametrize("dtype", DTYPES)
def test_gather_mm_routes_out_of_range_and_nan(dev, dtype, T):
    x, w, idx, dy = _case(dev, dtype, T, 5, 2, 24, 40)
    idx = idx.clamp(max=3)  # expert 4 has no routes
    want = _expected(x, w, idx, dy)
    bad = idx.clone()
    bad[1, 0], bad[2, 1], bad[3, 0] = -1, 5, 2 ** 30
    w = w.clone()
    w[4] = float("nan")  # of an expert that nobody asks for
    x.requires_grad_(True), w.requires_grad_(True)
    out = keep_amd.gather_mm(x, w, bad)
    ok = (bad >= 0) & (bad < 5)
    assert torch.isnan(out[~ok]).all()
    Bounded(want[0].v[ok], want[0].e[ok]).check(out[ok])
    dx, dw = torch.autograd.grad(out, (x, w), dy)
    assert torch.isnan(dx[~ok.all(1)]).all()
    Bounded(want[1].v[ok.all(1)], want[1].e[ok.all(1)]).check(dx[ok.all(1)])
    assert (dw[4] == 0).all()
    zeroed = dy.clone()
    zeroed[~ok] = 0
    _expected(x.detach(), w.detach().nan_to_num(0), idx, zeroed)[2].check(dw, "dw")
    # a NaN in a row of x stays in that row's outputs and the weights' gradients of its experts
    xn = x.detach().clone()
    xn[0, 3] = float("nan")
    xn.requires_grad_(True)
    out = keep_amd.gather_mm(xn, w, idx)
    assert torch.isnan(out[0]).all() and torch.isfinite(out[1:]).all()
    dw = torch.autograd.grad(out, w, dy)[0]
    hit = torch.zeros(5, dtype=torch.bool, device=dev)
    hit[idx[0].long()] = True
    assert torch.isnan(dw[hit][:, :, 3]).all() and torch.isfinite(dw[~hit]).all()
    # lhs out of range
    lhs = torch.arange(T, device=dev).repeat_interleave(2)
    lhs[1], lhs[4] = -1, T
    flat = keep_amd.gather_mm(x.detach(), w.detach(), idx.reshape(-1), lhs_indices=lhs)
    assert torch.isnan(flat[[1, 4]]).all() and torch.isfinite(flat[[0, 2, 3, 5]]).all()


@pytest.mark.parametrize("dtype", DTYPES)
def test_gather_mm_empty_calls(dev, dtype):
    w = torch.randn(3, 8, 16, device=dev).to(dtype).requires_grad_(True)
    for T, k in ((0, 2), (4, 0)):
        x = torch.zeros(T, 16, device=dev, dtype=dtype, requires_grad=True)
        idx = torch.zeros(T, k, device=dev, dtype=torch.int32)
        assert keep_amd.gather_mm(x.detach(), w.detach(), idx).shape == (T, k, 8)
        out = keep_amd.gather_mm(x, w, idx)
        dx, dw = torch.autograd.grad(out, (x, w), torch.zeros_like(out))
        assert dx.shape == x.shape and (dx == 0).all() and dw.shape == w.shape and (dw == 0).all()


def test_gather_mm_a_row_does_not_depend_on_the_others(dev):
    x, w, idx, _ = _case(dev, torch.bfloat16, 60, 4, 2, 96, 256)
    full = keep_amd.gather_mm(x, w, idx)
    assert torch.equal(full, keep_amd.gather_mm(x, w, idx))
    for t in (0, 31, 59):
        assert torch.equal(keep_amd.gather_mm(x[t:t + 1], w, idx[t:t + 1])[0], full[t])


def test_gather_mm_gradients_against_differences(dev):
    """The output is linear in each operand: a difference quotient is the gradient's product, up to rounding."""
    x, w, idx, dy = _case(dev, torch.float32, 150, 5, 2, 24, 32)
    x.requires_grad_(True), w.requires_grad_(True)
    dx, dw = torch.autograd.grad(keep_amd.gather_mm(x, w, idx), (x, w), dy)
    for t, g, of in ((x, dx, lambda v: keep_amd.gather_mm(v, w.detach(), idx)),
                     (w, dw, lambda v: keep_amd.gather_mm(x.detach(), v, idx))):
        for seed in range(3):
            step = torch.randn(t.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(seed))
            with torch.no_grad():
                up, down = of(t + step).double(), of(t - step).double()
            got = ((up - down) * dy).sum() / 2
            want = (g.double() * step).sum()
            # float32 outputs of 32 products near 1, their inputs t +- step rounded too: 34 half steps of each term
            scale = ((up.abs() + down.abs()) * dy.abs()).sum() + (g.double().abs() * step.abs()).sum()
            assert abs(got - want) <= 40 * 2.0 ** -23 * 8 * scale


def test_gather_mm_beyond_32_bit_offsets(dev):
    """The last expert's weights lie past 2^31 values."""
    E, N, K = 33, 8192, 8192
    w = torch.zeros(E, N, K, device=dev, dtype=torch.bfloat16)
    x, last, idx, dy = _case(dev, torch.bfloat16, 3, 1, 1, N, K, seed=3)
    w[-1] = last[0]
    want = _expected(x, last, idx, dy)
    for T in (3, 150):  # few routes, and a plan
        xs = x.repeat(T // 3, 1)
        at = torch.full((T, 1), E - 1, device=dev, dtype=torch.int32)
        want[0].check(keep_amd.gather_mm(xs, w, at)[:3])
    xg = x.clone().requires_grad_(True)
    at = torch.full((3, 1), E - 1, device=dev, dtype=torch.int32)
    w.requires_grad_(True)
    dx, dw = torch.autograd.grad(keep_amd.gather_mm(xg, w, at), (xg, w), dy)
    want[1].check(dx)
    want[2].check(dw[-1:])
    assert (dw[:-1].abs().amax(dim=(1, 2)) == 0).all()


def test_gather_mm_rows_of_more_than_4_gib(dev):
    """x past 2^31 values: the products through LDS leave their 32-bit offsets."""
    T, K, N = 262_200, 8192, 64
    x = torch.zeros(T, K, device=dev, dtype=torch.bfloat16)
    last, w, idx, dy = _case(dev, torch.bfloat16, 40, 2, 1, N, K, seed=4)
    x[-40:] = last
    want = _expected(last, w, idx, dy)
    full = torch.zeros(T, 1, device=dev, dtype=torch.int32)
    full[-40:] = idx
    x.requires_grad_(True), w.requires_grad_(True)
    out = keep_amd.gather_mm(x, w, full)
    want[0].check(out[-40:], "out")
    assert (out[:1000] == 0).all()
    g = torch.zeros(T, 1, N, device=dev, dtype=torch.bfloat16)
    g[-40:] = dy
    dx, dw = torch.autograd.grad(out, (x, w), g)
    want[1].check(dx[-40:], "dx")
    assert (dx[:1000] == 0).all()
    want[2].check(dw, "dw")


def _replays(fn, inputs, others):
    """``fn()`` captured, replayed several times with eager work between, on changing inputs: each replay's outputs
    are the eager ones'."""
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        fn()
    torch.cuda.current_stream().wait_stream(side)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        captured = fn()
    for values in others:
        with torch.no_grad():
            for t, v in zip(inputs, values):
                t.copy_(v)
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        eager = fn()
        for a, b in zip(captured, eager):
            assert torch.equal(a, b)
        del eager
        torch.randn(1 << 20, device=inputs[0].device).sum().item()


@pytest.mark.parametrize("T", [6, 300])
def test_gather_mm_in_graphs(dev, T):
    cases = [_case(dev, torch.bfloat16, T, 6, 2, 48, 64, seed=s) for s in range(4)]
    x, w, idx, dy = (t.clone() for t in cases[0])
    _replays(lambda: [keep_amd.gather_mm(x, w, idx)], (x, w, idx), [c[:3] for c in cases])

    def step():
        a, b = x.detach().requires_grad_(True), w.detach().requires_grad_(True)  # leaves of this graph alone
        out = keep_amd.gather_mm(a, b, idx)
        return [out.detach(), *torch.autograd.grad(out, (a, b), dy)]

    _replays(step, (x, w, idx, dy), cases)


def test_capture_on_leaves_of_a_live_eager_graph_is_refused(dev):
    x, w, idx, _ = _case(dev, torch.bfloat16, 6, 6, 2, 48, 64)
    w.requires_grad_(True)
    held = keep_amd.gather_mm(x, w, idx)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(g):
            torch.zeros(1, device=dev)
            keep_amd.gather_mm(x, w, idx)
    del held
    assert torch.isfinite(keep_amd.gather_mm(x, w, idx)).all()


def test_gather_mm_on_another_stream(dev):
    x, w, idx, dy = _case(dev, torch.bfloat16, 200, 6, 2, 48, 64)
    want = keep_amd.gather_mm(x, w, idx)
    torch.cuda.synchronize()
    s = torch.cuda.Stream()
    with torch.cuda.stream(s):
        got = keep_amd.gather_mm(x, w, idx)
        leaf = w.detach().requires_grad_(True)
        dw = torch.autograd.grad(keep_amd.gather_mm(x, leaf, idx), leaf, dy)[0]
    s.synchronize()
    assert torch.equal(got, want)
    _expected(x, w, idx, dy)[2].check(dw)


# --------------------------------------------------------------------------- combine


@pytest.mark.parametrize("dtype", DTYPES)
@pytest.mark.parametrize("od", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("T, k, H", [(1, 1, 4), (3, 2, 12), (5, 6, 1024), (70, 8, 520), (0, 2, 8)])
def test_route_combine_and_its_gradients(dev, dtype, od, T, k, H):
    g = torch.Generator(device=dev).manual_seed(1)
    y = torch.randn(T, k, H, device=dev, generator=g).to(dtype)
    w = torch.rand(T, k, device=dev, generator=g)
    d = torch.randn(T, H, device=dev, generator=g).to(od)
    want = (Bounded(w[:, None]) @ Bounded(y))[:, 0].round(od)
    plain = keep_amd.route_combine(y, w, od)
    want.check(plain, "out")
    y.requires_grad_(True), w.requires_grad_(True)
    out = keep_amd.route_combine(y, w, od)
    assert torch.equal(out, plain)
    dy, dw = torch.autograd.grad(out, (y, w), d)
    Bounded(d[:, None]).times(w[:, :, None]).round(dtype).check(dy, "dy")
    (Bounded(y.detach()) @ Bounded(d[:, :, None]))[:, :, 0].round(torch.float32).check(dw, "dw")
    only = torch.autograd.grad(keep_amd.route_combine(y.detach(), w, od), w, d)[0]
    assert torch.equal(only, dw)
    only = torch.autograd.grad(keep_amd.route_combine(y, w.detach(), od), y, d)[0]
    assert torch.equal(only, dy)


def test_route_combine_reads_16_bit_rows_as_their_float_copy(dev):
    y = torch.randn(33, 6, 2048, device=dev).bfloat16()
    w = torch.rand(33, 6, device=dev)
    assert torch.equal(ops.route_combine(y, w), ops.route_combine(y.float(), w))


# --------------------------------------------------------------------------- layers


def _layer(dev, dtype, E=6, H=64, I=48, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed)

    def weight(n, m):
        return (torch.randn(E, n, m, device=dev, generator=g) * m ** -0.5).to(dtype)
    return weight(I, H), weight(I, H), weight(H, I)


@pytest.mark.parametrize("T", [1, 3, 90])
def test_dense_experts_in_the_moe_layer(dev, T):
    """Router, three dense projections, combine, shared expert and residual, forward and backward, against the same
    formulas in float64 on float32 inputs (bounded by the sizes: sums of 64 terms, three products deep)."""
    E, H, I, k = 6, 64, 48, 2
    ws = [w.requires_grad_(True) for w in _layer(dev, torch.float32)]
    glu = keep_amd.QuantizedVQSwitchGLU(**{n: keep_amd.SwitchLinear(w) for n, w in
                                           zip(("gate_proj", "up_proj", "down_proj"), ws)})
    sh = [w[:1].detach().clone().requires_grad_(True) for w in _layer(dev, torch.float32, seed=5)]
    shared = keep_amd.QuantizedVQSwitchGLU(**{n: keep_amd.SwitchLinear(w) for n, w in
                                              zip(("gate_proj", "up_proj", "down_proj"), sh)})
    moe = keep_amd.RoutedVQMoE(glu, top_k=k, shared_experts=shared)
    g = torch.Generator(device=dev).manual_seed(9)
    x = torch.randn(T, H, device=dev, generator=g).requires_grad_(True)
    res = torch.randn(T, H, device=dev, generator=g).requires_grad_(True)
    logits = torch.randn(T, E, device=dev, generator=g)
    dout = torch.randn(T, H, device=dev, generator=g)
    out, r = moe(x, logits, residual=res)
    leaves = (x, res, *ws, *sh)
    grads = torch.autograd.grad(out, leaves, dout)
    dl = [t.detach().double().requires_grad_(True) for t in leaves]
    xd, rd, (gw, uw, dw_), (sg, su, sd) = dl[0], dl[1], dl[2:5], dl[5:8]

    def expert(v, a, b, c):
        return torch.nn.functional.silu(v @ a.T) * (v @ b.T) @ c.T
    rows = [sum(r.weight[t, j].double() * expert(xd[t], gw[r.idx[t, j]], uw[r.idx[t, j]], dw_[r.idx[t, j]])
                for j in range(k)) + expert(xd[t], sg[0], su[0], sd[0]) for t in range(T)]
    ref = rd + torch.stack(rows)
    want = torch.autograd.grad(ref, dl, dout.double())
    for a, b in zip((out, *grads), (ref, *want)):
        # each of about six chained operations of up to T + 64 float32 terms: (T + 64) 2^-24 of the largest value's size
        tol = 6 * (T + 64) * 2.0 ** -24 * max(1.0, b.abs().max().item()) * 8
        assert (a.double() - b).abs().max().item() <= tol


def test_dense_and_code_projections_side_by_side(dev):
    """Codes for gate and up, dense weights for down: each projection's own operator, in the layer's order."""
    from keep_amd import synth
    import numpy as np
    E, H, I, k, T = 4, 512, 256, 2, 5

    def codes(n, m, seed):
        c, s = synth.projection_np(E, n, m, seed=seed)[:2]
        return keep_amd.QuantizedVQSwitchLinear(
            input_dims=m, output_dims=n, num_experts=E, codes=torch.from_numpy(c.view(np.int16)).to(dev),
            scales=torch.from_numpy(s).to(dev), group_size=m // s.shape[-1], code_bits=16)
    gate, up = codes(I, H, 1), codes(I, H, 2)
    w = (torch.randn(E, H, I, device=dev) * I ** -0.5).half()
    glu = keep_amd.QuantizedVQSwitchGLU(gate_proj=gate, up_proj=up, down_proj=keep_amd.SwitchLinear(w))
    x = torch.randn(T, H, device=dev).half()
    idx = torch.randint(0, E, (T, k), device=dev, dtype=torch.int32)
    y = glu(x, idx)
    h = torch.nn.functional.silu(gate(x, idx)) * up(x, idx)
    assert torch.equal(y, keep_amd.gather_mm(h.reshape(T * k, I), w, idx.reshape(-1, 1)).reshape(T, k, H))
    with pytest.raises(ValueError, match="no gradient"):
        glu(x.clone().requires_grad_(True), idx)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_switch_linear_layouts_and_bias(dev, dtype):
    w = torch.randn(4, 24, 32, device=dev).to(dtype)
    b = torch.randn(4, 24, device=dev).to(dtype)
    lin = keep_amd.SwitchLinear(w, b)
    x = torch.randn(2, 3, 32, device=dev).to(dtype)
    idx = torch.randint(0, 4, (2, 3, 2), device=dev, dtype=torch.int32)
    y = lin(x, idx)
    for i in range(2):
        assert torch.equal(lin(x, idx[..., i]), y[:, :, i])
    flat = keep_amd.gather_mm(x.reshape(6, 32), w, idx.reshape(6, 2)).view(2, 3, 2, 24)
    assert torch.equal(y, flat + b[idx.long()])


@pytest.mark.parametrize("between", [lambda w: w.bfloat16(), lambda w: (w * 2).bfloat16().transpose(1, 2).contiguous().mT])
def test_capture_is_refused_through_a_cast_too(dev, between):
    x, w, idx, _ = _case(dev, torch.float32, 6, 6, 2, 48, 64)
    x, master = x.bfloat16(), w.requires_grad_(True)
    held = keep_amd.gather_mm(x, between(master), idx)
    g = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="eager graph"):
        with torch.cuda.graph(g):
            torch.zeros(1, device=dev)
            keep_amd.gather_mm(x, between(master), idx)
    del held
    assert torch.isfinite(keep_amd.gather_mm(x, between(master), idx)).all()


@pytest.mark.parametrize("transposed", [False, True])
def test_gather_mm_more_tiles_than_a_launch_has_blocks_along_an_axis(dev, transposed):
    g = torch.Generator(device=dev).manual_seed(2)
    T, E, N, K = 70_001, 1100, 12, 8  # no plan holds 1100 experts: a tile per route at most
    x = torch.randint(-4, 5, (T, K), device=dev, generator=g).float()
    w = torch.randint(-4, 5, (E, N, K), device=dev, generator=g).float()
    idx = torch.randint(0, E, (T, 1), device=dev, generator=g).int()
    if transposed:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    want = (w[idx[:, 0].long()] * x[:, None]).sum(2)  # whole numbers: exact in any order
    assert torch.equal(keep_amd.gather_mm(x, w, idx)[:, 0], want)


def test_route_combine_gradients_of_more_routes_than_a_launch_has_waves(dev):
    T = (1 << 25) + 5
    y = torch.arange(T * 4, device=dev).remainder(7).half().view(T, 1, 4).requires_grad_(True)
    w = torch.arange(T, device=dev).remainder(5).float().view(T, 1).requires_grad_(True)
    d = torch.arange(T * 4, device=dev).remainder(3).half().view(T, 4)
    dy, dw = torch.autograd.grad(keep_amd.route_combine(y, w, torch.float16), (y, w), d)
    assert torch.equal(dy[:, 0], d * w.detach().half())  # whole numbers below 2048
    assert torch.equal(dw[:, 0], (y.detach()[:, 0].float() * d.float()).sum(1))
