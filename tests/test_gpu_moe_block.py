"""Norm, gate, choice, experts, shared expert and combine as one feed-forward block, trained and served.

In float32 every step's sums run over at most 96 terms, 5 products behind each other and a norm before them: 5 x 96 x 2^-23 of
the terms' magnitudes, under 2^-14; 2^-12 of an output's largest value leaves four times as much for sums that cancel."""

import pytest
import torch

import keep_amd
from keep_amd import synth
from tests.test_gpu_dense import _replays

pytestmark = pytest.mark.gpu
NEAR = 2.0 ** -12


def _params(dev, E=8, H=96, I=48, seed=0, dtype=torch.float32):
    g = torch.Generator(device=dev).manual_seed(seed)

    def normal(*shape, std):
        return (torch.randn(*shape, device=dev, generator=g) * std).to(dtype)
    p = {"norm": 1 + normal(H, std=0.2), "gate": normal(E, H, std=H ** -0.5)}
    for where, lead in (("e", (E,)), ("s", ())):
        p[where + "_gate"], p[where + "_up"] = (normal(*lead, I, H, std=H ** -0.5) for _ in range(2))
        p[where + "_down"] = normal(*lead, H, I, std=I ** -0.5)
    return p


def _block(p, k=3, **kw):
    glu = keep_amd.QuantizedVQSwitchGLU(**{n + "_proj": keep_amd.SwitchLinear(p["e_" + n]) for n in ("gate", "up", "down")})
    shared = keep_amd.DenseGLU(**{n + "_proj": keep_amd.DenseLinear(p["s_" + n]) for n in ("gate", "up", "down")})
    gate = keep_amd.MoEGate(p["gate"], top_k=k, **kw)
    return keep_amd.RoutedVQMoE(glu, top_k=k, gate=gate, shared_experts=shared, out_dtype=torch.float32)


def _run(p, x, res, **kw):
    y, h = keep_amd.rmsnorm(x, p["norm"], residual=res)
    out, routes = _block(p, **kw)(y, residual=h)
    return out, routes


def _expected(p, x, res, idx, renormalize=True, score="sigmoid"):
    """In 64 bits, with the experts that were chosen."""
    h = res + x
    y = h / torch.sqrt((h * h).mean(-1, keepdim=True) + 1e-6) * p["norm"]
    z = y @ p["gate"].T
    s = (torch.sigmoid(z) if score == "sigmoid" else torch.softmax(z, 1)).gather(1, idx.long())
    w = s / s.sum(1, keepdim=True) if renormalize else s
    silu = torch.nn.functional.silu
    out = h + (silu(y @ p["s_gate"].T) * (y @ p["s_up"].T)) @ p["s_down"].T
    for j in range(idx.shape[1]):
        e = idx[:, j].long()
        g, u = (torch.bmm(p["e_" + n][e], y[:, :, None])[:, :, 0] for n in ("gate", "up"))
        out = out + w[:, j, None] * torch.bmm(p["e_down"][e], (silu(g) * u)[:, :, None])[:, :, 0]
    return out


KW = dict(score_func="sigmoid", groups=4, topk_groups=2, count_load=True)


@pytest.mark.parametrize("T", [1, 5, 70, 300])
def test_training_step(dev, T):
    p = _params(dev)
    g = torch.Generator(device=dev).manual_seed(T)
    x, res, dy = (torch.randn(T, 96, device=dev, generator=g) for _ in range(3))
    bias = torch.randn(8, device=dev, generator=g) * 0.05
    names = [*p, "x", "res"]
    leaves = [t.clone().requires_grad_(True) for t in (*p.values(), x, res)]
    q = dict(zip(names, leaves))
    out, routes = _run(q, q["x"], q["res"], bias=bias, **KW)
    grads = torch.autograd.grad(out, leaves, dy)
    assert int(routes.load.sum()) == 3 * T
    wide = [t.detach().double().requires_grad_(True) for t in leaves]
    w = dict(zip(names, wide))
    want = _expected(w, w["x"], w["res"], routes.idx)
    logits = torch.sigmoid((keep_amd.rmsnorm(x, p["norm"], residual=res)[0].double() @ p["gate"].double().T)) + bias.double()
    top = torch.sort(logits.view(T, 4, 2).sum(2), dim=1, descending=True).values
    sure = top[:, 1] - top[:, 2] > 1e-4  # the groups that are compared do not lie within float32's rounding of the logits
    chosen = torch.zeros(T, 8, dtype=torch.bool, device=dev).scatter_(1, routes.idx.long(), True)
    kept = chosen.view(T, 4, 2).any(2)
    best = torch.argsort(logits.view(T, 4, 2).sum(2), dim=1, descending=True)[:, :2]
    assert (torch.zeros_like(kept).scatter_(1, best, True) | ~kept)[sure].all()
    assert ((out.double() - want).abs().max() <= NEAR * want.abs().max())
    for name, got, ref in zip(names, grads, torch.autograd.grad(want, wide, dy.double())):
        assert got.shape == ref.shape
        assert (got.double() - ref).abs().max() <= NEAR * ref.abs().max(), name


def test_training_step_in_a_graph(dev):
    p = _params(dev)
    names = list(p)

    def inputs(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        return [torch.randn(40, 96, device=dev, generator=g) for _ in range(3)]
    c = [*(t.clone() for t in p.values()), *inputs(0)]

    def step():
        leaves = [t.detach().requires_grad_(True) for t in c[:-1]]
        out, routes = _run(dict(zip(names, leaves)), *leaves[-2:], **KW)
        return [out.detach(), routes.idx, routes.load, *torch.autograd.grad(out, leaves, c[-1])]
    _replays(step, c, [[*_params(dev, seed=s).values(), *inputs(s)] for s in range(3)])


def test_gate_over_experts_in_codes(dev):
    """Served through the layers on codes; the gate's weight trains while the input needs no gradient."""
    E, H, I, k = 8, 512, 256, 2
    to = lambda a: torch.from_numpy(a.view("int16") if a.dtype.name == "uint16" else a).to(dev)  # noqa: E731

    def proj(n, i, seed):
        codes, scales = synth.projection_np(E, n, i, seed=seed)
        return keep_amd.QuantizedVQSwitchLinear(input_dims=i, output_dims=n, num_experts=E, codes=to(codes),
                                                scales=to(scales), group_size=i, code_bits=16)
    glu = keep_amd.QuantizedVQSwitchGLU(gate_proj=proj(I, H, 1), up_proj=proj(I, H, 2), down_proj=proj(H, I, 3))
    weight = torch.randn(E, H, device=dev) * H ** -0.5
    for T in (1, 4, 40, 200):
        x = synth.rht_activations(T, H, seed=T, device=dev)
        moe = keep_amd.RoutedVQMoE(glu, top_k=k, gate=keep_amd.MoEGate(weight, top_k=k))
        out, routes = moe(x)
        logits = keep_amd.linear(x.float(), weight)
        by_hand, r = keep_amd.RoutedVQMoE(glu, top_k=k)(x, logits)
        assert torch.equal(routes.idx, r.idx)
        assert (out - by_hand).abs().max() <= 2e-3 * by_hand.abs().max()  # another path of the same layer: its own tolerance
        leaf = weight.clone().requires_grad_(True)
        trained, _ = keep_amd.RoutedVQMoE(glu, top_k=k, gate=keep_amd.MoEGate(leaf, top_k=k))(x)
        assert (trained.detach() - out).abs().max() <= 2e-3 * out.abs().max()
        g, = torch.autograd.grad(trained.sum(), leaf)
        assert torch.isfinite(g).all() and g.abs().max() > 0
        with pytest.raises(RuntimeError, match="no gradient"):
            xg = x.clone().requires_grad_(True)
            keep_amd.RoutedVQMoE(glu, top_k=k, gate=keep_amd.MoEGate(leaf, top_k=k))(xg)[0].sum().backward()


def test_eight_bit_serving_of_a_dense_expert(dev):
    """Normed rows in 8 bits through an 8-bit projection, against the 16-bit ones: each operand off by half a step of e4m3."""
    g = torch.Generator(device=dev).manual_seed(0)
    x, res = (torch.randn(33, 512, device=dev, generator=g).to(torch.bfloat16) for _ in range(2))
    w = torch.randn(256, 512, device=dev, generator=g) * 512 ** -0.5
    scale = w.view(2, 128, 4, 128).abs().amax((1, 3)) / 448
    each = scale.repeat_interleave(128, 0).repeat_interleave(128, 1)
    wq = (w / each).to(torch.float8_e4m3fn)
    q, s, h = keep_amd.rmsnorm_quant(x, residual=res)
    got = keep_amd.linear_q8(q, s, wq, scale, out_dtype=torch.float32).double()
    y, h16 = keep_amd.rmsnorm(x, residual=res)
    assert torch.equal(h, h16)
    want = y.double() @ w.double().T
    bound = (2 * 2.0 ** -4 + 2.0 ** -8 + 2.0 ** -8) * (y.double().abs() @ w.double().abs().T) + 2.0 ** -6
    assert ((got - want).abs() <= bound).all()


def test_update_bias(dev):
    gate = keep_amd.MoEGate(torch.randn(4, 64, device=dev), top_k=1, bias=torch.zeros(4, device=dev))
    gate.update_bias(torch.tensor([10, 2, 4, 4], dtype=torch.int32, device=dev), 0.5)
    assert gate.bias.tolist() == [-0.5, 0.5, 0.5, 0.5]
    x = torch.randn(500, 64, device=dev)
    gate.count_load = True
    first = gate(x).load
    for _ in range(60):
        gate.update_bias(gate(x).load, 0.02)
    last = gate(x).load
    assert int(last.sum()) == 500 and last.max() - last.min() < first.max() - first.min()
