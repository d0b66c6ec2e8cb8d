"""What the norm, the choice of experts and the dense projections refuse, on the CPU: before any launch."""

import pytest
import torch

import keep_amd
from keep_amd import _lib, block, ops, router


def _refused(name, args, over, msg):
    assert not set(over) - set(args)
    assert getattr(_lib.load(), name)(*{**args, **over}.values()) == _lib.KEEP_EINVAL
    assert msg in _lib.load().keep_last_error().decode()


NORM = dict(x=16, dt=2, res=16, rdt=2, T=4, n=64, w=16, wdt=2, eps=1e-6, h=16, y=16, rstd=None, stream=None)
QUANT = dict(x=16, dt=2, res=16, rdt=2, T=4, n=64, w=16, wdt=2, eps=1e-6, block=128, pow2=0, h=16, q=16, scales=16, stream=None)
NORM_GRAD = dict(h=16, hdt=2, dy=16, dydt=2, dh=None, rstd=16, T=4, n=64, w=16, wdt=2, dx=16, dres=16, dw=16, ws=16,
                 ws_bytes=1 << 20, stream=None)


@pytest.mark.parametrize("over, msg", [
    (dict(dt=3), "dtype"), (dict(wdt=-1), "dtype"), (dict(rdt=1), "x's dtype or float32"), (dict(n=0), "1..16384"),
    (dict(n=16385), "1..16384"), (dict(T=-1), "2^31"), (dict(T=1 << 31), "2^31"), (dict(eps=-1.0), "eps"),
    (dict(eps=float("nan")), "eps"), (dict(x=None), "null"), (dict(h=None), "null"), (dict(res=None), "null"),
    (dict(x=17), "misaligned"), (dict(h=17), "misaligned"), (dict(w=15), "misaligned"),
])
def test_norm_entries_refuse(over, msg):
    _refused("keep_rmsnorm", NORM, over, msg)
    _refused("keep_rmsnorm_quant", QUANT, over, msg)


@pytest.mark.parametrize("name, args, over, msg", [
    ("keep_rmsnorm", NORM, dict(y=None), "null"), ("keep_rmsnorm", NORM, dict(rstd=2), "misaligned"),
    ("keep_rmsnorm_quant", QUANT, dict(block=8), "power of two"), ("keep_rmsnorm_quant", QUANT, dict(block=96), "power of two"),
    ("keep_rmsnorm_quant", QUANT, dict(block=1024), "power of two"), ("keep_rmsnorm_quant", QUANT, dict(q=None), "null"),
    ("keep_rmsnorm_quant", QUANT, dict(scales=None), "null"), ("keep_rmsnorm_quant", QUANT, dict(scales=18), "misaligned"),
    ("keep_rmsnorm_grad", NORM_GRAD, dict(hdt=1), "dy's dtype or float32"), ("keep_rmsnorm_grad", NORM_GRAD, dict(dydt=5), "dtype"),
    ("keep_rmsnorm_grad", NORM_GRAD, dict(rstd=None), "null"), ("keep_rmsnorm_grad", NORM_GRAD, dict(w=None), "null"),
    ("keep_rmsnorm_grad", NORM_GRAD, dict(dx=None, dres=None, dw=None), "null"),
    ("keep_rmsnorm_grad", NORM_GRAD, dict(ws=None), "workspace"), ("keep_rmsnorm_grad", NORM_GRAD, dict(ws_bytes=8), "workspace"),
    ("keep_rmsnorm_grad", NORM_GRAD, dict(dh=17), "misaligned"), ("keep_rmsnorm_grad", NORM_GRAD, dict(n=20000), "1..16384"),
])
def test_norm_entry_refuses(name, args, over, msg):
    _refused(name, args, over, msg)


ROUTE = dict(z=16, dt=0, T=4, E=64, k=4, bias=None, groups=8, topk_groups=2, func=0, renorm=1, scale=1.0, idx=16, w=16,
             load=None, stream=None)
ROUTE_GRAD = dict(z=16, dt=0, T=4, E=64, k=4, idx=16, dw=16, func=0, renorm=1, scale=1.0, dz=16, stream=None)


@pytest.mark.parametrize("over, msg", [
    (dict(dt=3), "dtype"), (dict(E=0), "E must be"), (dict(E=1025), "E must be"), (dict(k=0), "k must be"),
    (dict(k=33), "k must be"), (dict(k=65), "k must be"), (dict(func=3), "score_func"), (dict(groups=0), "divide E"),
    (dict(groups=7), "divide E"), (dict(groups=65), "divide E"), (dict(topk_groups=9), "topk_groups"),
    (dict(topk_groups=0), "topk_groups"), (dict(topk_groups=1, k=9), "topk_groups"), (dict(T=(1 << 25) + 1), "2^25"),
    (dict(z=None), "null"), (dict(idx=None), "null"), (dict(w=None), "null"), (dict(z=18), "misaligned"),
    (dict(load=2), "misaligned"), (dict(bias=2), "misaligned"),
])
def test_route_entry_refuses(over, msg):
    _refused("keep_route_experts", ROUTE, over, msg)


@pytest.mark.parametrize("over, msg", [
    (dict(dt=3), "dtype"), (dict(E=2000), "E must be"), (dict(k=0), "k must be"), (dict(func=-1), "score_func"),
    (dict(dw=None), "null"), (dict(dz=None), "null"), (dict(dz=18), "misaligned"),
])
def test_route_grad_entry_refuses(over, msg):
    _refused("keep_route_experts_grad", ROUTE_GRAD, over, msg)


LINEAR = dict(x=16, x_ld=64, dt=2, M=20, w=16, w_ld=64, N=32, K=64, bias=None, bdt=0, act=0, res=None, rdt=0, u=None, out=16,
              odt=2, ws=16, ws_bytes=1 << 30, stream=None)
LINEAR_Q8 = dict(x=16, x_ld=64, xs=16, M=20, w=16, w_ld=64, ws_=16, N=32, K=64, bias=None, bdt=0, act=0, res=None, rdt=0, out=16,
                 odt=2, ws=16, ws_bytes=1 << 30, stream=None)
LINEAR_GRAD = dict(dy=16, u=16, act=2, x=16, x_ld=64, w=16, w_ld=64, dt=2, M=20, N=32, K=64, dx=16, dw=16, db=16, bdt=0, ws=256,
                   ws_bytes=1 << 30, stream=None)


@pytest.mark.parametrize("over, msg", [
    (dict(N=0), "2^20"), (dict(K=0), "2^20"), (dict(N=(1 << 20) + 1), "2^20"), (dict(M=-1), "2^31"),
    (dict(M=(1 << 31) - 1, N=1 << 20), "too many"), (dict(x=None), "null"), (dict(out=None), "null"), (dict(x=8), "x must be"),
    (dict(x_ld=60), "x must be"), (dict(x_ld=65), "x must be"), (dict(w=8), "weight must be"), (dict(w_ld=32), "weight must be"),
    (dict(w_ld=1 << 30), "weight must be"), (dict(act=5), "activation"), (dict(act=-1), "activation"), (dict(odt=3), "dtype"),
    (dict(bias=16, bdt=7), "dtype"), (dict(res=16, rdt=7), "dtype"), (dict(out=17), "misaligned"),
    (dict(bias=17, bdt=1), "misaligned"), (dict(res=18, rdt=0), "misaligned"),
])
def test_linear_entries_refuse(over, msg):
    _refused("keep_linear", LINEAR, over, msg)
    _refused("keep_linear_q8", LINEAR_Q8, over, msg)


@pytest.mark.parametrize("name, args, over, msg", [
    ("keep_linear", LINEAR, dict(dt=3), "dtype"), ("keep_linear", LINEAR, dict(u=17), "misaligned"),
    ("keep_linear", LINEAR, dict(K=65536, x_ld=65536, w_ld=65536, ws=None), "workspace"),
    ("keep_linear", LINEAR, dict(K=65536, x_ld=65536, w_ld=65536, ws_bytes=64), "workspace"),
    ("keep_linear_q8", LINEAR_Q8, dict(xs=None), "null"), ("keep_linear_q8", LINEAR_Q8, dict(ws_=None), "null"),
    ("keep_linear_q8", LINEAR_Q8, dict(xs=18), "misaligned"),
    ("keep_linear_grad", LINEAR_GRAD, dict(dt=4), "dtype"), ("keep_linear_grad", LINEAR_GRAD, dict(bdt=4), "dtype"),
    ("keep_linear_grad", LINEAR_GRAD, dict(act=9), "activation"), ("keep_linear_grad", LINEAR_GRAD, dict(u=None), "null"),
    ("keep_linear_grad", LINEAR_GRAD, dict(dy=None), "null"), ("keep_linear_grad", LINEAR_GRAD, dict(x=None), "null"),
    ("keep_linear_grad", LINEAR_GRAD, dict(w=None), "null"),
    ("keep_linear_grad", LINEAR_GRAD, dict(dx=None, dw=None, db=None), "null"),
    ("keep_linear_grad", LINEAR_GRAD, dict(x_ld=32), "x must be"), ("keep_linear_grad", LINEAR_GRAD, dict(w=8), "weight must be"),
    ("keep_linear_grad", LINEAR_GRAD, dict(ws=None), "workspace"), ("keep_linear_grad", LINEAR_GRAD, dict(ws=16), "workspace"),
    ("keep_linear_grad", LINEAR_GRAD, dict(ws_bytes=256), "workspace"), ("keep_linear_grad", LINEAR_GRAD, dict(db=18), "misaligned"),
])
def test_linear_entry_refuses(name, args, over, msg):
    _refused(name, args, over, msg)


def test_nothing_to_do_is_a_no_op():
    lib = _lib.load()
    for name, args, rows in (("keep_rmsnorm", NORM, "T"), ("keep_rmsnorm_quant", QUANT, "T"), ("keep_rmsnorm_grad", NORM_GRAD, "T"),
                             ("keep_route_experts", ROUTE, "T"), ("keep_route_experts_grad", ROUTE_GRAD, "T"),
                             ("keep_linear", LINEAR, "M"), ("keep_linear_q8", LINEAR_Q8, "M"),
                             ("keep_linear_grad", LINEAR_GRAD, "M")):
        none = {**args, rows: 0, **{n: None for n in args if n in ("x", "z", "h", "dy")}}
        assert getattr(lib, name)(*none.values()) == 0, name


def test_workspace_sizes():
    lib = _lib.load()
    assert lib.keep_rmsnorm_grad_workspace_bytes(4, 20000) == lib.keep_rmsnorm_grad_workspace_bytes(-1, 64) == 0
    assert 0 < lib.keep_rmsnorm_grad_workspace_bytes(1, 64) < lib.keep_rmsnorm_grad_workspace_bytes(1000, 64)
    assert lib.keep_linear_workspace_bytes(9, 4, 4, 4) == lib.keep_linear_workspace_bytes(2, 0, 4, 4) == 0
    assert lib.keep_linear_workspace_bytes(2, 4, 4, 1 << 21) == 0
    assert lib.keep_linear_workspace_bytes(2, 100, 100, 65536) > 0  # few tiles, a long sum: slices
    assert lib.keep_linear_grad_workspace_bytes(3, 4, 4, 4) == 0
    assert 0 < lib.keep_linear_grad_workspace_bytes(2, 4, 4, 4) < lib.keep_linear_grad_workspace_bytes(0, 400, 400, 4)


# --------------------------------------------------------------------------- Python


@pytest.fixture
def anywhere(monkeypatch):
    """The argument checks on CPU tensors: none of these calls reaches a launch."""
    for where in (ops, block, router):
        monkeypatch.setattr(where, "_dense_device", lambda *ts: torch.device("cpu"))
    monkeypatch.setattr(_lib, "call", lambda name, *a: pytest.fail(f"{name} was launched"))


def test_cpu_tensors_are_refused():
    x, w = torch.zeros(2, 16), torch.zeros(8, 16)
    for call in (lambda: keep_amd.rmsnorm(x), lambda: keep_amd.rmsnorm(x, residual=x, weight=w[0]), lambda: keep_amd.rmsnorm_quant(x),
                 lambda: keep_amd.route_experts(x, 2), lambda: keep_amd.linear(x, w),
                 lambda: keep_amd.DenseLinear(w)(x), lambda: keep_amd.MoEGate(w, top_k=1)(x),
                 lambda: keep_amd.linear_q8(x.to(torch.float8_e4m3fn), x[:, :1], w.to(torch.float8_e4m3fn), w[:1, :1])):
        with pytest.raises(ValueError, match="cuda device"):
            call()


@pytest.mark.parametrize("over, msg", [
    (dict(x=torch.zeros(2, 16).double()), "float32, float16"), (dict(x=torch.zeros(2, 0)), "1..16384"),
    (dict(x=torch.zeros(1, 16385)), "1..16384"), (dict(x=torch.zeros(())), "1..16384"), (dict(weight=torch.zeros(15)), "weight"),
    (dict(weight=torch.zeros(16).double()), "weight"), (dict(residual=torch.zeros(3, 16)), "residual"),
    (dict(residual=torch.zeros(2, 16).half()), "residual"), (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
])
def test_norms_refuse(anywhere, over, msg):
    args = {"x": torch.zeros(2, 16), **over}
    for f in (keep_amd.rmsnorm, keep_amd.rmsnorm_quant):
        with pytest.raises(ValueError, match=msg):
            f(**args)


@pytest.mark.parametrize("over, msg", [
    (dict(quant_block=8), "power of two"), (dict(quant_block=100), "power of two"), (dict(quant_block=1024), "power of two"),
    (dict(x=torch.zeros(2, 16, requires_grad=True)), "no gradient"),
    (dict(residual=torch.zeros(2, 16, requires_grad=True)), "no gradient"),
])
def test_quant_refuses(anywhere, over, msg):
    with pytest.raises(ValueError, match=msg):
        keep_amd.rmsnorm_quant(**{"x": torch.zeros(2, 16), **over})


@pytest.mark.parametrize("over, msg", [
    (dict(logits=torch.zeros(16)), "2D"), (dict(logits=torch.zeros(2, 16).double()), "2D"), (dict(k=0), "k must be"),
    (dict(k=17), "k must be"), (dict(logits=torch.zeros(2, 64), k=33), "k must be"), (dict(score_func="relu"), "score_func"),
    (dict(groups=3), "divide"), (dict(groups=0), "divide"), (dict(groups=4, topk_groups=5), "topk_groups"),
    (dict(groups=4, topk_groups=0), "topk_groups"), (dict(groups=4, topk_groups=1, k=5), "k must be"),
    (dict(logits=torch.zeros(2, 1025)), "1..1024"), (dict(logits=torch.zeros(2, 0)), "1..1024"),
    (dict(bias=torch.zeros(15)), "bias"), (dict(bias=torch.zeros(16, requires_grad=True)), "no gradient"),
])
def test_route_experts_refuses(anywhere, over, msg):
    with pytest.raises(ValueError, match=msg):
        keep_amd.route_experts(**{"logits": torch.zeros(2, 16), "k": 2, **over})


@pytest.mark.parametrize("over, msg", [
    (dict(x=torch.zeros(2, 8)), "trailing dimension"), (dict(weight=torch.zeros(16)), "2D"), (dict(weight=torch.zeros(0, 16)), "2D"),
    (dict(x=torch.zeros(())), "2D"), (dict(x=torch.zeros(2, 16).half()), "share a dtype"),
    (dict(x=torch.zeros(2, 16).double(), weight=torch.zeros(8, 16).double()), "share a dtype"),
    (dict(bias=torch.zeros(7)), "bias"), (dict(bias=torch.zeros(8).double()), "bias"), (dict(activation="tanh"), "activation"),
    (dict(residual=torch.zeros(2, 7)), "residual"), (dict(residual=torch.zeros(2, 8).half()), "one of|residual"),
    (dict(out_dtype=torch.float16), "out_dtype"), (dict(out_dtype=torch.float64), "out_dtype"),
])
def test_linear_refuses(anywhere, over, msg):
    with pytest.raises(ValueError, match=msg):
        keep_amd.linear(**{"x": torch.zeros(2, 16), "weight": torch.zeros(8, 16), **over})


@pytest.mark.parametrize("over, msg", [
    (dict(x=torch.zeros(2, 16)), "float8_e4m3fn"), (dict(x_scales=torch.zeros(2, 2)), "x_scales"),
    (dict(x_scales=torch.zeros(2, 1).half()), "x_scales"), (dict(weight_scales=torch.zeros(2, 1)), "weight_scales"),
    (dict(bias=torch.zeros(8, requires_grad=True)), "no gradients"), (dict(x_scales=torch.zeros(2, 1, requires_grad=True)), "no gradients"),
    (dict(out_dtype=torch.float64), "out_dtype"),
])
def test_linear_q8_refuses(anywhere, over, msg):
    e = torch.float8_e4m3fn
    with pytest.raises(ValueError, match=msg):
        keep_amd.linear_q8(**{"x": torch.zeros(2, 16).to(e), "x_scales": torch.zeros(2, 1), "weight": torch.zeros(8, 16).to(e),
                              "weight_scales": torch.zeros(1, 1), **over})


def test_layers_refuse():
    lin, down = keep_amd.DenseLinear(torch.zeros(8, 16)), keep_amd.DenseLinear(torch.zeros(16, 8))
    with pytest.raises(ValueError, match="2D"):
        keep_amd.DenseLinear(torch.zeros(16))
    with pytest.raises(ValueError, match="bias"):
        keep_amd.DenseLinear(torch.zeros(8, 16), torch.zeros(16))
    with pytest.raises(ValueError, match="activation"):
        keep_amd.DenseLinear(torch.zeros(8, 16), activation="tanh")
    with pytest.raises(ValueError, match="down_proj"):
        keep_amd.DenseGLU(gate_proj=lin, up_proj=lin, down_proj=lin)
    with pytest.raises(ValueError, match="must match"):
        keep_amd.DenseGLU(gate_proj=lin, up_proj=down, down_proj=down)
    with pytest.raises(ValueError, match="no activation"):
        keep_amd.DenseGLU(gate_proj=keep_amd.DenseLinear(torch.zeros(8, 16), activation="silu"), up_proj=lin, down_proj=down)
    with pytest.raises(ValueError, match="bias"):
        keep_amd.MoEGate(torch.zeros(4, 16), top_k=2, bias=torch.zeros(3))
    with pytest.raises(ValueError, match="no bias"):
        keep_amd.MoEGate(torch.zeros(4, 16), top_k=2).update_bias(torch.zeros(4), 0.1)
    experts = keep_amd.SwitchLinear(torch.zeros(4, 8, 16)), keep_amd.SwitchLinear(torch.zeros(4, 16, 8))
    glu = keep_amd.QuantizedVQSwitchGLU(gate_proj=experts[0], up_proj=experts[0], down_proj=experts[1])
    with pytest.raises(ValueError, match="the gate must route"):
        keep_amd.RoutedVQMoE(glu, top_k=2, gate=keep_amd.MoEGate(torch.zeros(5, 16), top_k=2))
    with pytest.raises(ValueError, match="the gate must route"):
        keep_amd.RoutedVQMoE(glu, top_k=3, gate=keep_amd.MoEGate(torch.zeros(4, 16), top_k=2))
    with pytest.raises(ValueError, match="slot_map"):
        keep_amd.RoutedVQMoE(glu, top_k=2, gate=keep_amd.MoEGate(torch.zeros(4, 16), top_k=2), slot_map=torch.zeros(4))
    with pytest.raises(ValueError, match="needs logits"):
        keep_amd.RoutedVQMoE(glu, top_k=2)(torch.zeros(2, 16))


@pytest.mark.parametrize("over", [dict(x=17), dict(w=17), dict(x_ld=63), dict(w_ld=63), dict(w_ld=1 << 23)])
def test_few_rows_of_any_pitch_are_refused_by_their_dtype(over):
    _refused("keep_linear", LINEAR, dict(M=16, **over), "x and weight must be")
