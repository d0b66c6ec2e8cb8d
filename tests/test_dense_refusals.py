"""What the dense routed product, the adapters and the combine refuse, on the CPU: before any launch."""

import pytest
import torch

import keep_amd
from keep_amd import _lib


def _lib_call(name, **args):
    return getattr(_lib.load(), name)(*args.values())


PLAN = dict(order=16, offsets=16, counts=16, te=16, to=16, tc=16, valid=16)


def _gather(**over):
    args = dict(x=16, dtype=1, x_rows=4, w=16, transposed=0, rhs=16, lhs=None, routes=4, x_div=1, E=2, N=8, K=16,
                order=None, offsets=None, counts=None, te=None, to=None, tc=None, valid=None, n_tiles=0, tile=0, out=16,
                odt=1, stream=None)
    assert not set(over) - set(args)
    return _lib_call("keep_gather_mm", **{**args, **over})


@pytest.mark.parametrize("over, msg", [
    (dict(dtype=7), "dtype"),
    (dict(odt=-1), "dtype"),
    (dict(E=0), "positive"),
    (dict(N=0), "positive"),
    (dict(K=-1), "2^31"),
    (dict(x=None), "null"),
    (dict(rhs=None), "null"),
    (dict(x_rows=0), "null"),
    (dict(x_div=0), "x_div"),
    (dict(x=17), "misaligned"),
    (dict(w=1), "misaligned"),
    (dict(out=3), "misaligned"),
    (dict(order=16), "all of its arrays"),
    (dict(te=16), "all of its arrays"),
    (dict(**PLAN, n_tiles=0), "n_tiles"),
    (dict(**PLAN, n_tiles=3, tile=64, dtype=0, odt=0), "16-bit rows"),
    (dict(**PLAN, n_tiles=3, tile=64, K=20), "16-bit rows"),
    (dict(**PLAN, n_tiles=3, tile=64, transposed=1, N=12), "16-bit rows"),
    (dict(**PLAN, n_tiles=3, tile=32), "16-bit rows"),
    (dict(**PLAN, n_tiles=3, tile=64, x=18), "16-byte aligned"),
    (dict(**PLAN, n_tiles=3, tile=64, odt=2), "16-byte aligned"),
    (dict(routes=1 << 30, N=1 << 20), "too many"),
])
def test_gather_mm_entry_refuses(over, msg):
    assert _gather(**over) == _lib.KEEP_EINVAL
    assert msg in _lib.load().keep_last_error().decode()


def test_no_routes_is_a_no_op():
    assert _gather(routes=0, x=None, rhs=None) == 0
    assert _lora(routes=0, x=None) == 0
    lib = _lib.load()
    assert lib.keep_route_combine_rows(None, 0, None, 0, 2, 8, None, 0, None) == 0
    assert lib.keep_route_combine_grad(None, 0, None, None, 0, 0, 2, 8, None, None, None) == 0


@pytest.mark.parametrize("over, msg", [
    (dict(R=0), "route count"), (dict(E=1025), "E must be"), (dict(tile=0), "tile must be"),
    (dict(max_tiles=3), "max_tiles"), (dict(ws=None), "null"), (dict(order=None), "null"), (dict(ws_bytes=10), "workspace"),
])
def test_plan_over_several_workgroups_refuses(over, msg):
    args = dict(rhs=16, R=9000, E=4, tile=16, order=16, inverse=16, counts=16, offsets=16, te=16, to=16, tc=16,
                max_tiles=1000, nt=16, ws=16, ws_bytes=1 << 20, stream=None)
    assert _lib_call("keep_route_plan_blocks", **{**args, **over}) == _lib.KEEP_EINVAL
    assert msg in _lib.load().keep_last_error().decode()


def _grad_weight(**over):
    args = dict(x=16, dtype=1, x_rows=4, dy=16, routes=4, x_div=1, E=2, N=8, K=16, order=16, offsets=16, counts=16,
                dw=16, stream=None)
    return _lib_call("keep_gather_mm_grad_weight", **{**args, **over})


@pytest.mark.parametrize("over, msg", [
    (dict(dtype=3), "dtype"), (dict(E=0), "positive"), (dict(x_div=0), "positive"), (dict(E=70000), "too many"),
    (dict(order=None), "null"), (dict(dw=None), "null"), (dict(dw=17), "misaligned"), (dict(routes=-1), "2^31"),
])
def test_grad_weight_entry_refuses(over, msg):
    assert _grad_weight(**over) == _lib.KEEP_EINVAL
    assert msg in _lib.load().keep_last_error().decode()


def _lora(**over):
    args = dict(x=16, dtype=1, x_rows=4, a=16, b=16, scales=None, idx=16, routes=4, x_div=1, n=2, rank=16, K=32, N=8,
                base=None, bdt=0, t_out=None, grouped=0, ws=16, ws_bytes=1 << 30, out=16, odt=1, stream=None)
    assert not set(over) - set(args)
    return _lib_call("keep_lora", **{**args, **over})


@pytest.mark.parametrize("over, msg", [
    (dict(dtype=5), "dtype"),
    (dict(base=16, bdt=0), "base out's"),
    (dict(odt=2), "x's dtype or float32"),
    (dict(rank=0), "rank"),
    (dict(rank=129), "rank"),
    (dict(n=0), "positive"),
    (dict(x_div=0), "positive"),
    (dict(idx=None), "null"),
    (dict(ws=None), "null"),
    (dict(routes=5), "need more"),
    (dict(routes=9, x_div=2), "need more"),
    (dict(a=17), "misaligned"),
    (dict(ws=8), "misaligned"),
    (dict(ws_bytes=10), "workspace needs"),
    (dict(n=1025, grouped=1), "at most 1024"),
    (dict(base=17, bdt=1), "misaligned"),
    (dict(routes=1 << 30, x_rows=1 << 30, N=1 << 20), "too many"),
])
def test_lora_entry_refuses(over, msg):
    assert _lora(**over) == _lib.KEEP_EINVAL
    assert msg in _lib.load().keep_last_error().decode()


def test_lora_sizes():
    lib = _lib.load()
    assert [lib.keep_lora_rank_stride(r) for r in (0, 1, 16, 17, 64, 65, 128, 129)] == [0, 16, 16, 32, 64, 128, 128, 0]
    need = lib.keep_lora_workspace_bytes
    assert need(1, -1, 4, 16, 64, 0) == need(9, 1, 4, 16, 64, 0) == need(1, 0, 4, 16, 64, 0) == 0
    assert 0 < need(1, 1, 4, 16, 64, 0) < need(1, 1, 4, 16, 64, 1)
    need = lib.keep_lora_backward_workspace_bytes
    assert need(1, 0, 1, 4, 16, 64, 32, 1, 1) == need(1, 4, 1, 4, 200, 64, 32, 1, 1) == 0
    assert 0 < need(1, 8, 2, 4, 16, 64, 32, 0, 0) < need(1, 8, 2, 4, 16, 64, 32, 1, 0) < need(1, 8, 2, 4, 16, 64, 32, 1, 1)


@pytest.mark.parametrize("over, msg", [
    (dict(dtype=5), "dtype"), (dict(rank=200), "rank"), (dict(n=0), "positive"), (dict(planned=0), "need a plan"),
    (dict(n=2000), "at most 1024"), (dict(routes=3), "rows of"), (dict(routes=5), "need more"), (dict(t=None), "null"),
    (dict(dy=None), "null"), (dict(da=17), "misaligned"), (dict(ws=16), "misaligned"),
    (dict(ws_bytes=100), "workspace needs"),
])
def test_lora_backward_entry_refuses(over, msg):
    args = dict(x=16, dtype=1, x_rows=4, a=16, b=16, scales=None, idx=16, routes=4, x_div=1, n=2, rank=16, K=32, N=8,
                t=16, dy=16, dx=16, da=16, db=16, planned=1, ws=256, ws_bytes=1 << 30, stream=None)
    assert not set(over) - set(args)
    assert _lib_call("keep_lora_backward", **{**args, **over}) == _lib.KEEP_EINVAL
    assert msg in _lib.load().keep_last_error().decode()


@pytest.mark.parametrize("args, msg", [
    ((16, 4, 16, 2, 2, 8, 16, 0, None), "dtype"), ((16, 0, 16, 2, 0, 8, 16, 0, None), "positive"),
    ((None, 0, 16, 2, 2, 8, 16, 0, None), "null"), ((16, 0, 16, -1, 2, 8, 16, 0, None), "2^31"),
])
def test_combine_rows_entry_refuses(args, msg):
    assert _lib.load().keep_route_combine_rows(*args) == _lib.KEEP_EINVAL
    assert msg in _lib.load().keep_last_error().decode()


@pytest.mark.parametrize("args, msg", [
    ((16, 4, 16, 16, 0, 2, 2, 8, 16, 16, None), "dtype"), ((16, 0, 16, 16, 0, 2, 2, 8, None, None, None), "null"),
    ((None, 0, 16, 16, 0, 2, 2, 8, 16, 16, None), "null"), ((16, 0, None, 16, 0, 2, 2, 8, 16, 16, None), "null"),
    ((16, 0, 16, 16, 0, 2, 0, 8, 16, 16, None), "positive"),
])
def test_combine_grad_entry_refuses(args, msg):
    assert _lib.load().keep_route_combine_grad(*args) == _lib.KEEP_EINVAL
    assert msg in _lib.load().keep_last_error().decode()


def test_cpu_tensors_are_refused():
    x, w, idx = torch.zeros(2, 16), torch.zeros(3, 8, 16), torch.zeros(2, 1, dtype=torch.int32)
    with pytest.raises(ValueError, match="cuda device"):
        keep_amd.gather_mm(x, w, idx)
    with pytest.raises(ValueError, match="cuda device"):
        keep_amd.gather_lora(x, torch.zeros(3, 4, 16), torch.zeros(3, 8, 4), idx)
    for grad in (False, True):
        with pytest.raises(ValueError, match="cuda device"):
            keep_amd.route_combine(torch.zeros(2, 1, 8, requires_grad=grad), torch.zeros(2, 1))


@pytest.fixture
def anywhere(monkeypatch):
    """The argument checks on CPU tensors: none of these calls reaches a launch."""
    from keep_amd import ops
    monkeypatch.setattr(ops, "_dense_device", lambda *ts: torch.device("cpu"))
    monkeypatch.setattr(_lib, "call", lambda name, *a: pytest.fail(f"{name} was launched"))


@pytest.mark.parametrize("over, msg", [
    (dict(x=torch.zeros(2, 3, 16)), "2D"),
    (dict(w=torch.zeros(8, 16)), "3D"),
    (dict(w=torch.zeros(3, 0, 16)), "3D"),
    (dict(x=torch.zeros(2, 16).half()), "share a dtype"),
    (dict(x=torch.zeros(2, 16).double(), w=torch.zeros(3, 8, 16).double()), "share a dtype"),
    (dict(x=torch.zeros(2, 8)), "trailing dimension"),
    (dict(idx=torch.zeros(2, dtype=torch.int32)), "tokens, top_k"),
    (dict(idx=torch.zeros(3, 1, dtype=torch.int32)), "tokens, top_k"),
    (dict(idx=torch.zeros(2, 1)), "integer dtype"),
    (dict(lhs=torch.zeros(3, dtype=torch.int32)), "same flattened shape"),
    (dict(x=torch.zeros(2, 16, requires_grad=True), lhs=torch.zeros(2, dtype=torch.int32)), "token layout only"),
    (dict(idx=torch.full((2, 1), 3), check=True), "rhs_indices must be in"),
])
def test_gather_mm_refuses(anywhere, over, msg):
    a = {"x": torch.zeros(2, 16), "w": torch.zeros(3, 8, 16), "idx": torch.zeros(2, 1, dtype=torch.int32), "lhs": None,
         "check": False, **over}
    with pytest.raises(ValueError, match=msg):
        keep_amd.gather_mm(a["x"], a["w"], a["idx"], lhs_indices=a["lhs"], validate_indices=a["check"])


@pytest.mark.parametrize("over, msg", [
    (dict(x=torch.zeros(16)), "2D"),
    (dict(a=torch.zeros(4, 16)), "lora_a and lora_b"),
    (dict(b=torch.zeros(3, 8, 5)), "lora_b must be"),
    (dict(b=torch.zeros(2, 8, 4)), "lora_b must be"),
    (dict(a=torch.zeros(3, 129, 16), b=torch.zeros(3, 8, 129)), "at most 128"),
    (dict(a=torch.zeros(3, 4, 16).half()), "share a dtype"),
    (dict(x=torch.zeros(2, 8)), "trailing dimension"),
    (dict(idx=torch.zeros(3, dtype=torch.int32)), "indices must be"),
    (dict(base=torch.zeros(2, 9)), "base must have shape"),
    (dict(base=torch.zeros(2, 8).double()), "base must have shape"),
    (dict(scales=torch.zeros(2)), "scales must have shape"),
    (dict(scales=torch.zeros(3, requires_grad=True)), "no gradient"),
    (dict(idx=torch.full((2,), 3), check=True), "below 3"),
])
def test_gather_lora_refuses(anywhere, over, msg):
    c = {"x": torch.zeros(2, 16), "a": torch.zeros(3, 4, 16), "b": torch.zeros(3, 8, 4),
         "idx": torch.zeros(2, dtype=torch.int32), "base": None, "scales": None, "check": False, **over}
    with pytest.raises(ValueError, match=msg):
        keep_amd.gather_lora(c["x"], c["a"], c["b"], c["idx"], base=c["base"], scales=c["scales"],
                             validate_indices=c["check"])


def test_layers_refuse():
    w = torch.zeros(3, 8, 16)
    with pytest.raises(ValueError, match="3D"):
        keep_amd.SwitchLinear(torch.zeros(8, 16))
    with pytest.raises(ValueError, match="bias"):
        keep_amd.SwitchLinear(w, torch.zeros(3, 7))
    with pytest.raises(ValueError, match="float32, float16"):
        keep_amd.SwitchLinear(w.double())
    with pytest.raises(ValueError, match="rank"):
        keep_amd.LoraAdapters(torch.zeros(2, 200, 16), torch.zeros(2, 8, 200))
    with pytest.raises(ValueError, match="adapters must be"):
        keep_amd.LoraAdapters(torch.zeros(2, 4, 16), torch.zeros(3, 8, 4))
    with pytest.raises(ValueError, match="scales"):
        keep_amd.LoraAdapters(torch.zeros(2, 4, 16), torch.zeros(2, 8, 4), torch.zeros(3))
    with pytest.raises(ValueError, match="routed experts"):
        keep_amd.SwitchLinear(w, adapters=keep_amd.LoraAdapters(torch.zeros(2, 4, 16), torch.zeros(2, 8, 4)))
    with pytest.raises(ValueError, match="the layer"):
        keep_amd.SwitchLinear(w, adapters=keep_amd.LoraAdapters(torch.zeros(2, 3, 4, 8), torch.zeros(2, 3, 8, 4)))
    lin = keep_amd.SwitchLinear(w)
    with pytest.raises(ValueError, match="layer with adapters"):
        lin(torch.zeros(2, 16), torch.zeros(2, 1, dtype=torch.int32), adapter_indices=torch.zeros(2))
    down = keep_amd.SwitchLinear(torch.zeros(3, 16, 8))
    glu = keep_amd.QuantizedVQSwitchGLU(gate_proj=lin, up_proj=lin, down_proj=down)
    with pytest.raises(ValueError, match="projection with adapters"):
        glu(torch.zeros(2, 16), torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2))


def test_adapter_indices_have_one_entry_per_row(anywhere):
    ad = keep_amd.LoraAdapters(torch.zeros(2, 4, 16), torch.zeros(2, 8, 4))
    with pytest.raises(ValueError, match="one adapter per row"):
        ad.add(torch.zeros(2, 8), torch.zeros(2, 16), torch.zeros(3, dtype=torch.int32))


def test_capture_check_marks_live_eager_graphs(monkeypatch):
    from keep_amd import _grad
    w = torch.zeros(3, requires_grad=True)
    capturing = [False]
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: capturing[0])
    _grad.mark(w * 2)  # nothing holds the node: the mark goes with it
    capturing[0] = True
    _grad.check_capture(w)
    capturing[0] = False
    held = _grad.mark((w * 2) * w)  # (a leaf beside an inner node)
    capturing[0] = True
    with pytest.raises(RuntimeError, match="eager graph"):
        _grad.check_capture(w)
    del held
    _grad.check_capture(w)
    capturing[0] = False
    held = _grad.mark(w.view(3, 1) * 2)  # under a view
    capturing[0] = True
    with pytest.raises(RuntimeError, match="eager graph"):
        _grad.check_capture(w.view(1, 3))
    del held
    _grad.check_capture(w.view(1, 3))


def test_combine_refuses_more_values_than_a_gpu_holds():
    lib = _lib.load()
    assert lib.keep_route_combine_rows(16, 1, 16, 1 << 30, 1 << 10, 8, 16, 1, None) == _lib.KEEP_EINVAL
    assert "too many" in lib.keep_last_error().decode()
    assert lib.keep_route_combine_grad(16, 1, 16, 16, 1, 1 << 30, 1 << 10, 8, 16, 16, None) == _lib.KEEP_EINVAL
    assert "too many" in lib.keep_last_error().decode()
