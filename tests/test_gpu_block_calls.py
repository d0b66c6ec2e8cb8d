"""Calls of the norms, the choice of experts and the dense projections that their own files do not make: tensors that are one
and the same, shared gradients, two streams at once, offsets past 32 bits, forward-mode tangents, captures on held leaves."""

import pytest
import torch
from torch.autograd import forward_ad

import keep_amd
from tests import test_gpu_norm, test_gpu_projection
from tests.bounded import Bounded
from tests.test_gpu_projection import _q8

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


@pytest.mark.parametrize("which", ["x", "residual", "weight", "bias", "logits"])
def test_tangents_are_refused(dev, which):
    t = {"x": torch.randn(4, 16, device=dev), "residual": torch.randn(4, 16, device=dev),
         "weight": torch.randn(16, 16, device=dev), "bias": torch.randn(16, device=dev),
         "logits": torch.randn(4, 16, device=dev)}
    norms = [lambda: keep_amd.rmsnorm(t["x"], t["bias"], residual=t["residual"]),
             lambda: keep_amd.rmsnorm_quant(t["x"], t["bias"], residual=t["residual"])]
    product = [lambda: keep_amd.linear(t["x"], t["weight"], t["bias"], residual=t["residual"])]
    choice = [lambda: keep_amd.route_experts(t["logits"], 2), lambda: keep_amd.route_experts(t["x"], 2, bias=t["logits"][0])]
    calls = {"x": norms + product, "residual": norms + product, "weight": product, "bias": norms + product, "logits": choice}
    with forward_ad.dual_level():
        t[which] = forward_ad.make_dual(t[which], torch.ones_like(t[which]))
        for call in calls[which]:
            with pytest.raises((NotImplementedError, ValueError)):
                call()
            with torch.no_grad(), pytest.raises((NotImplementedError, ValueError)):
                call()


@pytest.mark.parametrize("op", ["norm", "route", "linear"])
def test_capture_on_leaves_of_a_live_eager_graph_is_refused(dev, monkeypatch, op):
    """(Nothing is captured: what asks whether the stream is being captured is answered for it.)"""
    x, w = torch.randn(4, 16, device=dev, requires_grad=True), torch.randn(16, 16, device=dev, requires_grad=True)
    call = {"norm": lambda x: keep_amd.rmsnorm(x, w[0].detach(), residual=x.detach())[0],
            "route": lambda x: keep_amd.route_experts(x, 2).weight,
            "linear": lambda x: keep_amd.linear(x, w.detach())}[op]
    held = call(x)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="eager graph"):
            call(x)
        call(x.detach().requires_grad_())
        with torch.no_grad():
            call(x)
    del held


@pytest.mark.parametrize("dtype, res", [(BF16, BF16), (BF16, F32), (F32, F32)])
def test_the_norms_gradients_are_tensors_of_their_own(dev, dtype, res):
    """x and the residual have the same gradient: what one leaf's is changed by does not reach the other's."""
    x, r = torch.randn(5, 48, device=dev, dtype=dtype, requires_grad=True), torch.randn(5, 48, device=dev, dtype=res,
                                                                                      requires_grad=True)
    w = torch.randn(48, device=dev)
    y, h = keep_amd.rmsnorm(x, w, residual=r)
    (y.float().sum() + h.float().sum()).backward()
    kept = r.grad.clone()
    assert torch.equal(x.grad, r.grad.to(dtype))
    x.grad.zero_()
    assert torch.equal(r.grad, kept)
    y, h = keep_amd.rmsnorm(x, w, residual=r)  # and a second pass adds to each
    (y.float().sum() + h.float().sum()).backward()
    assert torch.equal(x.grad, kept.to(dtype)) and torch.equal(r.grad, kept + kept)


def test_the_same_tensor_twice(dev):
    """A leaf as x and residual, as x and weight, as bias of itself: its gradient is the sum of its parts."""
    x = torch.randn(6, 64, device=dev, requires_grad=True)
    a, b = x.detach().requires_grad_(True), x.detach().requires_grad_(True)
    dy, dh = torch.randn(6, 64, device=dev), torch.randn(6, 64, device=dev)
    one, = torch.autograd.grad(keep_amd.rmsnorm(x, residual=x), x, (dy, dh))
    two = torch.autograd.grad(keep_amd.rmsnorm(a, residual=b), (a, b), (dy, dh))
    assert torch.equal(one, two[0] + two[1])
    q = torch.randn(64, 64, device=dev, requires_grad=True)
    a, b = q.detach().requires_grad_(True), q.detach().requires_grad_(True)
    g = torch.randn(64, 64, device=dev)
    one, = torch.autograd.grad(keep_amd.linear(q, q, activation="silu"), q, g)
    two = torch.autograd.grad(keep_amd.linear(a, b, activation="silu"), (a, b), g)
    assert torch.equal(one, two[0] + two[1])
    out = keep_amd.linear(q, q, q[0], residual=q)
    assert torch.equal(out, keep_amd.linear(a, b, b[0].clone(), residual=a.clone()))


def test_broadcast_and_transposed_arguments(dev):
    """Views of stride 0 and of other orders: the values count, and a broadcast leaf's gradient is summed."""
    row = torch.randn(64, device=dev, dtype=F16, requires_grad=True)
    w = torch.randn(64, 40, device=dev, dtype=F16, requires_grad=True)
    x = row.expand(20, 64)
    out = keep_amd.linear(x, w.t(), w[0].expand(40), residual=w[1].expand(20, 40))
    again = keep_amd.linear(x.clone(), w.t().contiguous(), w[0].clone(), residual=w[1].expand(20, 40).clone())
    assert torch.equal(out, again)
    grads = [torch.autograd.grad(o.float().sum(), (row, w)) for o in (out, again)]  # (dy is of stride 0)
    assert all(torch.equal(a, b) for a, b in zip(*grads))
    y, h = keep_amd.rmsnorm(x, row, residual=torch.randn(64, 20, device=dev, dtype=F16).t())
    assert y.is_contiguous() and h.shape == (20, 64)
    assert torch.equal(keep_amd.rmsnorm(x, row), keep_amd.rmsnorm(x.clone(), row))
    z = torch.randn(16, 30, device=dev).t()
    for a, b in zip(keep_amd.route_experts(z, 4), keep_amd.route_experts(z.contiguous(), 4)):
        assert a is None and b is None or torch.equal(a, b)


@pytest.mark.parametrize("M, N, K, dtype", [(200, 96, 7168, BF16), (64, 64, 4096, F32), (1500, 136, 1000, F16), (300, 640, 520, BF16)])
def test_results_do_not_change_from_call_to_call(dev, M, N, K, dtype):
    x, w = torch.randn(M, K, device=dev).to(dtype).requires_grad_(), torch.randn(N, K, device=dev).to(dtype).requires_grad_()
    b, dy = torch.randn(N, device=dev, requires_grad=True), torch.randn(M, N, device=dev).to(dtype)

    def step():
        out = keep_amd.linear(x, w, b, activation="gelu")
        return [out.detach(), *torch.autograd.grad(out, (x, w, b), dy)]
    first = step()
    for _ in range(3):
        assert all(torch.equal(a, b) for a, b in zip(first, step()))


def test_two_streams_at_once(dev):
    """Calls that need workspaces, counts and row-block sums, on two streams and interleaved."""
    def work(seed):
        g = torch.Generator(device=dev).manual_seed(seed)
        x = torch.randn(200, 7168, device=dev, generator=g).to(BF16).requires_grad_()
        w = torch.randn(96, 7168, device=dev, generator=g).to(BF16).requires_grad_()
        n = torch.randn(7168, device=dev, generator=g).requires_grad_()
        torch.cuda.synchronize()

        def step():
            y = keep_amd.rmsnorm(x, n)
            r = keep_amd.route_experts(keep_amd.linear(y, w, out_dtype=F32), 6, groups=4, topk_groups=2, count_load=True)
            return [r.idx, r.load, r.weight.detach(), *torch.autograd.grad(r.weight.square().sum(), (x, w, n))]
        return step
    steps = [work(1), work(2)]
    alone = [s() for s in steps]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream(), torch.cuda.Stream()]
    got = [[], []]
    for _ in range(4):
        for i in (0, 1):
            with torch.cuda.stream(streams[i]):
                got[i].append(steps[i]())
    torch.cuda.synchronize()
    for i in (0, 1):
        for outs in got[i]:
            assert all(torch.equal(a, b) for a, b in zip(alone[i], outs))


def test_q8_nan_codes_stay_in_their_rows_and_columns(dev):
    for M in (5, 200):
        x, xs, w, ws = _q8(dev, M, 160, 272)
        want = keep_amd.linear_q8(x, xs, w, ws, out_dtype=F32)
        bad = x.clone()
        bad.view(torch.uint8)[3, 130] = 0x7F
        got = keep_amd.linear_q8(bad, xs, w, ws, out_dtype=F32)
        assert got[3].isnan().all() and torch.equal(torch.cat([got[:3], got[4:]]), torch.cat([want[:3], want[4:]]))
        bad = w.clone()
        bad.view(torch.uint8)[150, 271] = 0xFF
        got = keep_amd.linear_q8(x, xs, bad, ws, out_dtype=F32)
        assert got[:, 150].isnan().all() and torch.equal(got[:, :150], want[:, :150])
        assert torch.equal(got[:, 151:], want[:, 151:])


def test_values_past_32_bit_offsets(dev):
    """More than 2^32 bytes and 2^31 values: the last rows are those of a small call."""
    def last(t, n):
        return t[-n:].clone()
    T, n = (1 << 31) // 2048 + 5, 2056
    x = torch.empty(T, n, device=dev, dtype=BF16)
    x[-9:] = torch.randn(9, n, device=dev).to(BF16)
    w = torch.randn(n, device=dev)
    y, h = keep_amd.rmsnorm(x, w, residual=x)
    assert all(torch.equal(a, b) for a, b in zip((last(y, 9), last(h, 9)),
                                                 keep_amd.rmsnorm(last(x, 9), w, residual=last(x, 9))))
    del h
    q, s = keep_amd.rmsnorm_quant(x, w)
    few = keep_amd.rmsnorm_quant(last(x, 9), w)
    assert torch.equal(last(q, 9).view(torch.uint8), few[0].view(torch.uint8)) and torch.equal(last(s, 9), few[1])
    del q, s
    few = last(x, 9).requires_grad_()
    small, = torch.autograd.grad(keep_amd.rmsnorm(few, w), few, last(y, 9))
    large, = torch.autograd.grad(keep_amd.rmsnorm(x.requires_grad_(), w), x, y)
    assert torch.equal(last(large, 9), small)
    x = x.detach()
    del large, y
    z = x.view(-1)[: T * n // 1024 * 1024].view(-1, 1024)
    r, few = keep_amd.route_experts(z, 6), keep_amd.route_experts(last(z, 9), 6)
    assert torch.equal(last(r.idx, 9), few.idx) and torch.equal(last(r.weight, 9), few.weight)
    del r, z
    w = torch.randn(40, n, device=dev).to(BF16)
    out = keep_amd.linear(x, w, out_dtype=F32)  # (x past 32 bits)
    (Bounded(last(x, 9)) @ Bounded(w).T).round(F32).check(last(out, 9))
    del out, x
    x = torch.zeros((1 << 31) // 4096 + 300, 24, device=dev, dtype=BF16)
    x[-9:] = torch.randn(9, 24, device=dev).to(BF16)
    w = torch.randn(4104, 24, device=dev).to(BF16).requires_grad_()
    out = keep_amd.linear(x, w)  # (the output past 32 bits)
    (Bounded(last(x, 9)) @ Bounded(w.detach()).T).round(BF16).check(last(out.detach(), 9))
    dw, = torch.autograd.grad(out, w, out.detach())  # dW = dy^T x: rows of zeros but the last nine
    want = Bounded(last(out.detach(), 9)).T @ Bounded(last(x, 9))
    Bounded(want.v, want.e).round(BF16).check(dw)


@pytest.mark.parametrize("n", [2, 7, 9, 15, 17, 505, 1023, 1025, 2047, 4095, 4097, 8193, 12289])
@pytest.mark.parametrize("dtype, res, wdt", [(BF16, F32, F16), (F16, F16, F32), (F32, None, F32)])
def test_row_ends(dev, n, dtype, res, wdt):
    """Every place of a row's end in its last vector, in each of the kernels' widths, with values around the rows."""
    c = test_gpu_norm._case(dev, 11, n, dtype, res, wdt, seed=n)
    for k in ("x", "res", "dy", "dh"):  # inside larger tensors: what lies around a row is not zero
        if c[k] is not None:
            big = torch.full((13, n), 3.0e4, device=dev, dtype=c[k].dtype)
            big[1:12] = c[k]
            c[k] = big[1:12]
    test_gpu_norm._check(c)
    q, s = keep_amd.rmsnorm_quant(c["x"], c["w"], quant_block=16)[:2]
    y = test_gpu_norm._normed(c, c["x"])[0]
    each = s.double().repeat_interleave(16, 1)[:, :n]
    bound = y.e + (y.v.abs() + y.e) * 2.0 ** -4 + each * 2.0 ** -10 + y.v.abs() * 2.0 ** -23
    assert ((q.double() * each - y.v).abs() <= bound).all()


@pytest.mark.parametrize("M, N, K, dtype", [(1000, 1900, 6200, BF16), (1000, 2300, 328, F16), (1000, 2300, 300, F32),
                                            (70, 1500, 2900, F16), (600, 400, 4100, F32), (260, 2050, 4096, BF16)])
def test_tiles_and_slices_between_the_large_and_the_small(dev, M, N, K, dtype):
    test_gpu_projection._check(test_gpu_projection._case(dev, dtype, M, N, K, bias=F32), "silu")


@pytest.mark.parametrize("M, N, K", [(1000, 1900, 6208), (300, 2050, 2064), (64, 2048, 4096)])
def test_q8_tiles_and_slices(dev, M, N, K):
    x, xs, w, ws = _q8(dev, M, N, K)
    test_gpu_projection._q8_expected(x, xs, w, ws).round(BF16).check(keep_amd.linear_q8(x, xs, w, ws))


@pytest.mark.parametrize("M", [1, 3, 16])
@pytest.mark.parametrize("dtype", [F32, F16, BF16])
@pytest.mark.parametrize("K", [1, 2, 3, 5, 7, 8, 9, 31, 33, 70, 255, 257, 1029, 3925])
def test_few_rows_at_any_address(dev, M, dtype, K):
    """Rows of any length and start, with NaN around them: the sums of a copy."""
    c = test_gpu_projection._case(dev, dtype, M, 37, K, bias=F32)
    want = test_gpu_projection._expected(c, None, dtype, grads=False)[0]
    want.check(keep_amd.linear(c["x"], c["w"], c["b"]))

    def inside(t, left, right):
        big = torch.full((t.shape[0], left + t.shape[1] + right), float("nan"), device=dev, dtype=t.dtype)
        big[:, left:left + t.shape[1]] = t
        return big[:, left:left + t.shape[1]]
    for left, right in ((0, 1), (1, 0), (3, 2), (8, 8)):
        got = keep_amd.linear(inside(c["x"], left, right), inside(c["w"], right, left), c["b"])
        want.check(got)
    want.check(keep_amd.linear(c["x"].t().contiguous().t(), c["w"].t().contiguous().t(), c["b"]))
