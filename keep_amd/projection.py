"""Dense projections with their epilogue, ``residual + act(x W^T + bias)``, in one call, with their gradients.

``linear`` takes rows and weights of one float dtype (the router's own product, a shared expert's, a biased projection);
``linear_q8`` takes both in 8 bits (e4m3) with float32 scales, as ``rmsnorm_quant`` leaves its rows, for serving. Sums are
float32 and rounded once. Up to 16 rows stream the weights, more run through LDS, in slices of the summed index where there
are few tiles (``keep_linear``). Rows and weights may be views with a pitch; where more than 16 rows are no whole number of
16-byte pieces, or start off one, they and the weights are copied first, in every call.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from keep_amd import _grad, _lib, ops

ACTIVATIONS = {None: 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
SCALE_BLOCK = 128  # values of a row, and rows of the weight, that share a scale of the 8-bit form
MAX_DIMS = 1 << 20
_FEW = 16  # rows up to which the kernels read rows of any address and length
_E4M3 = 3


def _rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``t [n, K]`` as the kernels read it, whole 16-byte pieces a row, and the values between two rows. Where it lies
    otherwise it is copied, its rows filled up with zeros to ``[n, ld]``."""

    (n, K), (ld, one), size = t.shape, t.stride(), t.element_size()
    if one == 1 and K * size % 16 == 0 and t.data_ptr() % 16 == 0:
        if n <= 1:
            return t, K
        if K <= ld <= 4 * MAX_DIMS and ld * size % 16 == 0:
            return t, ld
    piece = 16 // size
    ld = (K + piece - 1) // piece * piece
    out = torch.empty((n, ld), dtype=t.dtype, device=t.device)
    out[:, :K] = t
    if ld > K:
        out[:, K:].zero_()
    return out, ld


def _few_rows(t: torch.Tensor) -> tuple[torch.Tensor, int]:
    """``_rows`` of a call on few rows, which reads them as they lie where their values are neighbours."""

    n, K = t.shape
    if t.stride(1) == 1 and (n <= 1 or K <= t.stride(0) <= 4 * MAX_DIMS):
        return t, K if n <= 1 else t.stride(0)
    return t.contiguous(), K


def _launch(x, weight, K: int, bias, act: int, residual, out_dtype, keep_u: bool):
    """``(out, u or None)`` for rows ``x`` and ``weight`` of ``K`` values from ``_rows``."""

    (x, x_ld), (weight, w_ld) = x, weight
    M, N, device = x.shape[0], weight.shape[0], x.device
    out = torch.empty((M, N), dtype=out_dtype, device=device)
    u = torch.empty((M, N), dtype=x.dtype, device=device) if keep_u else None
    if M == 0:
        return out, u
    dt = ops._DT[x.dtype]
    need = _lib.load().keep_linear_workspace_bytes(dt, M, N, K)
    ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
    _lib.call("keep_linear", x.data_ptr(), x_ld, dt, M, weight.data_ptr(), w_ld, N, K, ops._ptr(bias),
              0 if bias is None else ops._DT[bias.dtype], act, ops._ptr(residual),
              0 if residual is None else ops._DT[residual.dtype], ops._ptr(u), out.data_ptr(), ops._DT[out_dtype],
              ops._ptr(ws), need, ops._stream(device))
    return out, u


class _Linear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act, out_dtype):
        xr, wr = _rows(x), _rows(weight)
        out, u = _launch(xr, wr, x.shape[1], bias, act, residual, out_dtype, act != 0)
        # packed rows whole, their zeros too; the pitches are those of what a saved-tensor hook gives back
        ctx.save_for_backward(xr[0], wr[0], u)
        ctx.act, ctx.dims = act, x.shape[1]
        ctx.bias_dtype = None if bias is None else bias.dtype
        ctx.residual_dtype = None if residual is None else residual.dtype
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, u = ctx.saved_tensors
        nx, nw, nb, nr = ctx.needs_input_grad[:4]
        dres = dy.to(ctx.residual_dtype) if nr else None
        if not (nx or nw or nb):
            return None, None, None, dres, None, None
        with ops._on(x.device):
            dx, dw, db = _backward(ctx, x, weight, u, dy, nx, nw, nb)
        return dx, dw, db, dres, None, None


def _backward(ctx, x, weight, u, dy, nx: bool, nw: bool, nb: bool):
    M, K, N, dtype, device = x.shape[0], ctx.dims, weight.shape[0], x.dtype, x.device
    make = torch.empty if M else torch.zeros
    wide = dy.dtype != dtype
    if wide:  # a float32 output of 16-bit rows: its gradient keeps its bits and range, so the products are float32's
        x, weight, u = x.float(), weight.float(), None if u is None else u.float()
    (x, x_ld), (weight, w_ld) = _rows(x), _rows(weight)
    u = None if u is None else u.contiguous()
    dx = make((M, K), dtype=x.dtype, device=device) if nx else None
    dw = make((N, K), dtype=x.dtype, device=device) if nw else None
    db = make((N,), dtype=ctx.bias_dtype, device=device) if nb else None
    if M:
        dt, g = ops._DT[x.dtype], dy.contiguous()
        need = _lib.load().keep_linear_grad_workspace_bytes(dt, M, N, K)
        ws = torch.empty(need, dtype=torch.uint8, device=device)
        _lib.call("keep_linear_grad", g.data_ptr(), ops._ptr(u), ctx.act, x.data_ptr(), x_ld, weight.data_ptr(), w_ld,
                  dt, M, N, K, ops._ptr(dx), ops._ptr(dw), ops._ptr(db), 0 if db is None else ops._DT[db.dtype],
                  ws.data_ptr(), need, ops._stream(device))
    if wide:
        dx, dw = (None if t is None else t.to(dtype) for t in (dx, dw))
    return dx, dw, db


def _check(x, weight, bias, activation, residual, out_dtype, dtypes) -> tuple:
    """The shape of the output and the activation's number."""

    if x.ndim < 1 or weight.ndim != 2 or 0 in weight.shape or max(weight.shape) > MAX_DIMS:
        raise ValueError(f"weight must be 2D [out, in] of 1..{MAX_DIMS}, and x [..., in], found {tuple(weight.shape)} "
                         f"and {tuple(x.shape)}")
    if x.shape[-1] != weight.shape[1]:
        raise ValueError(f"x trailing dimension must be {weight.shape[1]}, found {x.shape[-1]}")
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation must be one of {list(ACTIVATIONS)}, found {activation!r}")
    if out_dtype not in dtypes:
        raise ValueError(f"out_dtype must be one of {list(dtypes)}, found {out_dtype}")
    shape = (*x.shape[:-1], weight.shape[0])
    if bias is not None and (tuple(bias.shape) != (weight.shape[0],) or bias.dtype not in ops._DT):
        raise ValueError(f"bias must have shape ({weight.shape[0]},) in a float dtype, found {tuple(bias.shape)} "
                         f"in {bias.dtype}")
    if residual is not None and (tuple(residual.shape) != shape or residual.dtype not in dtypes):
        raise ValueError(f"residual must have shape {shape} in one of {list(dtypes)}, found {tuple(residual.shape)} "
                         f"in {residual.dtype}")
    return shape, ACTIVATIONS[activation]


def linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None,
           residual: torch.Tensor | None = None, out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``residual + act(x W^T + bias)`` for ``x [..., K]`` and ``weight [N, K]`` of one dtype, ``bias [N]`` of any.

    ``activation``: ``"relu"``, ``"silu"``, ``"gelu"`` (by the error function) or ``"gelu_tanh"``. The output and
    ``residual`` (of the output's shape) have ``x``'s dtype or float32; the output takes ``residual``'s without
    ``out_dtype``. Differentiable in ``x``, ``weight``, ``bias`` and ``residual``: the values before the activation are
    kept in ``x``'s dtype, and the gradient before the products is rounded to it; a float32 output of 16-bit rows has
    its products formed in float32, several times as long.
    """

    device = ops._dense_device(x, weight, bias, residual)
    if x.dtype != weight.dtype or x.dtype not in ops._DT:
        raise ValueError("x and weight must share a dtype of float32, float16 or bfloat16, found "
                         f"{x.dtype} and {weight.dtype}")
    od = out_dtype or (x.dtype if residual is None else residual.dtype)
    shape, act = _check(x, weight, bias, activation, residual, od, (x.dtype, torch.float32))
    with ops._on(device):
        flat = x.ndim == 2  # (a reshape and a view that change nothing cost 2 us of a small call's 13)
        rows = x if flat else x.reshape(-1, x.shape[-1])
        b = None if bias is None else bias.contiguous()
        r = None if residual is None else (residual if flat else residual.reshape(-1, shape[-1])).contiguous()
        if not _grad.wanted(x, weight, bias, residual):
            lie = _few_rows if rows.shape[0] <= _FEW else _rows
            out = _launch(lie(rows), lie(weight), weight.shape[1], b, act, r, od, False)[0]
        else:
            _grad.check_capture(x, weight, bias, residual)
            out = _grad.mark(_Linear.apply(rows, weight, b, r, act, od))
        return out if flat else out.view(shape)


def linear_q8(x: torch.Tensor, x_scales: torch.Tensor, weight: torch.Tensor, weight_scales: torch.Tensor,
              bias: torch.Tensor | None = None, *, activation: str | None = None, residual: torch.Tensor | None = None,
              out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``linear`` on 8-bit operands: ``x [..., K]`` and ``weight [N, K]`` in ``torch.float8_e4m3fn`` with float32 scales
    per 128 values of a row of ``x`` (``[..., ceil(K / 128)]``, as ``rmsnorm_quant`` gives them) and per 128 x 128
    values of ``weight`` (``[ceil(N / 128), ceil(K / 128)]``). The output is bfloat16 without ``residual`` or
    ``out_dtype`` (float32, float16 or bfloat16, ``residual`` too). No gradients."""

    device = ops._dense_device(x, x_scales, weight, weight_scales, bias, residual)
    if x.dtype != torch.float8_e4m3fn or weight.dtype != torch.float8_e4m3fn:
        raise ValueError(f"x and weight must be float8_e4m3fn, found {x.dtype} and {weight.dtype}")
    od = out_dtype or (torch.bfloat16 if residual is None else residual.dtype)
    shape, act = _check(x, weight, bias, activation, residual, od, tuple(ops._DT))
    (N, K), blocks = weight.shape, (weight.shape[1] + SCALE_BLOCK - 1) // SCALE_BLOCK
    for name, t, want in (("x_scales", x_scales, (*x.shape[:-1], blocks)),
                          ("weight_scales", weight_scales, ((N + SCALE_BLOCK - 1) // SCALE_BLOCK, blocks))):
        if tuple(t.shape) != want or t.dtype != torch.float32:
            raise ValueError(f"{name} must be float32 of shape {want}, found {tuple(t.shape)} in {t.dtype}")
    if _grad.wanted(x, x_scales, weight, weight_scales, bias, residual):
        raise ValueError("the 8-bit product has no gradients")
    with ops._on(device):
        flat = x.ndim == 2
        (xr, x_ld), (wr, w_ld) = _rows(x if flat else x.reshape(-1, K)), _rows(weight)
        M = xr.shape[0]
        out = torch.empty((M, N), dtype=od, device=device)
        if M == 0:
            return out.view(shape)
        xs, ws = x_scales.contiguous(), weight_scales.contiguous()
        b = None if bias is None else bias.contiguous()
        r = None if residual is None else residual.contiguous()
        need = _lib.load().keep_linear_workspace_bytes(_E4M3, M, N, K)
        work = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        _lib.call("keep_linear_q8", xr.data_ptr(), x_ld, xs.data_ptr(), M, wr.data_ptr(), w_ld, ws.data_ptr(), N, K,
                  ops._ptr(b), 0 if b is None else ops._DT[b.dtype], act, ops._ptr(r),
                  0 if r is None else ops._DT[r.dtype], out.data_ptr(), ops._DT[od], ops._ptr(work), need,
                  ops._stream(device))
        return out if flat else out.view(shape)
