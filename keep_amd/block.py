"""The steps either side of the routed experts on the GPU.

- ``rmsnorm_quant_rht``: RMSNorm, block-wise FP8 e4m3 activation quantisation
  and the forward RHT in one row pass (``keep_rmsnorm_quant_rht``): the
  block's ``ffn_norm`` (``src/ramp/models/deepseek_v4_flash_adapter.py:1794,1806``),
  ``act_quant`` (``scripts/runpod/v41_reap/torch_kernel.py:40-53``), whose
  values the serving step feeds to the experts
  (``scripts/v41_build/omlx_lattice.py:332,357``), and ``apply_rht_mx``
  (``src/keep/quant/rht.py:84-91``).
- ``rmsnorm``, ``rmsnorm_quant``: the residual's addition and RMSNorm in one row
  pass, any width, with gradients, or with the normed rows in 8 bits and their
  scales (``keep_rmsnorm``, ``keep_rmsnorm_quant``).
- ``combine_add``: the routed sum plus the shared expert plus the residual,
  rounded once (``keep_moe_combine_add``; ``deepseek_v4_flash_adapter.py:1784``,
  ``omlx_lattice.py:374-388``).
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from keep_amd import _grad, _lib
from keep_amd.ops import _DT, _dense_device, _on, _ptr, _stream

NORM_WIDTH = 16384  # values of a row that the norms serve

def rmsnorm_quant_rht(x: torch.Tensor, gamma: torch.Tensor | None = None, eps: float = 1e-6, *,
                      quant_block: int = 128, pow2_scales: bool = False, rht_signs=None, return_normed: bool = False,
                      out_dtype: torch.dtype | None = None, validate_signs: bool = True):
    """``y = RMSNorm(x)`` (rounded to ``x``'s dtype), ``q = act_quant(y)`` per
    ``quant_block`` values (0: none), ``out = RHT(q, rht_signs)`` (no signs: q).
    Returns ``out`` or ``(out, y)`` with ``return_normed``."""

    from keep_amd.rht import check_signs

    if not x.is_cuda:
        raise ValueError("rmsnorm_quant_rht needs a device tensor")
    if x.dtype not in _DT:
        raise ValueError(f"x must be float32, float16 or bfloat16, found {x.dtype}")
    n = x.shape[-1]
    if n < 64 or n > 8192 or n & (n - 1):
        raise ValueError(f"rows must hold a power of two of 64..8192 values, found {n}")
    if quant_block and (quant_block < 16 or quant_block > min(1024, n) or quant_block & (quant_block - 1)):
        raise ValueError(f"quant_block must be 0 or a power of two in 16..{min(1024, n)}, found {quant_block}")
    od = out_dtype or x.dtype
    if od not in _DT:
        raise ValueError(f"unsupported output dtype {od}")
    g = None
    if gamma is not None:
        g = gamma.to(device=x.device).contiguous()
        if g.dtype not in _DT:
            g = g.float()
        if tuple(g.shape) != (n,):
            raise ValueError(f"gamma must have shape ({n},), found {tuple(g.shape)}")
    s = None
    if rht_signs is not None:
        s = torch.as_tensor(rht_signs, device=x.device).to(torch.float32).contiguous()
        if tuple(s.shape) != (n,):
            raise ValueError(f"rht_signs must have shape ({n},), found {tuple(s.shape)}")
        if validate_signs:
            check_signs(s)
    xc = x.contiguous()
    rows = xc.numel() // n
    out = torch.empty(x.shape, dtype=od, device=x.device)
    normed = torch.empty(x.shape, dtype=x.dtype, device=x.device) if return_normed else None
    _lib.call("keep_rmsnorm_quant_rht", xc.data_ptr(), _DT[xc.dtype], rows, n, None if g is None else g.data_ptr(),
              _DT[g.dtype] if g is not None else 0, float(eps), int(quant_block), int(bool(pow2_scales)),
              None if s is None else s.data_ptr(), None if normed is None else normed.data_ptr(), out.data_ptr(),
              _DT[od], _stream(x.device))
    return (out, normed) if return_normed else out


def _norm_args(x, weight, eps: float, residual) -> torch.device:
    device = _dense_device(x, weight, residual)
    if x.dtype not in _DT:
        raise ValueError(f"x must be float32, float16 or bfloat16, found {x.dtype}")
    if x.ndim < 1 or not 1 <= x.shape[-1] <= NORM_WIDTH:
        raise ValueError(f"rows must hold 1..{NORM_WIDTH} values, found {tuple(x.shape)}")
    if weight is not None and (tuple(weight.shape) != (x.shape[-1],) or weight.dtype not in _DT):
        raise ValueError(f"weight must have shape ({x.shape[-1]},) in a float dtype, found {tuple(weight.shape)} in "
                         f"{weight.dtype}")
    if residual is not None and (residual.shape != x.shape or residual.dtype not in (x.dtype, torch.float32)):
        raise ValueError(f"residual must have x's shape {tuple(x.shape)} in {x.dtype} or float32, found "
                         f"{tuple(residual.shape)} in {residual.dtype}")
    if not eps >= 0:
        raise ValueError(f"eps must be non-negative, found {eps}")
    return device


def _rmsnorm(x, weight, eps: float, residual, keep_rstd: bool):
    """``(y, h, rstd)`` of contiguous rows; h is x without a residual."""

    n = x.shape[-1]
    rows = x.numel() // n
    y = torch.empty_like(x)
    h = x if residual is None else torch.empty_like(residual)
    rstd = torch.empty(rows, dtype=torch.float32, device=x.device) if keep_rstd else None
    if rows:
        _lib.call("keep_rmsnorm", x.data_ptr(), _DT[x.dtype], _ptr(residual),
                  0 if residual is None else _DT[residual.dtype], rows, n, _ptr(weight),
                  0 if weight is None else _DT[weight.dtype], eps, None if residual is None else h.data_ptr(),
                  y.data_ptr(), _ptr(rstd), _stream(x.device))
    return y, h, rstd


class _RmsNorm(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, residual, weight, eps):
        y, h, rstd = _rmsnorm(x, weight, eps, residual, True)
        ctx.save_for_backward(h, weight, rstd)
        ctx.set_materialize_grads(False)
        return y if residual is None else (y, h)

    @staticmethod
    @once_differentiable
    def backward(ctx, dy, dh=None):
        h, weight, rstd = _grad.saved(ctx)
        nx, nr, nw = ctx.needs_input_grad[:3]
        if dy is None:  # h alone was used
            return dh if nx else None, dh if nr else None, torch.zeros_like(weight) if nw else None, None
        n = h.shape[-1]
        rows, same = h.numel() // n, dy.dtype == h.dtype
        g = dy.contiguous()
        dh = None if dh is None else dh.contiguous()
        dx = torch.empty_like(g) if nx or (nr and same) else None
        dr = torch.empty_like(h) if nr and not same else dx if nr else None  # one tensor where both are the same values
        dw = (torch.empty_like if rows else torch.zeros_like)(weight) if nw else None
        if rows and (nx or nr or nw):
            with _on(h.device):
                need = _lib.load().keep_rmsnorm_grad_workspace_bytes(rows, n) if nw else 0
                ws = torch.empty(need, dtype=torch.uint8, device=h.device) if nw else None
                _lib.call("keep_rmsnorm_grad", h.data_ptr(), _DT[h.dtype], g.data_ptr(), _DT[g.dtype], _ptr(dh),
                          rstd.data_ptr(), rows, n, _ptr(weight), 0 if weight is None else _DT[weight.dtype], _ptr(dx),
                          None if same else _ptr(dr), _ptr(dw), _ptr(ws), need, _stream(h.device))
        return dx if nx else None, dr, dw, None


def rmsnorm(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6, *,
            residual: torch.Tensor | None = None):
    """``y = h / sqrt(mean(h^2) + eps) * weight`` over the last axis (1..16384 values), in ``x``'s dtype.

    Without ``residual`` ``h = x``, and ``y`` is returned. With it (``x``'s shape, in ``x``'s dtype or float32)
    ``h = residual + x`` rounded to its dtype, the new residual stream, and ``(y, h)`` are returned: the norm is of the
    rounded stream. ``weight [n]`` of any float dtype. The squares' sum is float32's: values beyond 1e19 overflow it, and
    the row is 0. Differentiable in ``x``, ``residual`` and ``weight``; the gradients
    of ``x`` and a ``residual`` of its dtype are the same values, in one tensor."""

    device = _norm_args(x, weight, eps, residual)
    with _on(device):
        xc = x.contiguous()
        w = None if weight is None else weight.contiguous()
        r = None if residual is None else residual.contiguous()
        if not _grad.wanted(x, weight, residual):
            y, h, _ = _rmsnorm(xc, w, float(eps), r, False)
            return y if r is None else (y, h)
        _grad.check_capture(x, weight, residual)
        out = _RmsNorm.apply(xc, r, w, float(eps))
        _grad.mark(out if r is None else out[0])
        return out


def rmsnorm_quant(x: torch.Tensor, weight: torch.Tensor | None = None, eps: float = 1e-6, *,
                  residual: torch.Tensor | None = None, quant_block: int = 128, pow2_scales: bool = False):
    """``rmsnorm`` with its rows in 8 bits: ``(q, scales)``, with a residual ``(q, scales, h)``.

    ``q`` (``torch.float8_e4m3fn``, ``x``'s shape) times ``scales`` (float32 ``[..., ceil(n / quant_block)]``) are the
    normed values, rounded once. ``quant_block`` (a power of two in 16..512) neighbouring values share a scale,
    ``max(max |y|, 1e-4) / 448``, with ``pow2_scales`` the next power of two: ``act_quant``'s
    (``torch_kernel.py:40-53``). ``linear_q8`` reads blocks of 128. No gradients."""

    device = _norm_args(x, weight, eps, residual)
    if not 16 <= quant_block <= 512 or quant_block & (quant_block - 1):
        raise ValueError(f"quant_block must be a power of two in 16..512, found {quant_block}")
    if _grad.wanted(x, weight, residual):
        raise ValueError("8-bit rows have no gradient: use rmsnorm, or call this without recording")
    n = x.shape[-1]
    rows = x.numel() // n
    with _on(device):
        xc = x.contiguous()
        w = None if weight is None else weight.contiguous()
        r = None if residual is None else residual.contiguous()
        q = torch.empty(x.shape, dtype=torch.float8_e4m3fn, device=device)
        scales = torch.empty((*x.shape[:-1], (n + quant_block - 1) // quant_block), dtype=torch.float32, device=device)
        h = None if r is None else torch.empty_like(r)
        if rows:
            _lib.call("keep_rmsnorm_quant", xc.data_ptr(), _DT[xc.dtype], _ptr(r), 0 if r is None else _DT[r.dtype], rows,
                      n, _ptr(w), 0 if w is None else _DT[w.dtype], float(eps), quant_block, int(bool(pow2_scales)),
                      _ptr(h), q.data_ptr(), scales.data_ptr(), _stream(device))
    return (q, scales) if r is None else (q, scales, h)


def combine_add(routed: torch.Tensor, shared: torch.Tensor | None = None, residual: torch.Tensor | None = None,
                out_dtype: torch.dtype | None = None) -> torch.Tensor:
    """``round_out(residual + (routed + shared))`` with fp32 sums; ``routed`` is float32. Differentiable: every
    term's gradient is the output's, in its dtype."""

    if routed.dtype != torch.float32 or not routed.is_cuda:
        raise ValueError("routed must be a float32 device tensor")
    for name, t in (("shared", shared), ("residual", residual)):
        if t is not None and (tuple(t.shape) != tuple(routed.shape) or t.dtype not in _DT):
            raise ValueError(f"{name} must match routed's shape {tuple(routed.shape)} in a float dtype")
    od = out_dtype or (residual.dtype if residual is not None else torch.float32)
    with _on(routed.device):
        if not _grad.wanted(routed, shared, residual):
            return _combine_add(routed, shared, residual, od)
        _grad.check_capture(routed, shared, residual)
        return _grad.mark(_CombineAdd.apply(routed, shared, residual, od))


def _combine_add(routed, shared, residual, od: torch.dtype) -> torch.Tensor:
    r = routed.contiguous()
    sh = None if shared is None else shared.contiguous()
    rs = None if residual is None else residual.contiguous()
    out = torch.empty(routed.shape, dtype=od, device=routed.device)
    _lib.call("keep_moe_combine_add", r.data_ptr(), None if sh is None else sh.data_ptr(),
              _DT[sh.dtype] if sh is not None else 0, None if rs is None else rs.data_ptr(),
              _DT[rs.dtype] if rs is not None else 0, r.numel(), out.data_ptr(), _DT[od], _stream(routed.device))
    return out


class _CombineAdd(torch.autograd.Function):
    @staticmethod
    def forward(ctx, routed, shared, residual, od):
        ctx.dtypes = [None if t is None else t.dtype for t in (routed, shared, residual)]
        return _combine_add(routed, shared, residual, od)

    @staticmethod
    def backward(ctx, dout):
        return (*(None if dt is None or not need else dout.to(dt)
                  for dt, need in zip(ctx.dtypes, ctx.needs_input_grad)), None)
