"""Low-rank adapters of many requests at once beside a shared projection.

``gather_lora`` adds each row's own adapter to the projection's output,
``out[r] = base[r] + s[a] (x[r] A[a]^T) B[a]^T`` with ``a = indices[r]`` (negative:
no adapter; past the end: a NaN row), in two launches whatever the mix of
requests (``keep_lora``). Rows of one adapter lie together in a batch of requests;
scattered ones are right too, but read its factors once each. It is differentiable in ``x``, ``A``, ``B`` and
``base``. ``LoraAdapters`` holds the adapters of a layer: a dense projection
(``QuantizedVQLinear``) or routed experts, one adapter per expert
(``SwitchLinear``, ``QuantizedVQSwitchLinear``). Adapters of a lower rank than
the layer's are padded with zeros.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from keep_amd import _grad, _lib, ops

MAX_RANK = 128
# Routes (2D indices) from which a plan brings the routes of one adapter together first: rows of a request lie together
# as they are, its routes' experts do not. Microseconds without and with one, routes of random adapters, bf16, in a graph: 32
# adapters of r = 16, 2048 -> 1024: 128 routes 10 / 16, 256 12 / 22, 512 26 / 20, 4096 135 / 30; 64 of r = 32, 4096 -> 2048:
# 128 routes 16 / 19, 256 26 / 26, 512 57 / 26, 4096 327 / 52.
PLANNED_ROUTES = 256


def _forward(x, a, b, scales, idx, x_div: int, base, out_dtype, t_out=None) -> torch.Tensor:
    n, rank, K = a.shape
    R, N, device = idx.numel(), b.shape[1], x.device
    out = torch.empty((R, N), dtype=out_dtype, device=device)
    if R == 0:
        return out
    dt, od = ops._DT[x.dtype], ops._DT[out_dtype]
    grouped = int(x_div > 1 and R >= PLANNED_ROUTES and n <= ops.PLAN_EXPERTS)
    need = _lib.load().keep_lora_workspace_bytes(dt, R, n, rank, K, grouped)
    ws = torch.empty(need, dtype=torch.uint8, device=device)
    _lib.call("keep_lora", x.data_ptr(), dt, x.shape[0], a.data_ptr(), b.data_ptr(), ops._ptr(scales), idx.data_ptr(), R,
              x_div, n, rank, K, N, ops._ptr(base), od, ops._ptr(t_out), grouped, ws.data_ptr(), need, out.data_ptr(), od,
              ops._stream(device))
    return out


class _GatherLora(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, a, b, base, scales, idx, x_div, out_dtype):
        x, a, b = x.contiguous(), a.contiguous(), b.contiguous()
        # the scaled low-rank rows, for B's gradient
        t = torch.empty((idx.numel(), _lib.load().keep_lora_rank_stride(a.shape[1])), dtype=torch.float32,
                        device=x.device)
        ctx.base_shape = None if base is None else base.shape
        out = _forward(x, a, b, scales, idx, x_div, None if base is None else base.contiguous(), out_dtype, t)
        ctx.save_for_backward(x, a, b, scales, idx, t)
        ctx.x_div = x_div
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, a, b, scales, idx, t = _grad.saved(ctx)
        nx, na, nb, nbase = ctx.needs_input_grad[:4]
        (n, rank, K), N, R, device = a.shape, b.shape[1], idx.numel(), x.device
        make = torch.empty_like if R else torch.zeros_like
        # a float32 output over 16-bit rows: its gradient keeps its bits and range, so the products are float32's
        dtype, wide = x.dtype, dy.dtype != x.dtype and bool(R and (nx or na or nb))
        if wide:
            x, a, b = x.float(), a.float(), b.float()
        dx, da, db = (make(t_) if need else None for t_, need in ((x, nx), (a, na), (b, nb)))
        if R and (nx or na or nb):
            g, dt = dy.contiguous(), ops._DT[x.dtype]
            planned = int(na or nb or (ctx.x_div > 1 and R >= PLANNED_ROUTES and n <= ops.PLAN_EXPERTS))
            with ops._on(device):
                need = _lib.load().keep_lora_backward_workspace_bytes(dt, R, ctx.x_div, n, rank, K, N, int(nx), planned)
                ws = torch.empty(need, dtype=torch.uint8, device=device)
                _lib.call("keep_lora_backward", x.data_ptr(), dt, x.shape[0], a.data_ptr(), b.data_ptr(),
                          ops._ptr(scales), idx.data_ptr(), R, ctx.x_div, n, rank, K, N, t.data_ptr(), g.data_ptr(),
                          ops._ptr(dx), ops._ptr(da), ops._ptr(db), planned, ws.data_ptr(), need, ops._stream(device))
        if wide:
            dx, da, db = (None if g is None else g.to(dtype) for g in (dx, da, db))
        return dx, da, db, dy.reshape(ctx.base_shape) if nbase else None, None, None, None, None


def gather_lora(x: torch.Tensor, lora_a: torch.Tensor, lora_b: torch.Tensor, indices, *,
                base: torch.Tensor | None = None, scales: torch.Tensor | None = None,
                validate_indices: bool = False) -> torch.Tensor:
    """Each row's own low-rank adapter: ``x [T, K]``, ``lora_a [n, r, K]``, ``lora_b [n, N, r]`` (``r <= 128``).

    ``indices [T]`` -> ``[T, N]``; ``indices [T, k]`` (an adapter per route of a token) -> ``[T, k, N]``. ``base`` (of
    the output's shape) is added, in float32 with one rounding; the output has its dtype, without it ``x``'s. ``scales``
    (``[n]``, kept in float32) multiplies each adapter and takes no gradient. Gradients of the factors need
    ``n <= 1024``; over a float32 ``base`` they are formed in float32 and rounded once. The low-rank row is float32,
    and enters the second product with 22 bits (fp16) or 24.
    """

    device = ops._dense_device(x, lora_a, lora_b, base)
    if x.ndim != 2:
        raise ValueError(f"x must be 2D [tokens, hidden], found {tuple(x.shape)}")
    if lora_a.ndim != 3 or lora_b.ndim != 3 or 0 in lora_a.shape or 0 in lora_b.shape:
        raise ValueError(f"lora_a and lora_b must be [adapters, rank, in] and [adapters, out, rank], found "
                         f"{tuple(lora_a.shape)} and {tuple(lora_b.shape)}")
    n, rank, K = lora_a.shape
    N = lora_b.shape[1]
    if lora_b.shape[0] != n or lora_b.shape[2] != rank:
        raise ValueError(f"lora_b must be [{n}, out, {rank}], found {tuple(lora_b.shape)}")
    if rank > MAX_RANK:
        raise ValueError(f"the rank must be at most {MAX_RANK}, found {rank}")
    if x.dtype not in ops._DT or lora_a.dtype != x.dtype or lora_b.dtype != x.dtype:
        raise ValueError("x, lora_a and lora_b must share a dtype of float32, float16 or bfloat16, found "
                         f"{x.dtype}, {lora_a.dtype} and {lora_b.dtype}")
    if x.shape[1] != K:
        raise ValueError(f"x trailing dimension must be {K}, found {x.shape[1]}")
    idx = ops._index_tensor(indices, device)
    if idx.ndim not in (1, 2) or idx.shape[0] != x.shape[0]:
        raise ValueError(f"indices must be [{x.shape[0]}] or [{x.shape[0]}, top_k], found {tuple(idx.shape)}")
    x_div = idx.shape[1] if idx.ndim == 2 else 1
    shape = (*idx.shape, N)
    if base is not None and (tuple(base.shape) != shape or base.dtype not in (x.dtype, torch.float32)):
        raise ValueError(f"base must have shape {shape} in {x.dtype} or float32, found {tuple(base.shape)} "
                         f"in {base.dtype}")
    if scales is not None:
        if _grad.wanted(scales):
            raise ValueError("scales take no gradient")
        if tuple(scales.shape) != (n,):
            raise ValueError(f"scales must have shape ({n},), found {tuple(scales.shape)}")
        scales = ops._to_dev(scales.detach(), device, torch.float32)
    if validate_indices and idx.numel() and int(idx.max()) >= n:
        raise ValueError(f"indices must be below {n}, found {int(idx.max())}")
    od = x.dtype if base is None else base.dtype
    with ops._on(device):
        if not _grad.wanted(x, lora_a, lora_b, base):
            return _forward(x.contiguous(), lora_a.contiguous(), lora_b.contiguous(), scales, idx, max(x_div, 1),
                            None if base is None else base.contiguous(), od).view(shape)
        if (lora_a.requires_grad or lora_b.requires_grad) and n > ops.PLAN_EXPERTS:
            raise ValueError(f"gradients of the factors need at most {ops.PLAN_EXPERTS} adapters, found {n}")
        _grad.check_capture(x, lora_a, lora_b, base)
        return _grad.mark(_GatherLora.apply(x, lora_a, lora_b, base, scales, idx, max(x_div, 1), od)).view(shape)


class LoraAdapters:
    """The adapters of one layer, a row of factors per adapter: ``a [n, r, K]``, ``b [n, N, r]`` for a dense
    projection; ``a [n, E, r, K]``, ``b [n, E, N, r]`` for routed experts. ``scales [n]`` (e.g. alpha / r);
    routed experts' are copied here, once."""

    def __init__(self, a: torch.Tensor, b: torch.Tensor, scales: torch.Tensor | None = None):
        if a.ndim not in (3, 4) or b.ndim != a.ndim or a.shape[:-2] != b.shape[:-2] or a.shape[-2] != b.shape[-1]:
            raise ValueError("adapters must be a [n, r, K] and b [n, N, r], or with experts a [n, E, r, K] and "
                             f"b [n, E, N, r], found {tuple(a.shape)} and {tuple(b.shape)}")
        if not 1 <= a.shape[-2] <= MAX_RANK:
            raise ValueError(f"the rank must be in 1..{MAX_RANK}, found {a.shape[-2]}")
        if scales is not None and tuple(scales.shape) != (a.shape[0],):
            raise ValueError(f"scales must have shape ({a.shape[0]},), found {tuple(scales.shape)}")
        self.a, self.b, self.scales = a, b, scales
        self.num_adapters, self.rank = a.shape[0], a.shape[-2]
        self.num_experts = a.shape[1] if a.ndim == 4 else None
        self.input_dims, self.output_dims = a.shape[-1], b.shape[-2]
        # a scale per (adapter, expert), laid out once
        self._scales = scales if scales is None or a.ndim == 3 else scales.detach().repeat_interleave(a.shape[1])

    def check(self, layer) -> None:
        experts = getattr(layer, "num_experts", None)
        if self.num_experts != experts:
            raise ValueError("a dense projection takes adapters a [n, r, K]" if experts is None else
                             f"routed experts take adapters a [n, {experts}, r, K]")
        if self.input_dims != layer.input_dims or self.output_dims != layer.output_dims:
            raise ValueError(f"adapters map {self.input_dims} -> {self.output_dims}, the layer "
                             f"{layer.input_dims} -> {layer.output_dims}")

    def add(self, base: torch.Tensor, x: torch.Tensor, adapter_indices, experts: torch.Tensor | None = None):
        """``base`` plus the adapters of ``x``'s rows: ``x [T, K]``, ``adapter_indices [T]``; with ``experts [T, k]``
        the adapters of every route."""

        idx = ops._index_tensor(adapter_indices, x.device)
        if tuple(idx.shape) != (x.shape[0],):
            raise ValueError(f"adapter_indices must hold one adapter per row ({x.shape[0]}), found {tuple(idx.shape)}")
        if experts is None:
            return gather_lora(x, self.a, self.b, idx, base=base, scales=self._scales)
        if self.scales is not None and _grad.wanted(self.scales):  # the copy has no graph
            raise ValueError("scales take no gradient")
        E = self.num_experts
        e = ops._index_tensor(experts, x.device)
        # a route without an expert has a NaN base row already
        none = (idx < 0)[:, None] | (e < 0) | (e >= E)
        flat = torch.where(none, -1, idx.clamp(max=self.num_adapters)[:, None] * E + e)
        return gather_lora(x, self.a.flatten(0, 1), self.b.flatten(0, 1), flat, base=base, scales=self._scales)
