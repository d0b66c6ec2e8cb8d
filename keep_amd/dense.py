"""Routed products with dense expert weights, with their gradients.

``gather_mm`` is ``gather_vqmm`` for experts that stay unquantised: the same
token and per-route layouts, out-of-range routes as NaN rows, output in ``x``'s
dtype. Few routes are grouped inside the kernel and stream each hit expert's
weights once (``keep_gather_mm``); more run over a device route plan. ``x`` and
``weight`` share one float dtype; sums are float32.

Both operands are differentiable (token layout): ``dx[t] = sum_j W[e]^T dy[t, j]``
and ``dW[e] = sum dy x^T`` over the expert's routes, in float32 and in a fixed
order. A route out of range gives NaN in its token's ``dx`` too and no share in
``dW``.
"""

from __future__ import annotations

import torch
from torch.autograd.function import once_differentiable

from keep_amd import _grad, _lib, ops

ROUTE_TILE = 16  # routes per tile of the planned kernel
# Routes the kernel groups by itself: as many as its ballots hold; a plan costs 6 us and more on top.
WINDOW_ROUTES = 128
# Routes from which a plan takes several workgroups: 18 us either way at 16384; 25 against 13 at 32768, 54 against 13 at
# 65536.
PLAN_BLOCKS_ROUTES = 16384


class _Plan:
    """A device route plan in one allocation, as pointers."""

    def __init__(self, rhs: torch.Tensor, groups: int, tile: int):
        R = rhs.numel()
        n = min((R + tile - 1) // tile + groups, R)
        room = (R + tile - 1) // tile + groups
        lib = _lib.load()
        blocks = R >= PLAN_BLOCKS_ROUTES
        scratch = lib.keep_route_plan_blocks_workspace_bytes(R, groups) // 4 if blocks else 0
        self.buffer = torch.empty(2 * R + 2 * groups + 3 * room + 1 + scratch, dtype=torch.int32, device=rhs.device)
        p = self.buffer.data_ptr()
        self.order, inverse = p, p + 4 * R
        self.counts = p + 8 * R
        self.offsets = self.counts + 4 * groups
        self.tile_expert = self.offsets + 4 * groups
        self.tile_offset = self.tile_expert + 4 * room
        self.tile_count = self.tile_offset + 4 * room
        self.valid_tiles = self.tile_count + 4 * room
        self.n_tiles = n  # descriptors that can hold routes: those come first
        self.tile = tile
        args = (rhs.data_ptr(), R, groups, tile, self.order, inverse, self.counts, self.offsets, self.tile_expert,
                self.tile_offset, self.tile_count, room, self.valid_tiles)
        if blocks:
            _lib.call("keep_route_plan_blocks", *args, self.valid_tiles + 4, 4 * scratch, ops._stream(rhs.device))
        else:
            _lib.call("keep_route_plan", *args, ops._stream(rhs.device))


def _weight_layout(weight: torch.Tensor) -> tuple[torch.Tensor, bool]:
    """The weights as ``[E, N, K]`` memory, or (True) as ``[E, K, N]`` memory under a transposed view."""

    if weight.is_contiguous():
        return weight, False
    if weight.transpose(1, 2).is_contiguous():
        return weight, True
    return weight.contiguous(), False


def _launch(x, weight, transposed: bool, rhs, lhs, routes: int, x_div: int, N: int, K: int, plan: _Plan | None,
            out) -> torch.Tensor:
    if plan is None:
        tiles = (None,) * 7 + (0, 0)
    else:
        tile = plan.tile
        if tile != ROUTE_TILE and not _gemm_takes(x, weight, transposed, N, K, tile):
            plan = _Plan(rhs, weight.shape[0], ROUTE_TILE)
        tiles = (plan.order, plan.offsets, plan.counts, plan.tile_expert, plan.tile_offset, plan.tile_count,
                 plan.valid_tiles, plan.n_tiles, plan.tile)
    _lib.call("keep_gather_mm", x.data_ptr(), ops._DT[x.dtype], x.shape[0], weight.data_ptr(), int(transposed),
              rhs.data_ptr(), ops._ptr(lhs), routes, x_div, weight.shape[0], N, K, *tiles, out.data_ptr(),
              ops._DT[out.dtype], ops._stream(x.device))
    return out


def _gemm_takes(x, weight, transposed: bool, N: int, K: int, tile: int) -> bool:
    return (x.data_ptr() % 16 == 0 and weight.data_ptr() % 16 == 0
            and bool(_lib.load().keep_gather_mm_tile_supported(ops._DT[x.dtype], int(transposed), N, K, tile)))


def _tile(routes: int, experts: int) -> int:
    """Routes per tile of the plan, by the routes an expert gets on average.

    A small tile leaves out less of a partly filled one, a large one reads the weights fewer times. Microseconds of bf16
    products for tiles of 16 / 64 / 128 / 256:
    128 experts 7168 -> 2048: mean 1: 441 / 455 / 466 / 601; 2: 567 / 531 / 608 / 802; 4: 708 / 605 / 674; 32: 1990 /
    638 / 718 / 908; 64: - / 765 / 706 / 748; 96: - / 815 / 774 / 801; 128: - / 1077 / 1040 / 849; 192: - / 1363 / 1199 / 942.
    256 experts 4096 -> 2048: mean 1: 434 / 477 / 489; 2: 618 / 689; 4: 749 / 767 / 861; 8: 893 / 772 / 813.
    """

    mean = routes / experts
    return 16 if mean < 2 else 64 if mean < 48 else 128 if mean < 100 else 256


def _forward(x: torch.Tensor, weight: torch.Tensor, rhs: torch.Tensor, lhs: torch.Tensor | None, x_div: int):
    """``([R, N], plan or None)``."""

    E, N, K = weight.shape
    R = rhs.numel()
    out = torch.empty((R, N), dtype=x.dtype, device=x.device)
    if R == 0:
        return out, None
    w, transposed = _weight_layout(weight)
    plan = _Plan(rhs, E, _tile(R, E)) if R > WINDOW_ROUTES and E <= ops.PLAN_EXPERTS else None
    return _launch(x, w, transposed, rhs, lhs, R, x_div, N, K, plan, out), plan


class _GatherMM(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, rhs, k):
        xc = x.contiguous()
        out, plan = _forward(xc, weight, rhs, None, k)
        ctx.save_for_backward(xc, weight, rhs)
        ctx.plan, ctx.k = plan, k
        return out

    @staticmethod
    @once_differentiable
    def backward(ctx, dy):
        x, weight, rhs = ctx.saved_tensors
        x, rhs = x.contiguous(), rhs.contiguous()  # a saved-tensor hook may give back other strides
        with ops._on(x.device):
            return (*_backward(x, weight, rhs, ctx.plan, ctx.k, dy.contiguous(), ctx.needs_input_grad), None, None)


def _backward(x, weight, rhs, plan, k: int, dy, needs):
    E, N, K = weight.shape
    R = rhs.numel()
    dx = dw = None
    if plan is None and R and E <= ops.PLAN_EXPERTS and (needs[1] or R > WINDOW_ROUTES):
        plan = _Plan(rhs, E, _tile(R, E))
    if needs[0]:
        if R == 0:
            dx = torch.zeros_like(x)
        else:
            w, transposed = _weight_layout(weight)
            # routes of a token are added in float32 and rounded once
            rows = torch.empty((R, K), dtype=x.dtype if k == 1 else torch.float32, device=x.device)
            _launch(dy, w, not transposed, rhs, None, R, 1, K, N, plan, rows)
            dx = rows if k == 1 else ops._sum_routes(rows, k, x.dtype)
    if needs[1]:
        if R == 0:
            dw = torch.zeros((E, N, K), dtype=weight.dtype, device=x.device)
        else:
            dw = torch.empty((E, N, K), dtype=weight.dtype, device=x.device)
            _lib.call("keep_gather_mm_grad_weight", x.data_ptr(), ops._DT[x.dtype], x.shape[0], dy.data_ptr(), R, k, E,
                      N, K, plan.order, plan.offsets, plan.counts, dw.data_ptr(), ops._stream(x.device))
    return dx, dw


def gather_mm(x: torch.Tensor, weight: torch.Tensor, rhs_indices, *, lhs_indices=None,
              validate_indices: bool = False) -> torch.Tensor:
    """Routed product with dense expert weights ``weight [E, N, K]`` (contiguous, or a transposed view of contiguous
    ``[E, K, N]``; other strides are copied).

    Token layout: ``x [T, K]``, ``rhs_indices [T, k]`` -> ``[T, k, N]``, differentiable in ``x`` and ``weight`` (a
    gradient of ``weight`` needs ``E <= 1024``). Per-route layout: ``lhs_indices`` and ``rhs_indices`` of R routes ->
    ``[R, N]``, without gradients (index ``x`` and use the token layout with ``k = 1``). Indices out of range give NaN
    rows; ``validate_indices`` checks them on the host (it syncs).
    """

    device = ops._dense_device(x, weight)
    if x.ndim != 2:
        raise ValueError(f"x must be 2D [tokens, hidden], found {tuple(x.shape)}")
    if weight.ndim != 3 or 0 in weight.shape:
        raise ValueError(f"weight must be 3D [experts, out, in], none of them 0, found {tuple(weight.shape)}")
    if x.dtype != weight.dtype or x.dtype not in ops._DT:
        raise ValueError("x and weight must share a dtype of float32, float16 or bfloat16, found "
                         f"{x.dtype} and {weight.dtype}")
    E, N, K = weight.shape
    if x.shape[1] != K:
        raise ValueError(f"x trailing dimension must be {K}, found {x.shape[1]}")
    rhs = ops._index_tensor(rhs_indices, device)
    lhs = None if lhs_indices is None else ops._index_tensor(lhs_indices, device).reshape(-1)
    grad = _grad.wanted(x, weight)
    if lhs is not None:
        rhs = rhs.reshape(-1)
        if lhs.shape != rhs.shape:
            raise ValueError("lhs_indices and rhs_indices must have the same flattened shape")
        if grad:
            raise ValueError("gather_mm has gradients in the token layout only: index x and pass rhs_indices [T, 1]")
        shape, k = (rhs.numel(), N), 1
    else:
        if rhs.ndim != 2 or rhs.shape[0] != x.shape[0]:
            raise ValueError(f"rhs_indices must be [tokens, top_k] with {x.shape[0]} tokens, found {tuple(rhs.shape)}")
        k = rhs.shape[1]
        shape = (x.shape[0], k, N)
    if rhs.numel() and x.shape[0] == 0:
        raise ValueError("x holds no rows")
    if validate_indices:
        ops._host_check_indices("rhs_indices", rhs, E)
        if lhs is not None:
            ops._host_check_indices("lhs_indices", lhs, x.shape[0])
    with ops._on(device):
        if not grad:
            return _forward(x.contiguous(), weight, rhs, lhs, max(k, 1))[0].view(shape)
        if weight.requires_grad and E > ops.PLAN_EXPERTS:
            raise ValueError(f"a gradient of weight needs at most {ops.PLAN_EXPERTS} experts, found {E}")
        _grad.check_capture(x, weight)
        return _grad.mark(_GatherMM.apply(x, weight, rhs, max(k, 1))).view(shape)
