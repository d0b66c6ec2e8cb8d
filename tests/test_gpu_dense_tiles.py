"""The dense routed products over each size of tile that the plan's rule takes: more tiles than one round over the XCDs
holds, odd numbers of them, several blocks of columns, routes out of range, and weights in both layouts."""

import pytest
import torch

import keep_amd
from keep_amd import dense
from tests.bounded import Bounded
from tests.test_gpu_dense import _case, _expected

pytestmark = pytest.mark.gpu

# (tokens, experts, top_k, out, in), the tile the rule takes, and the least number of tiles that hold routes
SHAPES = [
    ((150, 128, 1, 72, 64), 16, 60),       # a tile per expert that is hit
    ((300, 24, 4, 264, 520), 128, 24),
    ((700, 60, 2, 520, 264), 64, 60),      # four rounds of turns, three blocks of columns and two of dx
    ((333, 41, 3, 600, 328), 64, 41),      # a last turn of one row of tiles
    ((2100, 67, 2, 264, 264), 128, 67),    # in runs
    ((5000, 33, 1, 300, 80), 256, 33),
    ((2100, 9, 2, 776, 520), 256, 9),
]


def _tiles(idx, experts, tile):
    counts = torch.bincount(idx[(idx >= 0) & (idx < experts)].long(), minlength=experts)
    return int(((counts + tile - 1) // tile).sum())


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("shape, tile, tiles", SHAPES)
def test_every_tile_size_and_its_gradients(dev, dtype, shape, tile, tiles, transposed):
    T, E, k = shape[:3]
    x, w, idx, dy = _case(dev, dtype, *shape, seed=11)
    assert dense._tile(T * k, E) == tile and T * k > dense.WINDOW_ROUTES
    assert _tiles(idx, E, tile) >= tiles * (0.9 if tile == 16 else 1)
    want = _expected(x, w, idx, dy)
    if transposed:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    x.requires_grad_(True), w.requires_grad_(True)
    out = keep_amd.gather_mm(x, w, idx)
    want[0].check(out, "out")
    dx, dw = torch.autograd.grad(out, (x, w), dy)
    want[1].check(dx, "dx")
    want[2].check(dw, "dw")


@pytest.mark.parametrize("transposed", [False, True])
@pytest.mark.parametrize("shape, tile, tiles", SHAPES)
def test_every_tile_size_with_routes_out_of_range(dev, shape, tile, tiles, transposed):
    """Whole tiles of routes without an expert among them (a quarter of all routes)."""
    T, E, k = shape[:3]
    x, w, idx, dy = _case(dev, torch.bfloat16, *shape, seed=12)
    g = torch.Generator(device=dev).manual_seed(13)
    bad = torch.rand(T, k, device=dev, generator=g) < 0.25
    got = idx.clone()
    got[bad] = torch.where(torch.rand(int(bad.sum()), device=dev, generator=g) < 0.5, -1, E + 7).int()
    want = _expected(x, w, idx, torch.where(bad[..., None], 0, dy))
    if transposed:
        w = w.transpose(1, 2).contiguous().transpose(1, 2)
    x.requires_grad_(True), w.requires_grad_(True)
    out = keep_amd.gather_mm(x, w, got)
    assert torch.isnan(out[bad]).all()
    Bounded(want[0].v[~bad], want[0].e[~bad]).check(out[~bad], "out")
    dx, dw = torch.autograd.grad(out, (x, w), dy)
    whole = ~bad.any(1)
    assert torch.isnan(dx[~whole]).all()
    Bounded(want[1].v[whole], want[1].e[whole]).check(dx[whole], "dx")
    want[2].check(dw, "dw")
