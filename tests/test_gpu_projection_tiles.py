"""Dense projections on every tile that their plan may choose, in each of the three products, with summed indexes that end
with a step and inside one, and with tiles cut at both sides (``test_projection_plan.py`` asks that none is left out)."""

import pytest
import torch

import keep_amd
from tests import test_gpu_projection as tp
from tests.bounded import Bounded

pytestmark = pytest.mark.gpu
F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16

HALF = [  # M, N, K: 16-bit rows
    (19, 18, 10), (20, 64, 8), (64, 20, 8), (17, 17, 64), (300, 72, 333),  # 64 x 64
    (19, 17, 3200), (17, 17, 2892), (17, 2880, 12), (20, 2614, 8), (4224, 21, 9), (2528, 22, 9),  # ... in slices
    (7168, 265, 320), (6848, 308, 200), (260, 320, 6959), (325, 200, 6851), (320, 277, 7104), (200, 3520, 663),  # 128, two groups
    (135, 7296, 6720), (145, 6152, 7215), (6120, 6592, 144), (6336, 6372, 137),  # ... in slices
    (528, 6592, 320), (1287, 3132, 200), (410, 320, 8298), (438, 200, 8337), (320, 6563, 518), (200, 529, 7232),  # 128 x 128
    (6528, 779, 320), (6210, 894, 200), (4032, 320, 1297), (6656, 200, 822), (320, 5093, 1044), (200, 704, 8128),  # 256 x 128
    (6990, 1878, 192), (3648, 4254, 200), (5634, 192, 2346), (7168, 200, 1856), (192, 8064, 1587), (200, 4629, 3104),  # 256 x 256
]
FLOAT = [  # float32 rows
    (25, 18, 8), (17, 32, 9), (32, 18, 9), (20, 19, 32), (300, 72, 333),
    (17, 24, 1312), (20, 19, 1377), (20, 2528, 8), (18, 1528, 13), (1280, 32, 8), (1459, 19, 10),
    (7278, 386, 160), (992, 3126, 100), (387, 160, 7520), (330, 100, 8864), (160, 4992, 596), (100, 7433, 420),
    (6752, 1026, 160), (2270, 3332, 99), (864, 160, 8256), (3424, 100, 2131), (160, 983, 7214), (100, 3776, 1944),
]
EIGHT = [  # 8-bit rows
    (17, 17, 128), (22, 16, 16), (19, 17, 2688), (18, 16, 3424), (7040, 267, 640), (640, 4096, 528), (138, 7815, 6784),
    (6784, 131, 6480), (6656, 546, 640), (778, 4666, 528), (6517, 804, 640), (5843, 1060, 528),
]


def _run(dev, dtype, M, N, K):
    tp._check(tp._case(dev, dtype, M, N, K, bias=F32, residual=dtype, seed=N), "silu")
    torch.cuda.empty_cache()  # (the float64 references of the larger ones)


@pytest.mark.parametrize("dtype", [F16, BF16])
@pytest.mark.parametrize("M, N, K", HALF)
def test_16_bits(dev, dtype, M, N, K):
    _run(dev, dtype, M, N, K)


@pytest.mark.parametrize("M, N, K", FLOAT)
def test_float32(dev, M, N, K):
    _run(dev, F32, M, N, K)


@pytest.mark.parametrize("M, N, K", EIGHT)
def test_8_bits(dev, M, N, K):
    x, xs, w, ws = tp._q8(dev, M, N, K)
    want = tp._q8_expected(x, xs, w, ws)
    b, r = torch.randn(N, device=dev), torch.randn(M, N, device=dev)
    both = Bounded(r) + tp._act(want + Bounded(b.expand(M, -1)), "silu")
    both.round(F32).check(keep_amd.linear_q8(x, xs, w, ws, b, activation="silu", residual=r))
    torch.cuda.empty_cache()
