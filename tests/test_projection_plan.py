"""The GPU tests of the dense projections reach every tile that the plan may choose: each instantiation of the products (type,
product, tile, a summed index that ends inside a step or not), and its slices. The plan is linear.hip's own, built for the
host (``tests/sanitize/plan_probe.cpp``)."""

import os
import random
import shutil
import subprocess
from pathlib import Path

import pytest

from tests import test_gpu_projection_tiles as tiles

ROOT = Path(__file__).resolve().parents[1]
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
F32, F16, BF16, E4M3 = 0, 1, 2, 3
STEP = {F32: 32, F16: 64, BF16: 64, E4M3: 128}  # summed values of a step


@pytest.fixture(scope="module")
def plan(tmp_path_factory):
    if not Path(HIPCC).exists() or shutil.which("g++") is None:
        pytest.skip("hipcc and g++ are needed for the plan's probe")
    where = tmp_path_factory.mktemp("plan")
    obj, exe = where / "plan.o", where / "plan"
    for cmd in ([HIPCC, "-x", "hip", "-O0", "-fPIE", "-std=c++17", "--offload-host-only", "-I", str(ROOT / "include"), "-c",
                 str(ROOT / "tests" / "sanitize" / "plan_probe.cpp"), "-o", str(obj)],
                ["g++", str(obj), "-Wl,--unresolved-symbols=ignore-all", "-o", str(exe)]):
        res = subprocess.run(cmd, capture_output=True, text=True, timeout=600)
        assert res.returncode == 0, res.stderr[-4000:]

    def of(dtype, shapes):
        """For each M, N, K the (product, tile, in slices, ends inside a step) of its products; few rows: product and tile."""
        text = "".join(f"{dtype} {M} {N} {K} {int(dtype != E4M3)}\n" for M, N, K in shapes)
        out = subprocess.run([str(exe)], input=text, capture_output=True, text=True, timeout=300, check=True).stdout
        for (M, N, K), line in zip(shapes, out.splitlines()):
            v = list(map(int, line.split()))
            for mode, tile, slices in zip(v[::3], v[1::3], v[2::3]):
                yield (mode, tile) if tile == 0 else (mode, tile, slices > 1, (K, N, M)[mode] % STEP[dtype] != 0)
    return of


@pytest.mark.parametrize("dtype, shapes", [(F32, tiles.FLOAT), (F16, tiles.HALF), (BF16, tiles.HALF), (E4M3, tiles.EIGHT)])
def test_every_tile_is_tested(plan, dtype, shapes):
    rng, step = random.Random(0), STEP[dtype]

    def size(lo, hi):
        n = int(2 ** rng.uniform(lo, hi))
        return max(step, n // step * step) if rng.random() < 0.5 else n
    drawn = [(size(4.1, 13), size(4, 13), size(3, 13.2)) for _ in range(40000)]
    reached = set(plan(dtype, [s for s in drawn if s[0] > 16]))
    assert len(reached) >= {F32: 24, F16: 42, BF16: 42, E4M3: 12}[dtype]
    assert reached <= set(plan(dtype, shapes)), sorted(reached - set(plan(dtype, shapes)))


def test_few_rows_take_no_tile(plan):
    few = [(M, N, K) for M in (1, 16) for N in (1, 64, 8192) for K in (16, 4096)]
    for dtype in STEP:
        assert {k for k in plan(dtype, few) if k[0] == 0} == {(0, 0)}
