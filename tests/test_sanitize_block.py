"""AddressSanitizer and UndefinedBehaviorSanitizer run of the norms', the choice of experts' and the dense projections'
entry points on the CPU (``tests/sanitize/block_probe.cpp``): argument checks only, nothing is launched. The build is
cached under ``keep_amd/_build/san`` and redone when a source changes."""

import hashlib
import os
import shutil
import subprocess
from pathlib import Path

import pytest

ROOT = Path(__file__).resolve().parents[1]
OUT = ROOT / "keep_amd" / "_build" / "san"
HIPCC = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
SOURCES = [*(ROOT / "keep_amd" / "csrc" / n for n in
             ("abi.cpp", "common.h", "dense_dev.h", "linear.hip", "linear_dev.h", "norm.hip", "norm_dev.h", "norm_grad.hip",
              "parts_dev.h", "route_dev.h", "route_experts.hip")),
           ROOT / "include" / "keep_amd.h", ROOT / "tests" / "sanitize" / "block_probe.cpp",
           ROOT / "tests" / "sanitize" / "build_block.sh"]


def test_argument_checks_under_asan_and_ubsan():
    if not Path(HIPCC).exists() or shutil.which("gcc") is None:
        pytest.skip("hipcc and gcc are needed for the sanitizer builds")
    h = hashlib.sha256()
    for p in SOURCES:
        h.update(p.name.encode())
        h.update(p.read_bytes())
    stamp, exe = OUT / "block.sha256", OUT / "block_probe"
    if not (stamp.exists() and stamp.read_text() == h.hexdigest() and exe.exists()):
        stamp.unlink(missing_ok=True)
        res = subprocess.run(["bash", str(ROOT / "tests" / "sanitize" / "build_block.sh"), str(OUT)],
                             capture_output=True, text=True, timeout=1200)
        assert res.returncode == 0, res.stderr[-4000:]
        stamp.write_text(h.hexdigest())
    # the HIP runtime keeps allocations until exit: leak reports would be its own
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "ASAN_OPTIONS": "detect_leaks=0:verify_asan_link_order=0"})
    assert r.returncode == 0 and "ok: 0 failures" in r.stdout, (r.stdout[-2000:], r.stderr[-4000:])
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr
