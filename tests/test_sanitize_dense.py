"""AddressSanitizer and UndefinedBehaviorSanitizer run of the dense products', the adapters', the combine's and the plan's
entry points on the CPU (``tests/sanitize/dense_probe.cpp``): argument checks only, nothing is launched. The build is
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
             ("abi.cpp", "plan.hip", "plan_dev.h", "combine.hip", "common.h", "dense.hip", "dense_dev.h", "dense_gemm.h",
              "dense_gemm.hip", "dense_outer.h", "lora.hip", "plan_blocks.hip")),
           ROOT / "include" / "keep_amd.h", ROOT / "tests" / "sanitize" / "dense_probe.cpp",
           ROOT / "tests" / "sanitize" / "build_dense.sh"]


def test_argument_checks_under_asan_and_ubsan():
    if not Path(HIPCC).exists() or shutil.which("gcc") is None:
        pytest.skip("hipcc and gcc are needed for the sanitizer builds")
    h = hashlib.sha256()
    for p in SOURCES:
        h.update(p.name.encode())
        h.update(p.read_bytes())
    stamp, exe = OUT / "dense.sha256", OUT / "dense_probe"
    if not (stamp.exists() and stamp.read_text() == h.hexdigest() and exe.exists()):
        stamp.unlink(missing_ok=True)
        res = subprocess.run(["bash", str(ROOT / "tests" / "sanitize" / "build_dense.sh"), str(OUT)],
                             capture_output=True, text=True, timeout=1200)
        assert res.returncode == 0, res.stderr[-4000:]
        stamp.write_text(h.hexdigest())
    # the HIP runtime keeps allocations until exit: leak reports would be its own
    r = subprocess.run([str(exe)], capture_output=True, text=True, timeout=300,
                       env={**os.environ, "ASAN_OPTIONS": "detect_leaks=0:verify_asan_link_order=0"})
    assert r.returncode == 0 and "ok: 0 failures" in r.stdout, (r.stdout[-2000:], r.stderr[-4000:])
    assert "runtime error" not in r.stderr and "AddressSanitizer" not in r.stderr
