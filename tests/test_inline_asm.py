"""Inline assembly of the kernels: M0, which many instructions read without naming it, is set by the compiler."""

import re
from pathlib import Path

CSRC = Path(__file__).resolve().parents[1] / "keep_amd" / "csrc"


def test_no_statement_writes_m0_behind_the_compilers_back():
    found = []
    for path in sorted([*CSRC.glob("*.hip"), *CSRC.glob("*.h")]):
        for m in re.finditer(r"\basm\s*(?:volatile)?\s*\((.*?)\);", path.read_text(), re.S):
            template = m.group(1).split(":", 1)[0]
            if re.search(r"\bm0\b", template):
                found.append(f"{path.name}: {template.strip()}")
    assert not found
