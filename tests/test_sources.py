"""Rules of the kernels' sources that no run would show broken."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parents[1] / "moe-gemm-parallel-bench_b200" / "csrc"
SOURCES = sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])


def code(path: Path) -> str:
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", path.read_text(), flags=re.S)


@pytest.mark.parametrize("path", SOURCES, ids=lambda p: p.name)
def test_kernels_that_start_early_read_by_ordinary_loads(path):
    """A kernel that waits for the grid before it (grid_dependency_wait) may be
    resident while that grid writes its inputs.  Non-coherent loads need memory
    that nothing writes during the kernel, and a pointer declared unaliased lets
    the compiler choose them."""
    text = code(path)
    if "grid_dependency_wait();" not in text:
        return
    found = re.findall(r"__ldg\b|__restrict__|\bld\.global[\w:.]*\.nc\b", text)
    assert not found, f"{path.name}: {sorted(set(found))}"
