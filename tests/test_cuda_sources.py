"""CPU: what the CUDA sources have to keep to wherever they are changed."""
from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "spikeinfer_b200" / "csrc"
SOURCES = sorted([*CSRC.glob("*.cu"), *CSRC.glob("*.cuh")])


@pytest.mark.parametrize("source", SOURCES, ids=lambda p: p.name)
def test_barriers_and_allocations_of_a_whole_warp_find_it_together(source):
    """The cluster's barriers and the tensor memory's allocation are .aligned: all lanes have to get there at once, and lanes that left a loop or a branch at different times
    need not.  The statement before each is a __syncwarp()."""
    lines = [line for line in source.read_text().splitlines() if line.strip() and not line.strip().startswith("//")]
    for i, line in enumerate(lines):
        if re.search(r'"(barrier\.cluster|tcgen05\.(de)?alloc)\S*\.aligned', line):
            assert line.strip().startswith("asm") and lines[i - 1].strip() == "__syncwarp();", f"{source.name}: {line.strip()}"
