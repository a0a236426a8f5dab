"""A kernel that takes tensor memory lets the kernel behind it start (mb_grid_dep_launch) only when it has its own.  That kernel allocates
before it waits for this one (mb_grid_dep_wait): if it came first on an SM, this one's allocation could wait for columns that are not given
back before it has ended itself."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "mace_b200", "csrc")


def _kernels(name):
    """The bodies of a source's kernels, comments taken out."""
    with open(os.path.join(CSRC, name)) as f:
        text = re.sub(r"//[^\n]*|/\*.*?\*/", "", f.read(), flags=re.S)
    bodies = []
    for start in [m.start() for m in re.finditer(r"__global__", text)]:
        at = text.index("{", start)
        depth = 0
        for end in range(at, len(text)):
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            if depth == 0:
                break
        bodies.append(text[at:end])
    return bodies


SOURCES = sorted(n for n in os.listdir(CSRC) if n.endswith((".cu", ".cuh")) and any("tmem_alloc" in b for b in _kernels(n)))


def test_the_kernels_are_found():
    assert {"gemm_mxfp4.cu", "gemm_u8_tc.cuh", "conv_u8.cu", "gemm_f32_tc.cu", "conv_f32_direct.cu"} <= set(SOURCES)


@pytest.mark.parametrize("name", SOURCES)
def test_allocation_comes_first(name):
    for body in _kernels(name):
        taken = [m.start() for m in re.finditer(r"tmem_alloc(_pair)?\s*\(", body)]
        if not taken:
            continue
        started = [m.start() for m in re.finditer(r"mb_grid_dep_launch\s*\(", body)]
        assert len(started) == 1 and started[0] > max(taken)
