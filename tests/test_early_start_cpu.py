"""Kernels that start before their predecessor in the stream has ended read
nothing through the read-only path: the predecessor may still be writing it."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "silarray_b200", "csrc")


def code(path):
    """The source without its comments."""
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)


SOURCES = {os.path.basename(p): code(p) for p in sorted(glob.glob(os.path.join(CSRC, "*.cu*")))}
# whoever waits for its predecessor, and the headers that their kernels are made of
EARLY = [n for n, s in SOURCES.items() if "wait_for_previous()" in s or n in ("elem.cuh", "loss_epilogue.cuh", "tc_common.cuh")]


def test_the_early_kernels_are_found():
    assert {"layer_norm.cu", "grad_norm.cu", "cross_entropy.cu", "loss_gemm.cuh"} <= set(EARLY)


@pytest.mark.parametrize("name", EARLY)
def test_no_read_only_loads(name):
    # __ldcs and __ldcg may be moved by the compiler as any load of unchanging memory
    found = re.findall(r"__ldg\b|__ldc[agsv]\b|__restrict__|\.nc\b|__ldlu\b", SOURCES[name])
    assert not found, f"{name}: {found}"


@pytest.mark.parametrize("name", EARLY)
def test_inline_loads_of_global_memory_are_ordered(name):
    """Each is volatile and clobbers memory, so that it stays behind the wait."""
    for m in re.finditer(r"asm\s*(volatile)?\s*\(\s*\"ld\.global[^;]*;\"(.*?)\);", SOURCES[name], re.S):
        assert m.group(1) and '"memory"' in m.group(2), f"{name}: {m.group(0)}"
