"""Kernels here start while their predecessor in the stream still runs and wait for it inside (griddepcontrol.wait). What they
read from global memory may therefore be written during their own life, for which the read-only load path is not defined,
and which a compiler may move over the wait: a load through __ldg or ld.global.nc, and any read through a pointer declared
const __restrict__, from which the compiler makes such loads by itself. The sources must hold none of them."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "qgemm_b200", "csrc")
READ_ONLY = re.compile(r"\b__ldg\b|\b__ldcs\b|\bld\.global\.nc\b|\bconst\s+\w+\s*\*\s*__restrict__")


def code(name):
    with open(os.path.join(CSRC, name)) as f:
        text = f.read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


SOURCES = sorted(n for n in os.listdir(CSRC) if n.endswith((".cu", ".cuh")) and "pdl_" in code(n))


def test_the_sources_are_found():
    assert {"ptx.cuh", "gemm_launch.cuh", "quantize_block.cu", "gemm_e8m0.cuh", "splitk_reduce.cu"} <= set(SOURCES)


@pytest.mark.parametrize("name", SOURCES)
def test_no_read_only_loads(name):
    found = READ_ONLY.findall(code(name))
    assert not found, found
