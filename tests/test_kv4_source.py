"""CPU: what holds for the source of the 4-bit K/V cache's kernels."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "madi_b200", "csrc")


@pytest.mark.parametrize("name", ["kv4.cu", "kv4_attn.cu", "kv4_flash.cu"])
def test_no_read_only_loads_of_memory_that_the_kernel_before_writes(name):
    """The kernels start while the one before them still runs, and wait for it inside (pdl_wait).  A
    const __restrict__ pointer (or __ldg, ld.global.nc) promises the compiler that its memory is constant
    for the kernel's lifetime, which then is not so."""
    src = open(os.path.join(CSRC, name)).read()
    src = re.sub(r"//[^\n]*", "", src)
    assert "pdl_wait()" in src
    for word in ("__restrict__", "__ldg", "ld.global.nc", "ldg_nc_"):
        assert word not in src, word
