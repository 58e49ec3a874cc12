"""What the sources of the low-bit kernels have to say themselves, because no run shows reliably that it is missing."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "onmf_ontf_ndl_amd", "csrc")


def kernels(name):
    """(kernel, its body) of a source, comments taken out."""
    text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
    for m in re.finditer(r"__global__[^;{]*?(\w+_kernel)\s*\([^{;]*\)\s*\{", text):
        depth, at = 1, m.end()
        while depth:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
        yield m.group(1), text[m.end():at]


@pytest.mark.parametrize("name,least", [("dict4.hip", 1), ("keep8.hip", 2)])
def test_kernels_that_load_straight_to_lds_wait_for_it(name, least):
    """A barrier waits for no load to LDS: every barrier of such a kernel carries the wait for the loads in flight."""
    found = 0
    for kernel, body in kernels(name):
        if "global_load_lds" not in body:
            continue
        found += 1
        assert "__syncthreads" not in body, kernel
        barriers = re.findall(r'asm volatile\("([^"]*s_barrier)"', body)
        assert barriers and all("s_waitcnt vmcnt(" in b for b in barriers), kernel
    assert found >= least
