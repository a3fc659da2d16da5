"""Rules of the kernels' text that no run may break to show them: a kernel that
broke one could hang the GPU."""
import os
import re

import pytest

from conftest import PKG_DIR

SRC = os.path.join(PKG_DIR, "csrc")


def source(name):
    """A file without its comments."""
    with open(os.path.join(SRC, name)) as f:
        return re.sub(r"/\*.*?\*/|//[^\n]*", "", f.read(), flags=re.S)


def kernels(name):
    """{kernel: body} of a file's __global__ functions."""
    text, found = source(name), {}
    for m in re.finditer(r"__global__\s+void\s+(?:__launch_bounds__\((?:[^()]|\([^()]*\))*\)\s*)?(\w+)\s*\(", text):
        at = text.index("{", m.end())
        depth, end = 1, at + 1
        while depth:
            depth += {"{": 1, "}": -1}.get(text[end], 0)
            end += 1
        found[m.group(1)] = text[at:end]
    assert found
    return found


@pytest.mark.parametrize("name", ["cross_attn.cu", "int8_matmul.cu"])
def test_tmem_is_held_before_the_next_kernel_may_start(name):
    """griddepcontrol.launch_dependents counts for a block from its first
    thread on.  A dependent kernel that starts before the block holds its TMEM
    may take the SM's and wait for this kernel's end: neither could go on.  So a
    barrier behind the allocation comes first."""
    for kernel, body in kernels(name).items():
        if "pdl_trigger()" not in body or "tcgen05.alloc" not in body:
            continue
        between = body[body.rindex("tcgen05.alloc"):body.index("pdl_trigger()")] if body.rindex("tcgen05.alloc") < body.index("pdl_trigger()") else ""
        assert "__syncthreads()" in between, kernel
