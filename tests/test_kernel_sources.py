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


@pytest.mark.parametrize("name", ["cross_attn.cu", "int8_matmul.cu"])
def test_a_wait_that_ran_out_leaves_no_copy_in_flight(name):
    """A block that leaves while a TMA copy is on its way lets it write the shared
    memory of the next one: behind the loading loop every kernel waits for the
    stages it has requested, whether a wait ran out before that or not."""
    for kernel, body in kernels(name).items():
        loads = [m.start() for m in re.finditer(r"\btma_load_\dd(_pair)?\(", body)]
        drains = [m.start() for m in re.finditer(r"\bmbar_drain\(", body)]
        if loads:
            assert drains and drains[-1] > loads[-1], kernel
        if any("tma_load_2d_pair" in body[at:at + 16] for at in loads):
            # the copies of both blocks of a pair: after they have met, and they meet again
            met = [m.start() for m in re.finditer(r"\bcluster_sync\(\)", body)]
            assert any(a < drains[-1] < b for a, b in zip(met[1:], met[2:])), kernel


@pytest.mark.parametrize("name", ["cross_attn.cu", "int8_matmul.cu"])
def test_a_wait_that_ran_out_leaves_no_product_in_flight(name):
    """TMEM that is freed under a running MMA may be another block's when the sums
    arrive: a warp that gives up commits what it has issued and waits for that."""
    for kernel, body in kernels(name).items():
        issuers = len(re.findall(r"\bumma_commit(?:_pair)?_e\(&(?:tfull|s_full|pv_done)\[", body))
        given_up = len(re.findall(r"if \(!ok\) \{\s*umma_commit(?:_pair)?_e\((&?done[^)]*)\);\s*mbar_drain\(\1, 0\);", body))
        assert given_up == issuers, kernel
