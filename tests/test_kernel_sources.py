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


@pytest.mark.parametrize("name", ["cross_attn.cu", "int8_matmul.cu", "tc_gemm.cu", "tc_attn.cu"])
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


MEET = r"__syncwarp\(\)|__syncthreads\(\)|warp_wait\(|__any_sync\("
LANES = r"if \((?:!?mine|in\b|!in\b|move|mx > |lane == 0|i >= it\.rows|n \+ j)|n \+ j < a\.N \?"


def enclosing_loops(text, at):
    """Starts and ends of the braced loop bodies around a place, the innermost first."""
    found, depth, i = [], 0, at
    while i > 0:
        i -= 1
        if text[i] == "}":
            depth += 1
        elif text[i] == "{" and depth:
            depth -= 1
        elif text[i] == "{":
            if re.search(r"for \([^{};]*;[^{};]*;[^{};]*\)\s*$", text[max(0, i - 200):i]):
                end, d = i + 1, 1
                while d:
                    d += {"{": 1, "}": -1}.get(text[end], 0)
                    end += 1
                found.append((i, end))
    return found


@pytest.mark.parametrize("name,calls", [("cross_attn.cu", r"\b(?:tmem_ld32_raw|tmem_st16|ldm4t?)\("),
                                        ("int8_matmul.cu", r"\btmem_ld16\(|\bcluster_sync\(\)")])
def test_warps_are_whole_where_an_instruction_takes_one(name, calls):
    """Matrix loads, TMEM accesses and cluster barriers are executed by whole
    warps.  Behind a branch that lanes take apart, in the text before them or
    in an earlier turn of their loop, the lanes meet first; that the compiler brings
    them together there is not its duty."""
    text = source(name)
    seen = 0
    for m in re.finditer(calls, text):
        if text[text.rindex("\n", 0, m.start()):m.start()].strip().startswith("__device__"):
            continue  # the helper itself
        seen += 1
        before = text[:m.start()]
        body = before.rindex("\n}\n")  # the end of the function before this one
        met = max((x.end() for x in re.finditer(MEET, before)), default=-1)
        apart = max((x.end() for x in re.finditer(LANES, before)), default=-1)
        assert met > body and (apart < body or met > apart), before[-400:]
        for a, b in enclosing_loops(text, m.start()):
            if a < body:
                break
            last = [x.start() for x in re.finditer(LANES, text[a:b])]
            meets = [x.start() for x in re.finditer(MEET, text[a:b])]
            if last and last[-1] > m.start() - a:  # a branch behind it, before its next turn
                assert any(x < m.start() - a or x > last[-1] for x in meets), text[a:m.start()][-400:]
    assert seen


def test_every_device_function_is_called():
    text = "\n".join(source(f) for f in sorted(os.listdir(SRC)))
    made = r"__device__[^;{}()]*?\b%s\("
    for name in set(re.findall(made % r"(\w+)", text)):
        assert len(re.findall(r"\b%s\b" % name, text)) > len(re.findall(made % name, text)), name
