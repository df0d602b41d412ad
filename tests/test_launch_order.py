"""Order of a kernel's launch trigger and its tensor-memory allocation, from the sources. A kernel that lets its dependent in
(griddepcontrol.launch_dependents) before it has allocated may find tensor memory taken by that dependent, which waits for
this kernel to end while this one waits for the columns: neither goes on. No GPU."""

from __future__ import annotations

import re
from pathlib import Path

import pytest

CSRC = Path(__file__).resolve().parent.parent / "llm_inference_engine_b200" / "csrc"


def kernels():
    """(file, name, body without comments) of every kernel that allocates tensor memory."""
    found = []
    for path in sorted(CSRC.glob("*.cu")):
        text = re.sub(r"//[^\n]*", "", path.read_text())
        for start in re.finditer(r"__global__", text):
            at = text.index("{", start.end())
            depth, end = 0, at
            while True:
                depth += {"{": 1, "}": -1}.get(text[end], 0)
                end += 1
                if depth == 0:
                    break
            body = text[at:end]
            if "tmem_alloc(" in body:
                found.append((path.name, re.search(r"(\w+_kernel)\s*\(", text[start.start() : at])[1], body))
    return found


KERNELS = kernels()


def test_the_sources_have_such_kernels():
    assert {n for _, n, _ in KERNELS} >= {"skinny_tc_kernel", "gemm_tc_kernel", "fp8_gemm_kernel", "cache_attn_tc_kernel"}


@pytest.mark.parametrize("file,name,body", KERNELS, ids=[n for _, n, _ in KERNELS])
def test_dependents_come_in_behind_the_allocation(file, name, body):
    alloc = body.index("tmem_alloc(")
    triggers = [m.start() for m in re.finditer(r"griddep_launch_dependents\(\)", body)]
    assert triggers, "the next kernel never comes in early"
    for at in triggers:
        assert at > alloc, "the trigger stands ahead of the allocation"
        between = body[alloc:at]
        # the allocating warp itself, or any thread once the CTA has met
        assert "}" not in between or "__syncthreads()" in between, "another warp may trigger before the allocation is made"
