"""Where kernels may let their dependents start, read from the sources (what goes wrong cannot be run: it would hang a GPU).

A kernel's CTAs hold tensor memory from tcgen05.alloc on, which blocks while there is none.  A dependent that has started
allocates some itself and then waits for its predecessor to end: a predecessor's CTA that has not allocated by then may never.
So every kernel with an allocation signals its dependents only behind it and a barrier of the whole CTA."""
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "intel-extension-for-pytorch_b200", "csrc")


def kernels():
    found = []
    for name in sorted(os.listdir(CSRC)):
        if not name.endswith(".cu"):
            continue
        text = re.sub(r"//[^\n]*", "", open(os.path.join(CSRC, name)).read())
        for body in re.split(r"\b__global__\b", text)[1:]:
            if re.search(r"\btmem_alloc\(|\bpair_tmem_alloc\(", body) and "grid_launch_dependents()" in body:
                found.append((name, body))
    return found


def test_there_are_such_kernels():
    assert {"woq_kv4_prompt.cu", "woq_pair_tc.cu", "woq_i8_pair.cu", "woq_i8_block_tc.cu"} <= {name for name, _ in kernels()}


@pytest.mark.parametrize("name, body", kernels(), ids=[f"{n}-{i}" for i, (n, _) in enumerate(kernels())])
def test_dependents_start_behind_the_allocation(name, body):
    alloc = re.search(r"\b(?:pair_)?tmem_alloc\(", body).start()
    signal = body.index("grid_launch_dependents()")
    assert alloc < signal, name
    assert "__syncthreads()" in body[alloc:signal], name
