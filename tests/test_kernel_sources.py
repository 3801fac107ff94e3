"""Orders inside the kernels that no run can show, read from their sources."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "asc_devkit_b200", "csrc")
SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.cu")))


def kernels(path):
    """(name, body) of every __global__ function of a file."""
    text = re.sub(r"//[^\n]*", "", open(path).read())
    for m in re.finditer(r"__global__", text):
        start = text.index("{", text.index(")\n{", m.end()))
        depth, at = 0, start
        while True:
            depth += {"{": 1, "}": -1}.get(text[at], 0)
            at += 1
            if depth == 0:
                break
        yield re.findall(r"(\w+)\s*\(", text[m.end():start].replace("__launch_bounds__(", ""))[0], text[start:at]


@pytest.mark.parametrize("path", SOURCES, ids=os.path.basename)
def test_tensor_memory_is_taken_before_a_dependent_launch_is_let_in(path):
    """A dependent CTA on the same SM could take the columns that this one still waits for, and then wait for this launch's end:
    every thread has to know that the CTA has them (a barrier) before one triggers the dependent launch."""
    for name, body in kernels(path):
        take, trigger = body.find("tmem_alloc"), body.find("griddepcontrol.launch_dependents")
        if take < 0 or trigger < 0:
            continue
        assert take < trigger, name
        last = max(m.start() for m in re.finditer("tmem_alloc", body))
        assert "__syncthreads();" in body[last:trigger], name


def test_the_sources_hold_such_kernels():
    both = [name for path in SOURCES for name, body in kernels(path) if "tmem_alloc" in body and "launch_dependents" in body]
    assert {"low_rank_inner_kernel", "low_rank_outer_kernel"} <= set(both) and len(both) >= 3, both


def test_only_kernels_behind_a_cluster_barrier_write_a_partners_abort_flag():
    """A wait that gives up may raise the flag in the partner's shared memory only where a cluster barrier was passed first; until then nothing says that
    the partner runs."""
    for path in SOURCES:
        for name, body in kernels(path):
            waits = [m.start() for m in re.finditer(r"mbar_wait_bounded(_\w+)?\(", body)]  # (the form without a partner is mbar_wait_bounded<false>)
            if waits:
                assert 0 <= body.find("cluster_wait();") < waits[0], name


def test_every_device_helper_is_called():
    text = "".join(re.sub(r"//[^\n]*", "", open(p).read()) for p in glob.glob(os.path.join(CSRC, "*")) if p.endswith((".cu", ".cuh", ".h", ".cpp")))
    names = set(re.findall(r"__device__ __forceinline__ (?:const )?[\w:<>, ]+?[ *&]+(\w+)\(", text))
    assert len(names) > 100
    assert not [n for n in sorted(names) if len(re.findall(rf"\b{n}\b", text)) < 2]
