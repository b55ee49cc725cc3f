"""CPU: the order of two instructions in every kernel that allocates tensor memory.  A dependent kernel that becomes resident beside a CTA may allocate tensor memory too and then
keeps it while it waits for that CTA's whole kernel; were it let in ahead of the CTA's own allocation, each could wait for the other for good (an allocation is no bounded
wait).  So dependents are released behind the allocation.  Such a hang is not provoked; the sources are read instead."""
import glob
import os
import re

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "lumi_b200", "csrc")


def kernels():
    """(file, body) of every __global__ function."""
    for path in sorted(glob.glob(os.path.join(CSRC, "*.cu*"))):
        text = re.sub(r"//[^\n]*", "", open(path).read())
        for piece in text.split("__global__")[1:]:
            start, depth = piece.index("{"), 0
            for end in range(start, len(piece)):
                depth += {"{": 1, "}": -1}.get(piece[end], 0)
                if depth == 0:
                    break
            yield os.path.basename(path), piece[start:end]


WITH_TMEM = [(f, b) for f, b in kernels() if "tcgen05.alloc" in b]


def test_there_are_such_kernels():
    assert len(WITH_TMEM) >= 6 and {f for f, _ in WITH_TMEM} >= {"gemm_i8.cu", "gemm_tcgen05.cu", "gemm_few_rows.cu", "gemm_rows_f32.cu"}


@pytest.mark.parametrize("f,body", WITH_TMEM, ids=["%s-%d" % (f, i) for i, (f, _) in enumerate(WITH_TMEM)])
def test_dependents_are_released_behind_the_allocation(f, body):
    release = [m.start() for m in re.finditer(r"griddepcontrol\.launch_dependents|pdl_release\(\)|pdl_launch_dependents\(\)", body)]
    alloc = [m.start() for m in re.finditer(r"tcgen05\.alloc", body)]
    barrier = body.find("tc_fence_after()", alloc[-1])        # every thread of the CTA is behind the allocation here
    assert barrier > 0
    assert all(r > barrier for r in release), f


@pytest.mark.parametrize("f,body", WITH_TMEM, ids=["%s-%d" % (f, i) for i, (f, _) in enumerate(WITH_TMEM)])
def test_one_verdict_on_an_earlier_timeout(f, body):
    """A kernel that does no work after a wait ran out elsewhere decides it once for all threads of a CTA: the word may change while they look, and warps that part over it would allocate
    tensor memory, or read it, with half their lanes."""
    for line in body.split("\n"):
        if "& STATUS_TIMEOUT" in line:
            assert "__syncthreads_or(" in line or re.match(r"\s*(tl\.|\*)skip = ", line), (f, line)      # (skip: one thread's word in shared memory)
