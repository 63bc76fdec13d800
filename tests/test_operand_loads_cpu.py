"""Kernels launched as programmatic dependents are resident while earlier kernels of the stream still write their operands, so none of them
may read through the read-only path (ld.global.nc, __ldg, const __restrict__ parameters), which is only defined for data that nobody writes
while the kernel lives. Checked on the sources, since a stale line rarely shows."""
import glob
import os
import re

import pytest

from conftest import ROOT

FILES = sorted(glob.glob(os.path.join(ROOT, "sglang_b200", "csrc", "*.cu*")))


def code(path):
    return re.sub(r"//[^\n]*", "", open(path).read())


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_no_load_takes_the_read_only_path(path):
    assert not re.search(r"__ldg\s*\(|ld\.global(?:\.\w+)*\.nc\b", code(path))


@pytest.mark.parametrize("path", FILES, ids=os.path.basename)
def test_dependents_have_no_read_only_parameters(path):
    for kernel in re.split(r"(?=\b__global__\b)", code(path))[1:]:
        head, body = kernel[:kernel.index(") {")], kernel[kernel.index(") {"):]
        body = body[:body.index("\n}")]
        if re.search(r"grid_dependency_(?:wait|zero)\(\)", body):
            assert not re.search(r"const\s+\w+\s*\*\s*__restrict__", head), head


def test_operand_loads_stay_behind_the_wait():
    """The compiler keeps volatile assembly in order, so neither the wait nor the loads may be anything else."""
    text = code(os.path.join(ROOT, "sglang_b200", "csrc", "common.cuh"))
    assert re.search(r'asm volatile\("griddepcontrol\.wait;" ::: "memory"\)', text)
    loads = re.findall(r"(?:ld_operand|ld_stream_16)\(const \w+\*? ?\*? ?p\) \{(.*?)\n\}", text, re.S)
    assert len(loads) == 4 and all("asm volatile(" in b for b in loads)
