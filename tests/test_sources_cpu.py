"""Rules that the kernels' sources keep and that no run shows."""
import glob
import os
import re

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "mixedgemm_b200", "csrc")


def code_of(path):
    """The file without its comments."""
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", open(path).read(), flags=re.S)


SOURCES = sorted(glob.glob(os.path.join(CSRC, "*.cu")) + glob.glob(os.path.join(CSRC, "*.cuh")))
OVERLAPPED = [s for s in SOURCES if "grid_dep_wait" in code_of(s)]


def test_the_overlapped_kernels_are_found():
    names = {os.path.basename(s) for s in OVERLAPPED}
    assert {"gemm.cu", "int8_gemm.cu", "norm_quant.cu", "reorder.cu", "calibrate.cu", "ptx_sm100.cuh"} <= names


@pytest.mark.parametrize("source", OVERLAPPED, ids=os.path.basename)
def test_overlapped_kernels_read_nothing_through_the_read_only_path(source):
    """A kernel that is launched programmatically is resident while the kernel before it may still write.  The
    read-only path is defined for data that does not change while the kernel is resident, so none of its
    spellings may stand in these files."""
    code = code_of(source)
    for spelling in (r"__ldg\s*\(", r"\bld\.global(\.\w+)*\.nc\b", r"__restrict__"):
        assert not re.search(spelling, code), spelling
