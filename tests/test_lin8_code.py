"""The code that the library's own flags give for the int8 product: what the kernels rely
on and no language rule or compiler check holds. Needs hipcc, no GPU.

* The one row of x that a workgroup quantizes lies in dynamic LDS, which begins where
  the static LDS ends, and is read 16 bytes at a time: that end is a multiple of 16.
* Loads to LDS are written as statements, in which the compiler looks for no hazards. A
  memory instruction that reads a scalar register needs five wait states behind a vector
  instruction that wrote it; so none of their scalar operands may come from one closer.
"""
from __future__ import annotations

import os
import re
import shutil
import subprocess

import pytest

from crosslane_amd import _build

WAIT_STATES = 5


@pytest.fixture(scope="module")
def code(tmp_path_factory):
    if not shutil.which(_build.HIPCC):
        pytest.skip("no hipcc")
    out = str(tmp_path_factory.mktemp("lin8") / "lin8.s")
    subprocess.run([_build.HIPCC, *_build.CFLAGS, "-S", "--cuda-device-only", os.path.join(_build.CSRC, "xl_lin8.hip"), "-o", out],
                   check=True, capture_output=True)
    return open(out).read()


def test_the_quantized_row_is_aligned(code):
    # the type of x is the kernel's fourth template argument; int8 (3) has no such row
    sizes = re.findall(r"\.amdhsa_kernel (\S*lin8_rows_kernelILi\d+ELi\d+ELb[01]ELi([0-3])E\S*)\n\s*\.amdhsa_group_segment_fixed_size (\d+)", code)
    assert sorted(t for _, t, _ in sizes if t != "3") == ["0", "0", "1", "1", "2", "2"]
    for name, kind, size in sizes:
        assert kind == "3" or int(size) % 16 == 0, (name, size)
