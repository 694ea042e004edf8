"""Launch plans of the operators of sequence models (mmp_plan.h), compiled for
the host."""
import ctypes
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "macmetalpy_amd",
                    "csrc")
SOURCE = r"""
#include "mmp_plan.h"
extern "C" {
int t_row_passes(long long rows) { return mmpi::row_passes(rows); }
}
"""


@pytest.fixture(scope="module")
def plans(tmp_path_factory):
    d = tmp_path_factory.mktemp("plan")
    src, so = str(d / "plan.cpp"), str(d / "plan.so")
    with open(src, "w") as f:
        f.write(SOURCE)
    cmd = [shutil.which("g++") or "g++", "-O2", "-std=c++17", "-Wall", "-Werror", "-shared", "-fPIC",
           f"-I{CSRC}", src, "-o", so]
    p = subprocess.run(cmd, capture_output=True, text=True)
    assert p.returncode == 0, p.stderr
    return ctypes.CDLL(so)


@pytest.mark.parametrize("rows", [1, 2, 255, 256, 257, 65_536, 65_537, 1 << 24, (1 << 24) + 1,
                                  20_000_000, 0x7fff0000, 1 << 32])
def test_row_passes_cover_the_rows_and_end(plans, rows):
    """As many passes of 8 bits as row numbers have, never one beyond the 32
    bits that they are held in."""
    got = plans.t_row_passes(ctypes.c_longlong(rows))
    assert got == max(1, -(-(rows - 1).bit_length() // 8)) <= 4
