"""Launch plans of the operators of sequence models (mmp_plan.h), compiled for
the host."""
import ctypes
import os
import shutil
import subprocess

import numpy as np
import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "macmetalpy_amd",
                    "csrc")
SOURCE = r"""
#include "mmp_plan.h"
extern "C" {
long long t_group_lds(long long rows) { return 4 * mmpi::group_bins(rows) * mmpi::group_waves(rows); }
int t_groups(long long n, long long rows) {
  return mmpi::in_groups(n, rows) + mmpi::in_one_group_pass(n, rows);
}
int t_row_passes(long long rows) { return mmpi::row_passes(rows); }
// extents as triples (from, to, written)
int t_overlap(const long long *e, int n) {
  mmpi::Extent x[64];
  for (int i = 0; i < n; ++i)
    x[i] = {(unsigned long long)e[3 * i], (unsigned long long)e[3 * i + 1], e[3 * i + 2] != 0};
  return mmpi::written_overlap(x, n);
}
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


def test_written_overlap(plans):
    """Against every pair of extents, one of which is written."""
    g = np.random.default_rng(5)
    seen = [0, 0]
    for _ in range(4000):
        n = int(g.integers(1, 12))
        at = g.integers(0, 60, n)
        e = [(int(a), int(a + g.integers(0, 9)), int(g.integers(0, 2))) for a in at]
        want = any((a[2] or b[2]) and max(a[0], b[0]) < min(a[1], b[1])
                   for i, a in enumerate(e) for b in e[:i])
        flat = (ctypes.c_longlong * (3 * n))(*[v for x in e for v in x])
        assert plans.t_overlap(flat, n) == want, e
        seen[want] += 1
    assert min(seen) > 500


def test_group_counters_fit(plans):
    """All row counts that are ordered in groups: counters of every row for each
    wave within 64 KiB, and filling more than half of it where they are many."""
    i64 = ctypes.c_longlong
    plans.t_group_lds.restype = i64
    for rows in {*range(1, 5000), *range(5000, (1 << 20) + 1, 509),
                 *(b + k for b in (1 << 18, 1 << 19, 1 << 20) for k in (-257, -256, -1, 0, 1))}:
        if plans.t_groups(i64(1), i64(rows)):
            lds = plans.t_group_lds(i64(rows))
            assert lds <= 64 << 10 and (lds > 32 << 10 or rows <= 1 << 17), rows
    assert plans.t_groups(i64(1 << 17), i64(1 << 20)) == 1 and plans.t_groups(i64(1), i64(1 << 20)) == 2
    assert not plans.t_groups(i64(1 << 17), i64((1 << 20) + 1))
    assert not plans.t_groups(i64((1 << 17) + 1), i64(5))
    for rows, most in ((1 << 18, 16_384), ((1 << 18) + 1, 8192), (1 << 19, 8192), ((1 << 19) + 1, 4096)):
        assert plans.t_groups(i64(most), i64(rows)) == 2 and plans.t_groups(i64(most + 1), i64(rows)) == 1
