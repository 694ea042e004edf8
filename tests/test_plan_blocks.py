"""Launch plans of ``cp.nn``'s block operators (mmp_plan.h), compiled for the host:
the choice against the times of all, measured."""
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
void t_prod16(long long m, long long n, int slabs, int *out) {
  const mmpi::Prod16Plan p = mmpi::prod16_plan(m, n, slabs, 256);
  out[0] = p.tile;
  out[1] = p.parts;
}
void t_projections(int elem, long long m, long long n, int slabs, int *out) {
  const mmpi::ProjectionsPlan p = mmpi::projections_plan(elem, m, n, slabs, 256);
  out[0] = p.rows;
  out[1] = p.parts;
}
void t_delta(long long heads, int values, int keys, int chunks, int *out) {
  const mmpi::DeltaPlan p = mmpi::delta_plan(heads, values, keys, chunks, 256);
  out[0] = p.segments;
  out[1] = p.span;
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


def chosen(f, *args):
    out = (ctypes.c_int * 2)()
    f(*(ctypes.c_longlong(a) if i in wide else ctypes.c_int(a) for i, a in enumerate(args)
        for wide in (f.wide,)), out)
    return tuple(out)


@pytest.mark.parametrize("rows,dim,hidden,times", [
    (8, 2048, 5632, {(256, 1): 45, (256, 4): 21, (128, 1): 23.4, (128, 2): 16.6, (128, 4): 14.6, (128, 8): 17.9}),
    (64, 1024, 4096, {(256, 1): 24.9, (128, 1): 11.9, (128, 2): 12.4, (128, 4): 12.9, (128, 8): 17.9}),
    (200, 2048, 2048, {(256, 1): 44.2, (256, 8): 24.1, (128, 1): 18.9, (128, 2): 17.7, (128, 4): 17.9, (128, 8): 22}),
    (512, 1024, 1024, {(256, 1): 26.9, (128, 1): 12, (128, 2): 15.2, (128, 4): 14.1}),
    (1024, 1024, 4096, {(256, 1): 31.4, (128, 1): 22.9, (128, 2): 51.9}),
    (1999, 1008, 2504, {(256, 1): 32.6, (128, 1): 39, (256, 2): 60.2}),
    (2048, 4096, 4096, {(256, 1): 112.2, (128, 1): 133.3, (256, 2): 151}),
    (4096, 512, 1024, {(256, 1): 19.6, (128, 1): 13.9, (128, 2): 43.2})])
def test_float16_products(plans, rows, dim, hidden, times):
    plans.t_prod16.wide = (0, 1)
    got = chosen(plans.t_prod16, rows, 2 * hidden, -(-dim // 64))
    assert times[got] <= 1.12 * min(times.values()), got


@pytest.mark.parametrize("rows,dim,hidden,times", [
    (515, 771, 1030, {(128, 1): 99.9, (128, 4): 51.6, (32, 1): 44.4, (32, 2): 38.6, (32, 4): 36.6, (32, 8): 41.3}),
    (81, 3849, 3558, {(128, 1): 484, (128, 8): 108, (32, 1): 221, (32, 2): 132, (32, 4): 96, (32, 8): 82}),
    (4032, 105, 11130, {(128, 1): 294, (128, 2): 725, (32, 1): 299}),
    (9123, 145, 176, {(128, 1): 21.2, (32, 1): 19.3, (32, 2): 36.1}),
    (2048, 2048, 2048, {(128, 1): 282, (128, 2): 322, (32, 1): 355}),
    (8, 2048, 2048, {(128, 1): 162, (128, 8): 29, (32, 1): 38, (32, 2): 24, (32, 4): 15.7, (32, 8): 14.8, (32, 16): 17}),
    (300, 300, 300, {(128, 1): 33, (32, 1): 11.1, (32, 2): 12.3})])
def test_projections(plans, rows, dim, hidden, times):
    plans.t_projections.wide = (1, 2)
    got = chosen(plans.t_projections, 4, rows, hidden, -(-dim // 32))
    assert times[got] <= 1.2 * min(times.values()), got


@pytest.mark.parametrize("heads,values,keys,chunks,times", [
    (8, 2, 2, 64, {1: 218, 2: 200, 4: 125, 8: 94, 16: 105, 32: 152}),
    (8, 2, 2, 512, {1: 1726, 2: 1427, 4: 770, 8: 452, 16: 371, 32: 420}),
    (16, 1, 1, 32, {1: 97, 2: 90, 4: 62, 8: 51, 16: 55, 32: 74}),
    (64, 2, 2, 16, {1: 78, 2: 117, 4: 139}),
    (5, 2, 2, 25, {1: 161, 2: 152, 4: 101, 7: 80, 8: 80, 16: 86}),
    (1, 4, 4, 32, {1: 222, 2: 200, 4: 146, 8: 157, 16: 207}),
    (128, 2, 2, 32, {1: 202, 2: 382, 4: 428})])
def test_delta_segments(plans, heads, values, keys, chunks, times):
    plans.t_delta.wide = (0,)
    segments, span = chosen(plans.t_delta, heads, values, keys, chunks)
    assert times[segments] <= 1.1 * min(times.values()), segments
    # every chunk is in one segment, and no segment is empty
    assert (segments - 1) * span < chunks <= segments * span


def test_no_heads(plans):
    plans.t_delta.wide = (0,)
    for args in ((0, 1, 1, 5), (3, 0, 1, 5), (3, 1, 1, 0), (3, 1, 1, 1)):
        segments, span = chosen(plans.t_delta, *args)
        assert segments == 1 and span >= 1
