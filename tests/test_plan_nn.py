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
int t_window(long long n, long long rows, int lanes) {
  return mmpi::row_window(n, lanes, mmpi::long_rows_whole(n, rows, lanes));
}
int t_whole(long long n, long long rows, int lanes) { return mmpi::long_rows_whole(n, rows, lanes); }
int t_recur(int back, int elem, long long batch, long long steps, long long dim) {
  return back ? mmpi::recur_grad_form(elem, batch, steps, dim) : mmpi::recur_form(elem, batch, steps, dim);
}
int t_past(int arrays, int elem, long long batch, long long steps, long long dim) {
  return mmpi::recur_past_caches(arrays, elem, batch, steps, dim);
}
// out: lanes, held vectors, parts
void t_loss(int grad, int elem, long long rows, long long classes, int may_split, int *out) {
  const mmpi::LossPlan p = mmpi::loss_plan(grad != 0, elem, rows, classes, 256, may_split != 0);
  out[0] = p.lanes;
  out[1] = p.held;
  out[2] = p.parts;
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


def _i64(*v):
    return tuple(ctypes.c_longlong(x) for x in v)


@pytest.mark.parametrize("n,rows,dim,elem,times", [
    (131_072, 5000, 8, 2, {16: 60, 32: 69, 64: 85}), (59_961, 478, 113, 2, {16: 45, 32: 58, 64: 72}),
    (131_072, 60_000, 128, 2, {16: 53, 32: 50, 64: 56}), (131_072, 64_000, 1024, 2, {16: 132, 32: 121, 64: 120}),
    (524_288, 60_000, 8, 2, {16: 95, 32: 92, 64: 106}), (800_000, 500, 77, 2, {16: 213, 32: 158, 64: 133})])
def test_windows_of_the_order(plans, n, rows, dim, elem, times):
    """The window that was quickest, or within a tenth of it."""
    lanes = 1
    while lanes < 256 and lanes * (16 // elem) < dim:
        lanes *= 2
    assert times[plans.t_window(*_i64(n, rows), lanes)] <= 1.1 * min(times.values())


@pytest.mark.parametrize("n,rows,lanes,whole,windows", [
    (2000, 30_000, 128, 30, 39), (8192, 30_000, 128, 42, 49), (4096, 2, 128, 27, 27),
    (16_384, 2, 128, 85, 32), (16_000, 200, 1, 25, 58), (16_000, 30_000, 128, 54, 56)])
def test_long_rows_whole_or_in_windows(plans, n, rows, lanes, whole, windows):
    got = whole if plans.t_whole(*_i64(n, rows), lanes) else windows
    assert got <= 1.1 * min(whole, windows)


THREADS, BRIEF, FEW, LONG, WIDE = range(5)
FORWARDS = [
    # float16
    (2, 1, 50_000, 100, {FEW: 36, LONG: 58, WIDE: 111}), (2, 1, 50_000, 300, {FEW: 43, LONG: 65, WIDE: 114}),
    (2, 1, 60_000, 1024, {FEW: 128, LONG: 96, WIDE: 122}), (2, 2, 16_000, 1024, {FEW: 60, LONG: 43, WIDE: 53}),
    (2, 4, 8000, 1024, {FEW: 59, LONG: 40, WIDE: 44}), (2, 16, 2000, 1024, {FEW: 58, LONG: 41, WIDE: 41}),
    (2, 64, 500, 1024, {FEW: 58, LONG: 40, WIDE: 39}),
    (2, 256, 256, 1021, {THREADS: 95, FEW: 168, LONG: 123, WIDE: 105}),
    (2, 256, 256, 1024, {THREADS: 86, WIDE: 83}), (2, 200, 200, 2000, {THREADS: 111, WIDE: 122}),
    (2, 200, 128, 1999, {THREADS: 76, WIDE: 76}), (2, 128, 500, 2048, {THREADS: 156, WIDE: 148}),
    (2, 100, 130, 1999, {THREADS: 32, WIDE: 57}), (2, 253, 170, 1390, {THREADS: 92, WIDE: 107}),
    (2, 281, 48, 2851, {BRIEF: 60, WIDE: 89}), (2, 100, 30, 1024, {BRIEF: 13, WIDE: 17}),
    # float32
    (4, 200, 130, 3000, {THREADS: 221, WIDE: 266}), (4, 200, 200, 2000, {THREADS: 218, WIDE: 186}),
    (4, 200, 90, 1999, {THREADS: 117, WIDE: 90}), (4, 4, 8000, 1024, {FEW: 145, LONG: 82, WIDE: 73}),
    (4, 3, 1999, 1001, {FEW: 37, LONG: 27, WIDE: 19}), (4, 16, 2000, 1024, {FEW: 147, LONG: 82, WIDE: 69}),
    (4, 1, 60_000, 1024, {FEW: 254, LONG: 157, WIDE: 146})]
BACKWARDS = [
    (2, 1, 50_000, 100, {FEW: 47, LONG: 66, WIDE: 227}), (2, 1, 50_000, 300, {FEW: 85, LONG: 78, WIDE: 218}),
    (2, 1, 60_000, 1024, {FEW: 285, LONG: 165, WIDE: 258}), (2, 2, 16_000, 1024, {FEW: 165, LONG: 95, WIDE: 108}),
    (2, 4, 8000, 1024, {FEW: 167, LONG: 94, WIDE: 89}), (2, 3, 1999, 1001, {FEW: 43, LONG: 31, WIDE: 27}),
    (2, 16, 2000, 1024, {FEW: 163, LONG: 91, WIDE: 80}), (2, 300, 2000, 64, {LONG: 98, WIDE: 277}),
    (2, 300, 2000, 32, {FEW: 60, LONG: 83}),
    (4, 1, 50_000, 100, {FEW: 56, LONG: 65, WIDE: 214}), (4, 1, 60_000, 1024, {FEW: 560, LONG: 291, WIDE: 302}),
    (4, 3, 1999, 1001, {FEW: 71, LONG: 53, WIDE: 34})]


@pytest.mark.parametrize("back,elem,batch,steps,dim,times",
                         [(0, *c) for c in FORWARDS] + [(1, *c) for c in BACKWARDS])
def test_recurrence_layouts(plans, back, elem, batch, steps, dim, times):
    """The layout that was quickest (us, as measured), or within a tenth of it."""
    assert times[plans.t_recur(back, elem, *_i64(batch, steps, dim))] <= 1.1 * min(times.values())


def test_recurrence_of_few_steps(plans):
    for elem in (2, 4, 8):
        for batch in (1, 200, 100_000):
            for dim in (1, 7, 1024, 5000):
                for steps in (0, 1, 15, 16):
                    for back in (0, 1):
                        assert plans.t_recur(back, elem, *_i64(batch, steps, dim)) == THREADS
                assert plans.t_recur(0, elem, *_i64(batch, 17, dim)) == BRIEF
                assert plans.t_recur(0, elem, *_i64(batch, 64, dim)) == BRIEF
                assert plans.t_recur(1, elem, *_i64(batch, 17, dim)) >= FEW
                assert plans.t_recur(0, elem, *_i64(batch, 5000, dim)) >= FEW


def test_recurrence_past_the_caches(plans):
    assert plans.t_past(3, 2, *_i64(16, 2048, 2048)) and plans.t_past(6, 2, *_i64(16, 2048, 2048))
    assert not plans.t_past(3, 2, *_i64(1, 30_000, 1024)) and not plans.t_past(6, 2, *_i64(1, 60_000, 500))
    assert plans.t_past(3, 8, *_i64(1 << 20, 1 << 20, 1 << 20))  # no 64 bit product


def _loss(plans, grad, elem, rows, classes, may_split=True):
    out = (ctypes.c_int * 3)()
    plans.t_loss(grad, elem, *_i64(rows, classes), int(may_split), out)
    return tuple(out)


@pytest.mark.parametrize("elem", [2, 4, 8])
def test_loss_layouts_hold_their_rows(plans, elem):
    """Threads and registers for a row wherever it begins, and no layout that
    is more than four times what it needs; parts that have vectors each."""
    for classes in [*range(1, 3000, 7), *(int(1.07 ** k) for k in range(118, 300)), 0x7FFF0000]:
        vecs = classes // (16 // elem) + 2
        worst = -(-(16 // elem - 1 + classes) // (16 // elem))  # the row begins at the last element
        for rows in (1, 2, 50, 170, 600, 10 ** 6):
            lanes, held, parts = _loss(plans, 1, elem, rows, classes)
            if parts:
                assert 3 <= parts and rows * parts <= 512 and vecs >= 1024 * parts >= 1024
                lanes, held, parts = _loss(plans, 1, elem, rows, classes, False)
            assert parts == 0 and worst <= vecs
            assert lanes * held >= vecs if held else vecs > 1024 * 16
            assert not held or lanes * held <= 32 or lanes * held < 4 * vecs
            lanes, held, parts = _loss(plans, 0, elem, rows, classes)
            if parts:
                assert 2 <= parts and rows * parts <= 512 and vecs >= 8192
                lanes, held, parts = _loss(plans, 0, elem, rows, classes, False)
            assert parts == 0 and held == 0 and lanes in (8, 16, 32, 64, 256, 512)
            assert lanes >= 64 or vecs <= 4 * lanes


def test_loss_parts(plans):
    """A few long rows: parts where two launches (13 us; 17 with the gradient) beat
    one workgroup a row, by its 16-byte vectors."""
    for vecs, alone, grad in ((4096, 10, 13), (6250, 12, 14), (12_500, 18, 18), (32_500, 32, 32)):
        for g, one, two in ((0, alone, 13), (1, grad, 17)):
            got = two if _loss(plans, g, 2, 1, vecs * 8)[2] else one
            assert got <= 1.1 * min(one, two)
    assert _loss(plans, 1, 2, 250, 16_250 * 8)[2] == 0
    assert _loss(plans, 1, 2, 60_000, 250)[0] == 16 and _loss(plans, 0, 2, 60_000, 250)[0] == 16
