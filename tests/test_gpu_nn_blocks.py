"""``cp.nn``'s gated feed-forward product and dropout against plain NumPy in 64
bits.

Tolerances, all derived from the formulas: U is half a unit of the result's
type (its one rounding), E of the type that sums are held in, TINY half of the
smallest number that the result's type holds.
"""
import math

import numpy as np
import pytest
from scipy.special import erfc

import macmetalpy_amd as cp
from macmetalpy_amd import nn

pytestmark = pytest.mark.gpu

FLOATS = [np.float16, np.float32, np.float64]
U = {np.float16: 2.0 ** -11, np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
E = {np.float16: 2.0 ** -24, np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
TINY = {np.float16: 2.0 ** -25, np.float32: 2.0 ** -126, np.float64: 2.0 ** -1022}
by_name = {"ids": lambda v: getattr(v, "__name__", None) or str(v)}


def near(got, want, bound, dt):
    """Each element within `bound` and the rounding of the result's type."""
    assert got.dtype == dt
    got, want = got.get().astype(np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    off = np.abs(got - want) - (bound + (U[dt] * 1.001) * (np.abs(want) + bound) + TINY[dt])
    assert not off.size or np.nanmax(off) <= 0, f"off by {np.nanmax(off):.3g} more than the bound"
    assert np.array_equal(np.isnan(got), np.isnan(want))


# ---------------------------------------------------------- feed-forward
def activation(name, g):
    """a and a' in 64 bits."""
    if name == "gelu":
        phi = 0.5 * erfc(-g / math.sqrt(2.0))
        return g * phi, phi + g * np.exp(-0.5 * g * g) / math.sqrt(2.0 * math.pi)
    f = 1.0 / (1.0 + np.exp(-g))
    return (g * f, f + g * f * (1.0 - f)) if name == "silu" else (f, f * (1.0 - f))


# the largest |a'| and |a''| of each: silu 1.0999, 0.5; gelu 1.1290, 0.7979;
# sigmoid 0.25, 0.0963
SLOPE = {"silu": 1.1, "gelu": 1.13, "sigmoid": 0.25}
BEND = {"silu": 0.5, "gelu": 0.8, "sigmoid": 0.1}


def projections(x, w, dt):
    """g, u and how far sums in E's type may be off them: dim + 1 roundings of
    partial sums of at most |x| @ |w|."""
    h = w.shape[1] // 2
    x, w = x.reshape(-1, x.shape[-1]).astype(np.float64), w.astype(np.float64)
    both, size = x @ w, np.abs(x) @ np.abs(w)
    off = (x.shape[1] + 1) * E[dt] * size
    return both[:, :h], both[:, h:], off[:, :h], off[:, h:]


def ffn_want(x, w, name, dt):
    g, u, dg, du = projections(x, w, dt)
    a, _ = activation(name, g)
    # f is off by up to 16 E of itself (float16's), a's own product and the last one by one each
    bound = SLOPE[name] * dg * (np.abs(u) + du) + np.abs(a) * du + 20 * E[dt] * np.abs(a * u)
    if name == "gelu":  # the complementary error function's argument is rounded: g^2 E of phi
        bound = bound + E[dt] * g * g * np.abs(a * u) + 20 * E[dt] * np.abs(u) * (g * g > 170) * 1e-35
    return a * u, bound


def ffn_grad_want(grad, x, w, name, dt):
    g, u, og, ou = projections(x, w, dt)
    a, slope = activation(name, g)
    d = grad.reshape(g.shape).astype(np.float64)
    e = E[dt]
    up, gate = d * a, d * u * slope
    # every value of D: from g and u being off, a few roundings, and its own type's
    off_up = np.abs(d) * (SLOPE[name] * og + (24 + g * g) * e * np.abs(a)) + U[dt] * np.abs(up) + TINY[dt]
    off_gate = np.abs(d) * (SLOPE[name] * ou + (np.abs(u) + ou) * (BEND[name] * og + (32 + g * g) * e * SLOPE[name])) \
        + U[dt] * np.abs(gate) + TINY[dt]
    both, off = np.concatenate([gate, up], 1), np.concatenate([off_gate, off_up], 1) * 1.001
    x, w = x.reshape(-1, x.shape[-1]).astype(np.float64), w.astype(np.float64)
    size = np.abs(both) + off
    gx, ox = both @ w.T, off @ np.abs(w).T + (both.shape[1] + 1) * e * (size @ np.abs(w).T)
    gw, ow = x.T @ both, np.abs(x).T @ off + (len(x) + 1) * e * (np.abs(x).T @ size)
    return gx, ox, gw, ow


SIZES = [(1, 1, 1), (1, 7, 3), (3, 8, 8), (2, 64, 40), (17, 33, 29), (64, 128, 64), (5, 1000, 130),
         (129, 65, 257), (300, 72, 100), (8, 520, 1032), (31, 2049, 65), (260, 300, 515)]


@pytest.mark.parametrize("name", ["silu", "gelu", "sigmoid"])
@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("rows,dim,hidden", SIZES)
def test_feed_forward(dt, name, rows, dim, hidden):
    g = np.random.default_rng(rows * dim + hidden)
    x = g.standard_normal((rows, dim)).astype(dt)
    w = (g.standard_normal((dim, 2 * hidden)) * (1.5 / dim ** 0.5)).astype(dt)
    want, bound = ffn_want(x, w, name, dt)
    dx, dw = cp.array(x), cp.array(w)
    got = nn.gated_feed_forward(dx, dw, name)
    near(got, want, bound, dt)
    assert np.array_equal(nn.gated_feed_forward(dx, dw, name).get(), got.get())
    grad = g.standard_normal((rows, hidden)).astype(dt)
    gx, ox, gw, ow = ffn_grad_want(grad, x, w, name, dt)
    got_x, got_w = nn.gated_feed_forward_grad(cp.array(grad), dx, dw, name)
    near(got_x, gx, ox, dt)
    near(got_w, gw, ow, dt)


@pytest.mark.parametrize("rows,dim,hidden", [(2000, 64, 64), (512, 1024, 1024), (40, 4096, 512), (1100, 520, 1300)])
def test_feed_forward_many(rows, dim, hidden):
    """Several tiles, k ranges and their ends, float16."""
    dt = np.float16
    g = np.random.default_rng(rows)
    x = g.standard_normal((rows, dim)).astype(dt)
    w = (g.standard_normal((dim, 2 * hidden)) * (1.5 / dim ** 0.5)).astype(dt)
    grad = g.standard_normal((rows, hidden)).astype(dt)
    want, bound = ffn_want(x, w, "silu", dt)
    near(nn.gated_feed_forward(cp.array(x), cp.array(w)), want, bound, dt)
    gx, ox, gw, ow = ffn_grad_want(grad, x, w, "silu", dt)
    got_x, got_w = nn.gated_feed_forward_grad(cp.array(grad), cp.array(x), cp.array(w))
    near(got_x, gx, ox, dt)
    near(got_w, gw, ow, dt)


@pytest.mark.parametrize("dt", FLOATS, **by_name)
def test_feed_forward_views(dt):
    """Parts of larger arrays, reversed, transposed, broadcast and of other shapes."""
    g = np.random.default_rng(5)
    big_x, big_w = (g.standard_normal(s).astype(dt) for s in ((6, 40, 90), (90, 300)))
    dx, dw = cp.array(big_x), cp.array(big_w)
    for xv in (lambda a: a[:, :, 3:53], lambda a: a[1, ::2, :50], lambda a: a[2, 5, 40:],
               lambda a: a[::-1, 3, 8:58], lambda a: a[:2, 4:5, 20:70]):
        for wv in (lambda a: a[:50, 10:94], lambda a: a[40:, 1:101], lambda a: a[::-1][:50, ::2]):
            x, w = xv(big_x), wv(big_w)
            want, bound = ffn_want(x, w, "gelu", dt)
            got = nn.gated_feed_forward(xv(dx), wv(dw), "gelu")
            near(got, want.reshape(x.shape[:-1] + (w.shape[1] // 2,)),
                 bound.reshape(x.shape[:-1] + (w.shape[1] // 2,)), dt)
            grad = g.standard_normal(got.shape[::-1]).astype(dt)
            gx, ox, gw, ow = ffn_grad_want(grad.T, x, w, "gelu", dt)
            got_x, got_w = nn.gated_feed_forward_grad(cp.array(grad).T, xv(dx), wv(dw), "gelu")
            near(got_x, gx.reshape(x.shape), ox.reshape(x.shape), dt)
            near(got_w, gw, ow, dt)
    one = cp.broadcast_to(dx[0, 0, :50], (7, 50))
    want, bound = ffn_want(np.broadcast_to(big_x[0, 0, :50], (7, 50)), big_w[:50, :60], "silu", dt)
    near(nn.gated_feed_forward(one, dw[:50, :60]), want, bound, dt)


def test_feed_forward_types_and_empty():
    g = np.random.default_rng(0)
    x, w = g.standard_normal((4, 6)).astype(np.float16), g.standard_normal((6, 10)).astype(np.float32)
    want, bound = ffn_want(x, w, "silu", np.float32)
    near(nn.gated_feed_forward(cp.array(x), cp.array(w)), want, bound, np.float32)
    for dt in FLOATS:
        z = lambda *s: cp.zeros(s, dtype=dt)  # noqa: E731
        assert nn.gated_feed_forward(z(0, 6), z(6, 10)).shape == (0, 5)
        assert nn.gated_feed_forward(z(3, 0), z(0, 10)).get().tolist() == [[0.0] * 5] * 3
        assert nn.gated_feed_forward(z(3, 6), z(6, 0)).shape == (3, 0)
        a, b = nn.gated_feed_forward_grad(z(0, 5), z(0, 6), z(6, 10))
        assert a.shape == (0, 6) and b.get().tolist() == [[0.0] * 10] * 6
        a, b = nn.gated_feed_forward_grad(z(3, 0), z(3, 6), z(6, 0))
        assert a.get().tolist() == [[0.0] * 6] * 3 and b.shape == (6, 0)
        a, b = nn.gated_feed_forward_grad(z(3, 5), z(3, 0), z(0, 10))
        assert a.shape == (3, 0) and b.shape == (0, 10)


@pytest.mark.parametrize("dt", FLOATS, **by_name)
def test_feed_forward_spoiled_rows(dt):
    """A NaN or an infinity stays in its row; rows before and after are as without."""
    g = np.random.default_rng(2)
    x, w = g.standard_normal((70, 37)).astype(dt), g.standard_normal((37, 46)).astype(dt)
    clean = nn.gated_feed_forward(cp.array(x), cp.array(w)).get()
    x[5, 3], x[69, 36] = np.nan, np.inf
    got = nn.gated_feed_forward(cp.array(x), cp.array(w)).get()
    rest = np.delete(np.arange(70), [5, 69])
    assert np.array_equal(got[rest], clean[rest]) and np.isnan(got[5]).all()
    assert not np.isfinite(got[69]).all()


@pytest.mark.parametrize("name", ["silu", "gelu", "sigmoid"])
def test_feed_forward_differences(name):
    """The gradient against differences of the operator itself, in 64 bits."""
    g = np.random.default_rng(4)
    x, w, d = g.standard_normal((5, 7)), g.standard_normal((7, 12)), g.standard_normal((5, 6))
    gx, gw = nn.gated_feed_forward_grad(cp.array(d), cp.array(x), cp.array(w), name)
    value = lambda x, w: float((nn.gated_feed_forward(cp.array(x), cp.array(w), name).get() * d).sum())  # noqa: E731
    step = 1e-5
    for i in range(6):
        vx, vw = g.standard_normal(x.shape), g.standard_normal(w.shape)
        slope = (value(x + step * vx, w + step * vw) - value(x - step * vx, w - step * vw)) / (2 * step)
        want = float((gx.get() * vx).sum() + (gw.get() * vw).sum())
        # third derivatives of order 1e3 times step^2 / 6, and 2^-53 of values of some 1e2 over step
        assert abs(slope - want) <= 1e3 * step ** 2 + 1e2 * 2.0 ** -53 / step * 10


# --------------------------------------------------------------- dropout
def words(first, count, seed):
    """Words of the Philox4x32-10 stream, from their definition."""
    low, half = np.uint64(0xFFFFFFFF), np.uint64(32)
    block = np.array([(first // 4 + i) % 2 ** 64 for i in range((first % 4 + count + 3) // 4)], np.uint64)
    c = [block & low, block >> half, 0 * block, 0 * block]
    k = [seed % 2 ** 32, seed >> 32]
    for _ in range(10):
        p, q = np.uint64(0xD2511F53) * c[0], np.uint64(0xCD9E8D57) * c[2]
        c = [(q >> half) ^ c[1] ^ np.uint64(k[0]), q & low, (p >> half) ^ c[3] ^ np.uint64(k[1]), p & low]
        k = [(k[0] + 0x9E3779B9) % 2 ** 32, (k[1] + 0xBB67AE85) % 2 ** 32]
    return np.stack(c, 1).reshape(-1)[first % 4:][:count]


def dropout_want(x, rate, seed, offset, residual=None):
    """The same operations in the same types: equal to the last bit."""
    wide = np.float64 if x.dtype == np.float64 else np.float32
    keep = words(offset, x.size, seed).reshape(x.shape) >= math.floor(rate * 2 ** 32 + 0.5)
    with np.errstate(all="ignore"):
        y = np.where(keep, x.astype(wide) * wide(1.0 / (1.0 - rate)), wide(0))
        return (y if residual is None else y + residual.astype(wide)).astype(x.dtype)


def test_published_words():
    """The known answers that the generator was published with."""
    assert [hex(w) for w in words(0, 4, 0)] == ["0x6627e8d5", "0xe169c58d", "0xbc57ac4c", "0x9b00dbd8"]


@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("n", [0, 1, 2, 3, 4, 5, 7, 8, 9, 31, 2047, 2048, 2049, 10_007])
def test_dropout(dt, n):
    g = np.random.default_rng(n)
    x, r = g.standard_normal(n).astype(dt), g.standard_normal(n).astype(dt)
    for rate, seed, offset in ((0.0, 0, 0), (0.1, 7, 1), (0.5, 2 ** 64 - 1, 2), (0.9, 2 ** 33 + 5, 3),
                               (0.25, 12345, 2 ** 34 - 3), (0.3, 1, 2 ** 63 - 1), (1.0 - 2.0 ** -40, 3, 4)):
        want = dropout_want(x, rate, seed, offset)
        got = nn.dropout(cp.array(x), rate, seed, offset)
        assert got.dtype == dt and np.array_equal(got.get(), want)
        got = nn.dropout(cp.array(x), rate, seed, offset, cp.array(r))
        assert np.array_equal(got.get(), dropout_want(x, rate, seed, offset, r))


def test_dropout_places_and_gradient():
    g = np.random.default_rng(1)
    x = g.standard_normal((64, 33)).astype(np.float32)
    d = cp.array(x)
    whole = nn.dropout(d, 0.4, 99, 17).get()
    assert np.array_equal(nn.dropout(d[10:20], 0.4, 99, 17 + 330).get(), whole[10:20])
    assert np.array_equal(nn.dropout(d.T, 0.4, 99).get(), dropout_want(x.T, 0.4, 99, 0))
    assert np.array_equal(nn.dropout(d[:, ::2], 0.4, 99).get(), dropout_want(x[:, ::2], 0.4, 99, 0))
    at = cp.array(np.array(17, np.int64))
    assert np.array_equal(nn.dropout(d, 0.4, 99, at).get(), whole)
    assert np.array_equal(nn.dropout(d, 0.4, 99, cp.array(np.array(17, np.int32))).get(), whole)
    # linear in x, so the gradient is the same call
    grad = g.standard_normal(x.shape).astype(np.float32)
    keep = nn.dropout(cp.ones(x.shape, dtype=np.float32), 0.4, 99, 17).get()
    assert np.array_equal(nn.dropout(cp.array(grad), 0.4, 99, 17).get(), grad * keep)
    # a dropped infinity or NaN is 0
    x[:] = np.inf
    x[::2] = np.nan
    got = nn.dropout(cp.array(x), 0.4, 99, 17).get()
    assert np.array_equal(got == 0, keep == 0) and not np.isfinite(got[keep != 0]).any()


def test_dropout_rate():
    """The share that is dropped, within five standard deviations."""
    n = 1 << 20
    for rate in (0.05, 0.5, 0.8):
        gone = float((nn.dropout(cp.ones(n, dtype=np.float16), rate, 5).get() == 0).mean())
        assert abs(gone - rate) < 5 * (rate * (1 - rate) / n) ** 0.5


def test_refusals():
    z = lambda *s, dt=np.float32: cp.zeros(s, dtype=dt)  # noqa: E731
    for x, w, act, error in ((z(3, 4), z(5, 6), "silu", ValueError), (z(3, 4), z(4, 5), "silu", ValueError),
                             (z(3, 4), z(4, 6), "relu", ValueError), (z(3, 4), z(4, 6), None, ValueError),
                             (z(3, 4, dt=np.int32), z(4, 6), "silu", TypeError), (z(3, 4), z(4), "silu", ValueError),
                             (z(3, 4), z(2, 4, 6), "silu", ValueError), (cp.array(np.float32(1)), z(1, 2), "silu", ValueError)):
        with pytest.raises(error):
            nn.gated_feed_forward(x, w, act)
        with pytest.raises(error):
            nn.gated_feed_forward_grad(z(3, 3), x, w, act)
    with pytest.raises(ValueError):
        nn.gated_feed_forward_grad(z(3, 4), z(3, 4), z(4, 6))
    x = z(3, 4)
    for args, error in (((x, -0.1, 0), ValueError), ((x, 1.0, 0), ValueError), ((x, float("nan"), 0), ValueError),
                        ((x, "0.1", 0), TypeError), ((x, 0.1, -1), ValueError), ((x, 0.1, 2 ** 64), ValueError),
                        ((x, 0.1, 1.5), TypeError), ((x, 0.1, True), TypeError), ((x, 0.1, 0, -1), ValueError),
                        ((x, 0.1, 0, 2 ** 63), ValueError), ((x, 0.1, 0, 1.0), TypeError),
                        ((x, 0.1, 0, z(1, dt=np.int64)), ValueError), ((x, 0.1, 0, cp.array(np.array(1.0))), TypeError),
                        ((x, 0.1, 0, 0, z(3, 5)), ValueError), ((x, 0.1, 0, 0, z(3, 4, dt=np.float16)), ValueError),
                        ((z(3, dt=np.int32), 0.1, 0), TypeError)):
        with pytest.raises(error):
            nn.dropout(*args)
