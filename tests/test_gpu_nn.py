"""``cp.nn`` against plain NumPy in 64 bits.

Tolerances, all derived from the formulas: U is half a unit of the result's
type (its one rounding), E of the type that sums are held in, TINY half of the
smallest number that the result's type holds.
"""
import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import nn

pytestmark = pytest.mark.gpu

FLOATS = [np.float16, np.float32, np.float64]
U = {np.float16: 2.0 ** -11, np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
E = {np.float16: 2.0 ** -24, np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
# float32's own: the hardware's exponential gives 0 below the normal range
TINY = {np.float16: 2.0 ** -25, np.float32: 2.0 ** -126, np.float64: 2.0 ** -1022}
by_name = {"ids": lambda v: getattr(v, "__name__", None) or str(v)}


def near(got, want, bound, dt):
    """Each element within `bound` and the rounding of the result's type."""
    got, want = got.get().astype(np.float64), np.asarray(want, np.float64)
    assert got.shape == want.shape
    off = np.abs(got - want) - (bound + (U[dt] * 1.001) * (np.abs(want) + bound) + TINY[dt])
    assert not off.size or np.nanmax(off) <= 0, f"off by {np.nanmax(off):.3g} more than the bound"
    assert np.array_equal(np.isnan(got), np.isnan(want))


# ------------------------------------------------------------- embedding
@pytest.mark.parametrize("it", [np.int32, np.int64, np.int16, np.uint32], **by_name)
@pytest.mark.parametrize("dt", FLOATS, **by_name)
def test_embedding(dt, it):
    g = np.random.default_rng(0)
    for rows, dim, shape in ((1, 1, (1,)), (5, 3, (2, 7)), (100, 8, (33,)), (77, 129, (4, 1, 9)),
                             (300, 1000, (65,)), (19, 4099, (5,)), (9, 17, (1000,)), (40, 7, ())):
        table = g.standard_normal((rows, dim)).astype(dt)
        tok = g.integers(0, rows, shape).astype(it)
        if it != np.uint32 and tok.ndim:
            tok[..., ::3] = -1
        if tok.ndim:
            tok[..., 1:2] = rows  # past the end
        wide = np.float64 if dt == np.float64 else np.float32
        there = (tok >= 0) & (tok < rows)
        want = np.where(there[..., None], table[np.where(there, tok, 0)].astype(wide) * wide(1.5),
                        wide(0)).astype(dt)
        got = nn.embedding(cp.array(table), cp.array(tok), scale=1.5)
        assert got.dtype == dt and np.array_equal(got.get(), want)


def test_embedding_views():
    g = np.random.default_rng(1)
    h = g.standard_normal((50, 41)).astype(np.float32)
    d, tok = cp.array(h), g.integers(0, 20, (6, 8))
    for view in (lambda a: a[3:, 5:], lambda a: a[::2, :33], lambda a: a[::-1], lambda a: a.T,
                 lambda a: a[:, ::2], lambda a: a[:, 40:]):
        for t in (tok, tok.T, tok[::2, 1:]):
            got = nn.embedding(view(d), cp.array(np.ascontiguousarray(tok))
                               if t is tok else cp.array(t))
            assert np.array_equal(got.get(), view(h)[t])
    dt = cp.array(tok)
    assert np.array_equal(nn.embedding(d, dt[::2, 1:].T).get(), h[tok[::2, 1:].T])
    one = cp.broadcast_to(d[:1], (30, 41))
    assert np.array_equal(nn.embedding(one, dt).get(), np.broadcast_to(h[:1], (30, 41))[tok])


def test_embedding_empty():
    t = cp.array(np.ones((4, 5), np.float32))
    assert nn.embedding(t, cp.array(np.zeros((0,), np.int64))).shape == (0, 5)
    assert nn.embedding(t[:, :0], cp.array(np.zeros(3, np.int64))).shape == (3, 0)
    assert np.array_equal(nn.embedding(t[:0], cp.array(np.zeros(3, np.int64))).get(),
                          np.zeros((3, 5)))
    assert nn.embedding_grad(t[:0], cp.array(np.zeros(0, np.int64)), 3).get().tolist() == [[0] * 5] * 3
    assert nn.embedding_grad(t, cp.array(np.zeros(4, np.int64)), 0).shape == (0, 5)
    assert nn.embedding_grad(t[:, :0], cp.array(np.zeros(4, np.int64)), 2).shape == (2, 0)


def _grad_want(grad, tok, rows, scale):
    g = grad.reshape(tok.size, -1).astype(np.float64)
    t = tok.reshape(-1).astype(np.int64)
    keep = (t >= 0) & (t < rows)
    want, size = np.zeros((rows, g.shape[1])), np.zeros((rows, g.shape[1]))
    np.add.at(want, t[keep], g[keep])
    np.add.at(size, t[keep], np.abs(g[keep]))
    n = np.bincount(t[keep], minlength=rows)[:, None]
    return want * scale, size * scale, n


@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("rows,dim,n,spread", [
    (1, 1, 1, 1), (1, 5, 300, 1), (7, 3, 50, 7), (100, 33, 1000, 100), (5000, 17, 300, 5000),
    (300, 1001, 700, 300), (40, 64, 5000, 3), (3000, 2, 70_000, 3000), (300_000, 4, 1000, 300_000),
    (50, 4097, 130, 50), (1000, 256, 9000, 2), (64, 8, 65, 64)])
def test_embedding_grad(dt, rows, dim, n, spread):
    """`spread` tokens in use: few of them make rows of thousands of addends."""
    g = np.random.default_rng(n)
    tok = (g.integers(0, spread, n) * (rows // spread)).astype(np.int64)
    tok[::11] = -1
    tok[5:6] = rows
    grad = g.standard_normal((n, dim)).astype(dt)
    want, size, count = _grad_want(grad, tok, rows, 0.75)
    got = nn.embedding_grad(cp.array(grad), cp.array(tok), rows, scale=0.75)
    assert got.dtype == dt
    # every addition rounds a partial sum of at most `size`
    near(got, want, (count + 2) * E[dt] * size, dt)
    again = nn.embedding_grad(cp.array(grad), cp.array(tok.astype(np.int32)), rows, scale=0.75)
    assert np.array_equal(again.get(), got.get())


def test_embedding_grad_skewed():
    """Words' frequencies as in a text: some rows of thousands, many of none."""
    g = np.random.default_rng(3)
    rows, n, dim = 20_011, 60_000, 72
    tok = np.minimum(np.exp(g.random(n) * np.log(rows)).astype(np.int64) - 1, rows - 1)
    grad = g.standard_normal((4, n // 4, dim)).astype(np.float16)
    want, size, count = _grad_want(grad, tok, rows, 1.0)
    got = nn.embedding_grad(cp.array(grad), cp.array(tok.reshape(4, -1)), rows)
    near(got, want, (count + 2) * E[np.float16] * size, np.float16)


@pytest.mark.parametrize("rows,spread", [(1, 1), (3, 3), (257, 257), (70_001, 70_001), (70_001, 2),
                                         (1_100_000, 1_100_000), (70_001, 0)])
@pytest.mark.parametrize("n", [131_072, 200_003])
def test_embedding_grad_many_tokens(n, rows, spread):
    """On both sides of 2^17 tokens; spread 0: not one of them has a row."""
    g = np.random.default_rng(n + rows + spread)
    tok = g.integers(0, spread, n) * (rows // spread) if spread else np.full(n, -1)
    tok[::13] = -1
    grad = g.standard_normal((n, 3)).astype(np.float32)
    want, size, count = _grad_want(grad, tok, rows, 0.5)
    near(nn.embedding_grad(cp.array(grad), cp.array(tok), rows, scale=0.5), want,
         (count + 2) * E[np.float32] * size, np.float32)


@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("n,rows,dim,spread", [
    (16_384, 5, 40, 5), (16_385, 5, 40, 5), (17_000, 3, 1001, 3), (17_000, 700, 4097, 20),
    (16_300, 9, 1001, 2), (20_000, 300, 1, 7), (12_000, 300, 1, 7), (8192, 270_000, 3, 3),
    (8193, 270_000, 3, 3), (4096, 600_000, 2, 4096), (4097, 600_000, 2, 4096), (129, 256, 33, 1),
    (129, 257, 8200, 1), (40_000, 600, 65, 600), (40_000, 600, 64, 3), (150_000, 600, 65, 9)])
def test_embedding_grad_forms(dt, n, rows, dim, spread):
    """Tokens that one workgroup's registers hold, and one more; rows of many
    positions, whole and in windows."""
    g = np.random.default_rng(n + dim)
    tok = g.integers(0, spread, n) * (rows // spread) - 1  # -1 among them
    grad = g.standard_normal((n, dim)).astype(dt)
    want, size, count = _grad_want(grad, tok, rows, 2.0)
    got = nn.embedding_grad(cp.array(grad), cp.array(tok), rows, scale=2.0)
    near(got, want, (count + 2) * E[dt] * size, dt)
    assert np.array_equal(nn.embedding_grad(cp.array(grad), cp.array(tok), rows, scale=2.0).get(),
                          got.get())


def test_embedding_grad_views():
    g = np.random.default_rng(4)
    h = g.standard_normal((60, 50)).astype(np.float32)
    tok = g.integers(0, 9, 30)
    for view in (lambda a: a[::2, 3:48], lambda a: a[29::-1], lambda a: a.T[:30], lambda a: a[:30, ::3]):
        want, size, count = _grad_want(np.ascontiguousarray(view(h)), tok, 9, 1.0)
        near(nn.embedding_grad(view(cp.array(h)), cp.array(tok), 9), want,
             (count + 2) * E[np.float32] * size, np.float32)
    ones = cp.broadcast_to(cp.array(np.ones(1, np.float32)), (30, 50))
    want, _, _ = _grad_want(np.ones((30, 50), np.float32), tok, 9, 1.0)
    assert np.array_equal(nn.embedding_grad(ones, cp.array(tok), 9).get(), want)


def test_embedding_past_32_bits():
    rows, dim = (1 << 21) + 3, 1025  # 2^31 elements and more
    table = cp.zeros((rows, dim), dtype=np.float16)
    line = np.arange(dim, dtype=np.float16)
    table[rows - 1] = cp.array(line)
    got = nn.embedding(table, cp.array(np.array([rows - 1, 5, rows - 1]))).get()
    assert np.array_equal(got, np.stack([line, np.zeros_like(line), line]))
    tok = cp.full((rows,), -1, dtype=np.int64)
    tok[rows - 1] = 1
    tok[rows - 2] = 1
    back = nn.embedding_grad(table, tok, 3).get()
    assert np.array_equal(back, np.stack([0 * line, line, 0 * line]))
    # and where the gradient's own rows are that many
    del back
    back = nn.embedding_grad(cp.array(np.stack([line, line])), cp.array(np.array([rows - 1, 0])), rows)
    assert np.array_equal(back[rows - 3:].get(), np.stack([0 * line, 0 * line, line]))
    assert np.array_equal(back[:2].get(), np.stack([line, 0 * line]))


# ------------------------------------------------------------ recurrence
def _factors(gate, x, logits):
    gate, x = gate.astype(np.float64), x.astype(np.float64)
    if not logits:
        return gate, np.ones_like(gate), x
    with np.errstate(over="ignore"):
        f, u = 1 / (1 + np.exp(-gate)), 1 / (1 + np.exp(gate))
    return f, u, u * x


def _recur(gate, x, initial, logits, e):
    """h, and a bound on its error: each step rounds the factor (exponential,
    reciprocal and product, at most 10 E), its product with neighbouring
    factors, the addend and the sum, and hands on the error of the step before."""
    f, _, b = _factors(gate, x, logits)
    h, bound = np.empty_like(b), np.empty_like(b)
    s, size, off = initial.astype(np.float64), np.abs(initial.astype(np.float64)), 0.0
    for t in range(b.shape[-2]):
        s = f[..., t, :] * s + b[..., t, :]
        size = np.abs(f[..., t, :]) * size + np.abs(b[..., t, :])
        off = np.abs(f[..., t, :]) * off + 16 * e * size
        h[..., t, :], bound[..., t, :] = s, off
    return h, s, bound, off


def _recur_grad(grad, gate, x, h, initial, grad_final, logits, e):
    f, u, _ = _factors(gate, x, logits)
    grad, x = grad.astype(np.float64), x.astype(np.float64)
    before = np.concatenate([initial.astype(np.float64)[..., None, :],
                             h.astype(np.float64)[..., :-1, :]], -2)
    d, off = np.empty_like(grad), np.empty_like(grad)
    c = grad_final.astype(np.float64)
    size, lost = np.abs(c), np.zeros_like(c)
    for t in range(grad.shape[-2] - 1, -1, -1):
        d[..., t, :] = grad[..., t, :] + c
        size = size + np.abs(grad[..., t, :])
        lost = lost + 2 * e * size
        off[..., t, :] = lost
        c = f[..., t, :] * d[..., t, :]
        size, lost = np.abs(f[..., t, :]) * size, np.abs(f[..., t, :]) * (lost + 14 * e * size)
    to_gate = (before - x) * f * u if logits else before
    to_x = u if logits else np.ones_like(u)
    more = 32 * e
    return ((d * to_gate, np.abs(to_gate) * (off + more * np.abs(d))),
            (d * to_x, np.abs(to_x) * (off + more * np.abs(d))), (c, lost + 2 * e * size))


SHAPES = [(1, 1, 1), (3, 1, 5), (1, 2, 64), (2, 7, 33), (5, 31, 3), (1, 64, 130), (2, 129, 17),
          (1, 1000, 65), (3, 257, 128), (1, 4099, 8), (130, 3, 9), (2, 515, 257)]


def _sequence(g, shape, dt, logits):
    gate = g.standard_normal(shape) * 2 + 2
    if not logits:
        gate = np.where(g.random(shape) < 0.05, 0.0, 1 / (1 + np.exp(-gate))) * g.choice([-1, 1], shape)
    state = np.float64 if dt == np.float64 else np.float32
    return (gate.astype(dt), g.standard_normal(shape).astype(dt),
            g.standard_normal(shape[:-2] + shape[-1:]).astype(state))


@pytest.mark.parametrize("logits", [True, False])
@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("shape", SHAPES, **by_name)
def test_recurrence(shape, dt, logits):
    g = np.random.default_rng(sum(shape))
    gate, x, initial = _sequence(g, shape, dt, logits)
    h, final = nn.gated_recurrence(cp.array(gate), cp.array(x), cp.array(initial), logits=logits)
    want, last, bound, off = _recur(gate, x, initial, logits, E[dt])
    assert h.dtype == dt and final.dtype == initial.dtype
    near(h, want, bound, dt)
    near(final, last, off, initial.dtype.type)
    none, final0 = nn.gated_recurrence(cp.array(gate), cp.array(x), logits=logits)
    want, last, bound, off = _recur(gate, x, 0 * initial, logits, E[dt])
    near(none, want, bound, dt)
    near(final0, last, off, initial.dtype.type)


@pytest.mark.parametrize("logits", [True, False])
@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("shape", SHAPES, **by_name)
def test_recurrence_grad(shape, dt, logits):
    g = np.random.default_rng(sum(shape) + 1)
    gate, x, initial = _sequence(g, shape, dt, logits)
    h = _recur(gate, x, initial, logits, 0.0)[0].astype(dt)
    grad = g.standard_normal(shape).astype(dt)
    end = g.standard_normal(initial.shape).astype(initial.dtype)
    for grad_final in (end, None):
        got = nn.gated_recurrence_grad(*map(cp.array, (grad, gate, x, h, initial)),
                                       None if grad_final is None else cp.array(end), logits=logits)
        want = _recur_grad(grad, gate, x, h, initial, end if grad_final is not None else 0 * end,
                           logits, E[dt])
        for a, (w, bound), t in zip(got, want, (dt, dt, initial.dtype.type)):
            assert a.dtype == t
            near(a, w, bound, t)
    got = nn.gated_recurrence_grad(*map(cp.array, (grad, gate, x, h)), logits=logits)
    want = _recur_grad(grad, gate, x, h, 0 * initial, 0 * end, logits, E[dt])
    for a, (w, bound), t in zip(got, want, (dt, dt, initial.dtype.type)):
        near(a, w, bound, t)


@pytest.mark.parametrize("dt,shape", [
    (np.float16, (300, 70, 1001)), (np.float32, (150, 70, 1001)), (np.float64, (66, 67, 1001)),
    (np.float16, (300, 16, 1001)), (np.float16, (300, 15, 3)), (np.float16, (20, 64, 3)),
    (np.float16, (20, 200, 7)), (np.float32, (20, 200, 1)), (np.float32, (20, 400, 1001)),
    (np.float16, (40, 400, 1001)), (np.float64, (20, 300, 1001)), (np.float16, (70, 700, 30)),
    (np.float16, (30, 700, 65)), (np.float32, (70, 700, 15)), (np.float32, (70, 300, 64))],
    **by_name)
def test_recurrence_many_sequences(dt, shape):
    """Sequences enough for a thread to go through its channels' steps, odd rows."""
    g = np.random.default_rng(shape[0])
    gate, x, initial = _sequence(g, shape, dt, True)
    h, final = nn.gated_recurrence(cp.array(gate), cp.array(x), cp.array(initial))
    want, last, bound, off = _recur(gate, x, initial, True, E[dt])
    near(h, want, bound, dt)
    near(final, last, off, initial.dtype.type)
    grad = g.standard_normal(shape).astype(dt)
    got = nn.gated_recurrence_grad(*map(cp.array, (grad, gate, x)), h, cp.array(initial))
    want = _recur_grad(grad, gate, x, h.get(), initial, 0 * initial, True, E[dt])
    for a, (w, lim), t in zip(got, want, (dt, dt, initial.dtype.type)):
        near(a, w, lim, t)


@pytest.mark.parametrize("logits", [True, False])
@pytest.mark.parametrize("dt", FLOATS, **by_name)
def test_recurrence_past_the_caches(dt, logits):
    """Arrays of more than 256 MiB, here one sequence that is every sequence."""
    g = np.random.default_rng(21)
    batch, steps, dim = (64, 700, 1024) if dt == np.float16 else (64, 350, 1024)
    gate, x, initial = _sequence(g, (steps, dim), dt, logits)
    grad = g.standard_normal((steps, dim)).astype(dt)
    every = lambda a: cp.broadcast_to(cp.array(a), (batch,) + a.shape)  # noqa: E731
    h, final = nn.gated_recurrence(every(gate), every(x), every(initial), logits=logits)
    got = nn.gated_recurrence_grad(every(grad), every(gate), every(x), h, every(initial),
                                   logits=logits)
    want, last, bound, off = _recur(gate, x, initial, logits, E[dt])
    wants = [(want, bound), (last, off)]
    wants += _recur_grad(grad, gate, x, h[0].get(), initial, 0 * initial, logits, E[dt])
    kinds = (dt, initial.dtype.type, dt, dt, initial.dtype.type)
    for a, (w, lim), t in zip((h, final) + got, wants, kinds):
        near(a[0], w, lim, t)
        assert bool((a == a[:1]).all())


@pytest.mark.parametrize("logits", [True, False])
def test_recurrence_differences(logits):
    """The gradients against central differences of a weighted sum of outputs."""
    g = np.random.default_rng(8)
    shape = (2, 9, 3)
    gate, x, initial = _sequence(g, shape, np.float64, logits)
    wh, wf = g.standard_normal(shape), g.standard_normal((2, 3))

    def value(a, b, c):
        h, final = nn.gated_recurrence(cp.array(a), cp.array(b), cp.array(c), logits=logits)
        return float((h.get() * wh).sum() + (final.get() * wf).sum())

    h, _ = nn.gated_recurrence(cp.array(gate), cp.array(x), cp.array(initial), logits=logits)
    got = nn.gated_recurrence_grad(cp.array(wh), cp.array(gate), cp.array(x), h, cp.array(initial),
                                   cp.array(wf), logits=logits)
    step = 1e-5  # rounding 1e-16 / 1e-5, third derivatives times 1e-10
    for k, d in enumerate(got):
        d = d.get().reshape(-1)
        for i in range(d.size):
            ends = []
            for s in (step, -step):
                args = [gate.copy(), x.copy(), initial.copy()]
                args[k].reshape(-1)[i] += s
                ends.append(value(*args))
            assert abs((ends[0] - ends[1]) / (2 * step) - d[i]) < 1e-7


@pytest.mark.parametrize("dt", [np.float16, np.float32], **by_name)
def test_recurrence_views(dt):
    """Gate and x as the halves of one product, other strides, 2 and 4 axes."""
    g = np.random.default_rng(9)
    both = g.standard_normal((4, 70, 2 * 37)).astype(dt)
    d = cp.array(both)
    views = [(lambda a: a[:, :, :37], lambda a: a[:, :, 37:]),
             (lambda a: a[:, ::-1, :37], lambda a: a[:, ::-1, 1:38]),
             (lambda a: a[::2, :, 3:9], lambda a: a[1::2, :, 3:9]),
             (lambda a: a[:, :, ::2], lambda a: a[:, :, 1::2]),
             (lambda a: a.transpose(0, 2, 1), lambda a: a.transpose(0, 2, 1)),
             (lambda a: a[0, :, :37], lambda a: a[1, :, 37:]),
             (lambda a: a.reshape(2, 2, 70, 74)[:, :, 5:], lambda a: a.reshape(2, 2, 70, 74)[:, :, 5:]),
             (lambda a: a.reshape(2, 2, 70, 74).swapaxes(0, 1)[:, :, :, :9],
              lambda a: a.reshape(2, 2, 70, 74)[:, :, :, :9])]
    for va, vb in views:
        a, b = np.ascontiguousarray(va(both)), np.ascontiguousarray(vb(both))
        zero = np.zeros(a.shape[:-2] + a.shape[-1:], np.float32)
        want, last, bound, off = _recur(a, b, zero, True, E[dt])
        h, final = nn.gated_recurrence(va(d), vb(d))
        near(h, want, bound, dt)
        near(final, last, off, np.float32)
        got = nn.gated_recurrence_grad(vb(d), va(d), vb(d), va(d))
        for o, (w, lim), t in zip(got, _recur_grad(b, a, b, a, zero, zero, True, E[dt]),
                                  (dt, dt, np.float32)):
            near(o, w, lim, t)
    line = cp.broadcast_to(cp.array(both[0, 0]), (4, 70, 74))  # one gate for every step
    want, _, bound, _ = _recur(np.broadcast_to(both[0, 0], both.shape), both,
                               np.zeros((4, 74), np.float32), True, E[dt])
    near(nn.gated_recurrence(line, d)[0], want, bound, dt)


def test_recurrence_resets_and_extremes():
    g = np.random.default_rng(10)
    gate, x, initial = _sequence(g, (2, 300, 40), np.float32, True)
    gate[:, 100], gate[:, 200] = -np.inf, np.inf  # starts anew, keeps all
    gate[:, 150], gate[:, 250] = -200.0, 200.0
    want, last, bound, off = _recur(gate, x, initial, True, E[np.float32])
    h, final = nn.gated_recurrence(cp.array(gate), cp.array(x), cp.array(initial))
    near(h, want, bound, np.float32)
    assert np.array_equal(h.get()[:, 100], x[:, 100])
    # the same state in 64 bits; each of the two is within its bound of it
    assert (np.abs(h.get()[:, 200] - h.get()[:, 199].astype(np.float64))
            <= 1.001 * (bound[:, 200] + bound[:, 199] + 2 * U[np.float32] * np.abs(want[:, 200]))).all()
    grad = g.standard_normal(gate.shape).astype(np.float32)
    got = nn.gated_recurrence_grad(cp.array(grad), cp.array(gate), cp.array(x), h, cp.array(initial))
    ref = _recur_grad(grad, gate, x, h.get(), initial, 0 * initial, True, E[np.float32])
    for a, (w, lim) in zip(got, ref):
        near(a, w, lim, np.float32)
    # a NaN stays in its channel, from its step on
    x[1, 120, 7] = np.nan
    h = nn.gated_recurrence(cp.array(gate), cp.array(x), cp.array(initial))[0].get()
    assert np.isnan(h[1, 120:, 7]).all()
    h[1, 120:, 7] = 0
    assert np.isfinite(h).all()


def test_recurrence_step_by_step():
    """Single tokens, each from the state of the one before, and the whole
    sequence give the same states."""
    g = np.random.default_rng(11)
    gate, x, initial = _sequence(g, (6, 50, 100), np.float16, True)
    h, final = nn.gated_recurrence(cp.array(gate), cp.array(x), cp.array(initial))
    s, rows = cp.array(initial), []
    for t in range(50):
        one, s = nn.gated_recurrence(cp.array(gate[:, t:t + 1]), cp.array(x[:, t:t + 1]), s)
        rows.append(one.get())
    _, last, _, off = _recur(gate, x, initial, True, E[np.float16])
    near(s, last, off, np.float32)
    near(final, last, off, np.float32)
    whole = np.concatenate(rows, 1).astype(np.float64)
    assert np.abs(whole - h.get()).max() <= 2.0 ** -10 * np.abs(whole).max()


def test_recurrence_empty():
    z = lambda *s: cp.array(np.zeros(s, np.float16))  # noqa: E731
    start = cp.array(np.arange(6, dtype=np.float32).reshape(2, 3))
    h, final = nn.gated_recurrence(z(2, 0, 3), z(2, 0, 3), start)
    assert h.shape == (2, 0, 3) and np.array_equal(final.get(), start.get())
    assert np.array_equal(nn.gated_recurrence(z(2, 0, 3), z(2, 0, 3))[1].get(), np.zeros((2, 3)))
    got = nn.gated_recurrence_grad(*[z(2, 0, 3)] * 4, None, start)
    assert np.array_equal(got[2].get(), start.get()) and got[0].shape == (2, 0, 3)
    for shape in ((0, 4, 3), (2, 4, 0)):
        h, final = nn.gated_recurrence(z(*shape), z(*shape))
        assert h.shape == shape and final.shape == (shape[0], shape[2])
        assert nn.gated_recurrence_grad(*[z(*shape)] * 4)[0].shape == shape


def test_recurrence_long_repeats():
    """A long axis over few channels: the same bits every time."""
    g = np.random.default_rng(12)
    gate, x, initial = _sequence(g, (1, 30_011, 70), np.float32, True)
    gate += 4
    args = [cp.array(a) for a in (gate, x, initial)]
    h, final = nn.gated_recurrence(*args)
    want, last, bound, off = _recur(gate, x, initial, True, E[np.float32])
    near(h, want, bound, np.float32)
    near(final, last, off, np.float32)
    grad = cp.array(g.standard_normal(gate.shape).astype(np.float32))
    first = nn.gated_recurrence_grad(grad, args[0], args[1], h, args[2])
    for a, (w, lim) in zip(first, _recur_grad(grad.get(), gate, x, h.get(), initial, 0 * initial,
                                              True, E[np.float32])):
        near(a, w, lim, np.float32)
    h0 = h.get()
    for _ in range(10):
        assert np.array_equal(nn.gated_recurrence(*args)[0].get(), h0)
        for a, b in zip(nn.gated_recurrence_grad(grad, args[0], args[1], h, args[2]), first):
            assert np.array_equal(a.get(), b.get())


@pytest.mark.parametrize("logits", [True, False])
@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("shape", [(1, 5003, 30), (1, 5003, 95), (2, 2100, 700), (1, 1025, 1000),
                                   (40, 700, 300), (100, 129, 257), (70, 200, 64), (9, 17, 513)],
                         **by_name)
def test_recurrence_layouts(shape, dt, logits):
    """Few channels and many steps, many channels, and in between; sequences
    that end inside a tile."""
    g = np.random.default_rng(sum(shape) + 2)
    gate, x, initial = _sequence(g, shape, dt, logits)
    h, final = nn.gated_recurrence(cp.array(gate), cp.array(x), cp.array(initial), logits=logits)
    want, last, bound, off = _recur(gate, x, initial, logits, E[dt])
    near(h, want, bound, dt)
    near(final, last, off, initial.dtype.type)
    grad = g.standard_normal(shape).astype(dt)
    end = g.standard_normal(initial.shape).astype(initial.dtype)
    got = nn.gated_recurrence_grad(*map(cp.array, (grad, gate, x)), h, cp.array(initial),
                                   cp.array(end), logits=logits)
    for a, (w, lim), t in zip(got, _recur_grad(grad, gate, x, h.get(), initial, end, logits, E[dt]),
                              (dt, dt, initial.dtype.type)):
        near(a, w, lim, t)


@pytest.mark.parametrize("dt", FLOATS, **by_name)
def test_recurrence_without_predecessors(dt):
    """Tiles that find no earlier tile's state in time join its steps
    themselves: the same bits."""
    from macmetalpy_amd._backend import HipBackend
    g = np.random.default_rng(13)
    for shape, logits in (((2, 4500, 70), True), ((2, 2100, 700), False), ((2, 2100, 700), True),
                          ((40, 700, 300), False), ((40, 700, 300), True)):
        gate, x, initial = _sequence(g, shape, dt, logits)
        args = [cp.array(a) for a in (gate, x, initial)]
        h, final = nn.gated_recurrence(*args, logits=logits)
        grads = nn.gated_recurrence_grad(args[1], args[0], args[1], h, args[2], logits=logits)
        HipBackend().debug_fail_next(4)
        h2, final2 = nn.gated_recurrence(*args, logits=logits)
        HipBackend().debug_fail_next(4)
        grads2 = nn.gated_recurrence_grad(args[1], args[0], args[1], h, args[2], logits=logits)
        for a, b in zip((h, final, *grads), (h2, final2, *grads2)):
            assert np.array_equal(a.get(), b.get())


def test_recurrence_past_32_bits():
    steps, dim = (1 << 20) + 5, 2053  # 2^31 elements and more
    gate = cp.zeros((steps, dim), dtype=np.float16)
    x = cp.zeros((steps, dim), dtype=np.float16)
    line = np.arange(dim, dtype=np.float16)
    x[steps - 1] = cp.array(line)
    x[steps - 3] = cp.array(line)
    h, final = nn.gated_recurrence(gate, x, logits=False)
    assert np.array_equal(final.get(), line.astype(np.float32))
    assert np.array_equal(h[steps - 4:].get(), np.stack([0 * line, line, 0 * line, line]))
    _, grad_x, _ = nn.gated_recurrence_grad(x, gate, x, h, logits=False)
    assert np.array_equal(grad_x[steps - 4:].get(), np.stack([0 * line, line, 0 * line, line]))


# ------------------------------------------------------------------ loss
def _loss_want(x, t, w, e, strips):
    """Loss and gradient in 64 bits, and bounds: the sum of exponentials, each
    with the rounding of x - m, is added in strips of `strips` elements and then joined."""
    x = x.astype(np.float64)
    classes = x.shape[-1]
    keep = (t >= 0) & (t < classes)
    at = np.where(keep, t, 0)[..., None]
    with np.errstate(invalid="ignore", divide="ignore", over="ignore"):
        m = x.max(-1, keepdims=True)
        ex = np.exp(x - m)
        s = ex.sum(-1, keepdims=True)
        xt = np.take_along_axis(x, at, -1)
        loss = (np.log(s) + (m - xt))[..., 0]
        spread = np.abs(np.where(np.isfinite(x - m), x - m, 0.0))
        rel = e * ((ex * spread).sum(-1, keepdims=True) / s + strips + 40)
        p = ex / s
        grad = p.copy()
        np.put_along_axis(grad, at, np.take_along_axis(p, at, -1) - 1, -1)
        w = np.broadcast_to(np.asarray(w, np.float64), t.shape)[..., None]
        lim = np.abs(w) * (p * (rel + e * (spread + 8)) + 4 * e * np.abs(grad))
        near_by = rel[..., 0] + e * (np.abs(m - xt)[..., 0] + 4 * np.abs(np.log(s))[..., 0])
    zero = np.zeros_like
    return (np.where(keep, loss, 0.0), np.where(keep, near_by, 0.0),
            np.where(keep[..., None], grad * w, zero(grad)), np.where(keep[..., None], lim, zero(lim)))


CLASSES = [1, 2, 7, 63, 64, 65, 500, 1000, 2049, 4097, 8193, 16_385, 33_000, 50_021, 66_000, 131_073,
           270_001]


@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("classes", CLASSES)
def test_cross_entropy(classes, dt):
    g = np.random.default_rng(classes)
    for rows in ((1, 9) if classes > 9000 else (1, 5, 70) if classes > 600 else (1, 3, 700)):
        x = (g.standard_normal((rows, classes)) * 4).astype(dt)
        t = g.integers(0, classes, rows)
        t[::4] = -1
        t[2::5] = classes
        t[-1] = classes - 1
        w = g.random(rows).astype(np.float64 if dt == np.float64 else np.float32) + 0.5
        want = _loss_want(x, t, w, E[dt], classes / 64 + 1)
        loss, grad = nn.cross_entropy_grad(cp.array(x), cp.array(t), cp.array(w))
        wide = w.dtype.type
        assert loss.dtype == wide and grad.dtype == dt
        near(loss, want[0], want[1], wide)
        near(grad, want[2], want[3], dt)
        near(nn.cross_entropy(cp.array(x), cp.array(t.astype(np.int32))), want[0], want[1], wide)


def test_cross_entropy_weights_and_shapes():
    g = np.random.default_rng(20)
    x = g.standard_normal((3, 4, 50)).astype(np.float32)
    t = g.integers(0, 50, (3, 4))
    for w in (1.0, 0.125, 0, np.float32(3)):
        want = _loss_want(x, t, w, E[np.float32], 50)
        loss, grad = nn.cross_entropy_grad(cp.array(x), cp.array(t), w)
        near(loss, want[0], want[1], np.float32)
        near(grad, want[2], want[3], np.float32)
    d = cp.array(x)
    for view in (lambda a: a[:, ::2, 3:40], lambda a: a.transpose(1, 0, 2), lambda a: a[::-1],
                 lambda a: a[..., ::5], lambda a: a[1, 2], lambda a: a[:, :0]):
        v = np.ascontiguousarray(view(x))
        tt = np.asarray(g.integers(0, v.shape[-1], v.shape[:-1]))
        want = _loss_want(v, tt, 1.0, E[np.float32], 50)
        loss, grad = nn.cross_entropy_grad(view(d), cp.array(tt))
        near(loss, want[0], want[1], np.float32)
        near(grad, want[2], want[3], np.float32)


@pytest.mark.parametrize("classes", [10, 1000, 40_000, 140_000])
@pytest.mark.parametrize("dt", FLOATS, **by_name)
def test_cross_entropy_extremes(dt, classes):
    g = np.random.default_rng(21)
    x = (g.standard_normal((12, classes)) * 2).astype(dt)
    t = g.integers(0, classes, 12)
    x[0, : classes - 3] = -np.inf  # classes that cannot be
    t[0] = classes - 1
    x[1, t[1]] = -np.inf           # the answer among them
    x[2] = -np.inf                 # nothing left
    x[3, 5] = np.inf
    x[4, 6] = np.nan
    x[5] = np.finfo(dt).min        # a mask of the lowest value on every class
    x[6, 1:] = np.finfo(dt).min
    t[6] = 0
    x[7] = np.finfo(dt).max
    x[8], t[8] = np.nan, -1        # ignored rows may hold anything
    x[9], t[9] = -np.inf, -1
    x[10] = -60.0
    x[10, 3] = 0.0
    with np.errstate(all="ignore"):
        want = _loss_want(x, t, 1.0, E[dt], classes / 64 + 1)
    loss, grad = nn.cross_entropy_grad(cp.array(x), cp.array(t))
    got, gg = loss.get(), grad.get()
    assert np.isnan(got[2:5]).all() and np.isnan(gg[2]).all() and np.isnan(gg[4]).all()
    assert np.isposinf(got[1]) and np.isfinite(gg[1]).all() and (gg[0, : classes - 3] == 0).all()
    assert (got[8:10] == 0).all() and (gg[8:10] == 0).all()
    ok = [0, 5, 6, 7, 10, 11]
    wide = np.float64 if dt == np.float64 else np.float32
    near(loss[cp.array(np.array(ok))], want[0][ok], want[1][ok], wide)
    ok.append(1)
    near(grad[cp.array(np.array(ok))], want[2][ok], want[3][ok], dt)
    assert np.array_equal(nn.cross_entropy(cp.array(x), cp.array(t)).get(), got, equal_nan=True)


def test_cross_entropy_differences():
    g = np.random.default_rng(22)
    x, t, w = g.standard_normal((3, 6)), np.array([2, -1, 5]), g.random(3)
    _, grad = nn.cross_entropy_grad(cp.array(x), cp.array(t), cp.array(w))
    grad, step = grad.get(), 1e-5
    for i in range(3):
        for c in range(6):
            ends = []
            for s in (step, -step):
                y = x.copy()
                y[i, c] += s
                ends.append(float((nn.cross_entropy(cp.array(y), cp.array(t)).get() * w).sum()))
            assert abs((ends[0] - ends[1]) / (2 * step) - grad[i, c]) < 1e-8


def test_cross_entropy_past_32_bits():
    rows, classes = 65_541, 32_800  # 2^31 elements and more
    x = cp.zeros((rows, classes), dtype=np.float16)
    x[rows - 1, classes - 1] = 5.0
    t = cp.full((rows,), classes - 1, dtype=np.int64)
    loss, grad = nn.cross_entropy_grad(x, t)
    last = np.log(classes - 1 + np.exp(5.0)) - 5.0
    loss = loss.get()
    assert np.allclose(loss[:-1], np.log(classes), rtol=1e-6) and np.isclose(loss[-1], last, rtol=1e-6)
    end = grad[rows - 1].get().astype(np.float64)
    assert np.isclose(end[-1], np.exp(-last) - 1, rtol=1e-3)
    assert np.allclose(end[:-1], np.exp(-last - 5.0), rtol=1e-2, atol=2.0 ** -25)


# ------------------------------------------------------------------ norm
def _arrays(g, sizes, dts):
    return [(g.standard_normal(n) * 0.3).astype(dt) for n, dt in zip(sizes, dts)]


@pytest.mark.parametrize("sizes", [(1,), (0, 5, 0), (3, 1, 4, 1, 5), (100_003, 7, 65_536), (70,) * 130,
                                   (3_000_001, 2_000_003), (1_000_001, 4096, 4097, 4095, 1)], **by_name)
@pytest.mark.parametrize("dts", [(np.float16,), (np.float32,), (np.float64,),
                                 (np.float16, np.float32), (np.float32, np.float64, np.float16)],
                         ids=lambda d: "-".join(t.__name__ for t in d))
def test_clip_by_global_norm(sizes, dts):
    g = np.random.default_rng(len(sizes))
    dts = [dts[i % len(dts)] for i in range(len(sizes))]
    host = _arrays(g, sizes, dts)
    wide = np.float64 if np.float64 in dts else np.float32
    norm = np.sqrt(sum((h.astype(np.float64) ** 2).sum() for h in host))
    dev = [cp.array(h) for h in host]
    got = nn.global_norm(dev)
    assert got.dtype == wide and got.shape == ()
    near(got, norm, 2e-15 * max(sizes) ** 0.5 * norm + 1e-14 * norm, wide)
    for limit in (0.5 * norm, 2.0 * norm, 0.0, np.inf):
        clipped, again = nn.clip_by_global_norm(dev, limit)
        assert again.get() == got.get()
        by = min(1.0, limit / norm) if norm else 1.0
        for c, h, dt in zip(clipped, host, dts):
            assert c.dtype == dt
            if by == 1.0:
                assert np.array_equal(c.get(), h)
            # the factor is rounded to 32 bits, and so is its product
            near(c, h.astype(np.float64) * by, 2.1 * E[dt] * np.abs(h.astype(np.float64) * by)
                 + 1e-14 * np.abs(h.astype(np.float64)), dt)
        assert all(np.array_equal(d.get(), h) for d, h in zip(dev, host))


def test_clip_in_place_and_views():
    g = np.random.default_rng(31)
    host = [g.standard_normal((40, 30)).astype(np.float32), g.standard_normal(9).astype(np.float16)]
    dev = [cp.array(h) for h in host]
    norm = np.sqrt(sum((h.astype(np.float64) ** 2).sum() for h in host))
    later = dev[0] + 1.0  # not evaluated yet: reads the values of before
    for limit in (100.0, 1.0):
        out, got = nn.clip_by_global_norm(dev, limit, out=dev)
        assert out[0] is dev[0] and np.isclose(got.get(), norm, rtol=1e-6)
        by = min(1.0, limit / norm)
        for d, h in zip(dev, host):
            assert np.allclose(d.get(), h.astype(np.float64) * by, rtol=2e-3 if d.dtype == np.float16 else 1e-6)
    assert np.array_equal(later.get(), host[0] + 1)
    d = cp.array(host[0])
    for view in (lambda a: a.T, lambda a: a[::2, 1:], lambda a: a[1:, :], lambda a: a[3, 1:]):
        (c,), got = nn.clip_by_global_norm([view(d)], 1.0)
        v = view(host[0]).astype(np.float64)
        assert np.allclose(got.get(), np.linalg.norm(v), rtol=1e-6)
        assert np.allclose(c.get(), v / max(1.0, np.linalg.norm(v)), rtol=1e-6)
    part = d[1:, :]  # a view written in place leaves the rest alone
    nn.clip_by_global_norm([part], 1.0, out=[part])
    assert np.array_equal(d.get()[0], host[0][0])
    assert np.allclose(d.get()[1:], host[0][1:] / np.linalg.norm(host[0][1:]), rtol=1e-6)


def test_norm_extremes():
    small = cp.array(np.full(1000, 1e-30, np.float32))  # and vanish in them
    assert np.isclose(float(nn.global_norm([small]).get()), 1e-30 * 1000 ** 0.5, rtol=1e-6)
    half = cp.array(np.full(100_000, 6e4, np.float16))
    assert np.isclose(float(nn.global_norm([half]).get()), float(np.float16(6e4)) * 1e5 ** 0.5, rtol=1e-6)
    mid = cp.array(np.full(4, 1e30, np.float32))
    (c,), n = nn.clip_by_global_norm([mid], 1.0)
    assert np.isclose(float(n.get()), 2e30, rtol=1e-6) and np.allclose(c.get(), 0.5, rtol=1e-6)
    h = np.ones(10, np.float32)
    h[3] = np.inf
    (c,), n = nn.clip_by_global_norm([cp.array(h)], 1.0)
    assert np.isposinf(n.get()) and np.isnan(c.get()[3]) and (np.delete(c.get(), 3) == 0).all()
    h[3] = np.nan
    (c,), n = nn.clip_by_global_norm([cp.array(h), ], 1.0)
    assert np.isnan(n.get()) and np.isnan(c.get()).all()
    clipped, n = nn.clip_by_global_norm([], 1.0)
    assert clipped == [] and float(n.get()) == 0.0


def test_norm_repeats():
    g = np.random.default_rng(32)
    dev = [cp.array(h) for h in _arrays(g, (3_000_001, 77, 500_000), [np.float32] * 3)]
    first = nn.global_norm(dev).get()
    assert all(nn.global_norm(dev).get() == first for _ in range(10))


# -------------------------------------------------------------- refusals
def test_refusals():
    f = lambda *s: cp.array(np.zeros(s, np.float32))  # noqa: E731
    i = lambda *s: cp.array(np.zeros(s, np.int64))  # noqa: E731
    with pytest.raises(TypeError, match="table must be floating"):
        nn.embedding(i(4, 4), i(3))
    with pytest.raises(TypeError, match="tokens must be integers"):
        nn.embedding(f(4, 4), f(3))
    with pytest.raises(ValueError, match="two axes"):
        nn.embedding(f(4), i(3))
    with pytest.raises(TypeError, match="scale must be a number"):
        nn.embedding(f(4, 4), i(3), scale="x")
    with pytest.raises(ValueError, match="does not fit tokens"):
        nn.embedding_grad(f(4, 5), i(3), 7)
    with pytest.raises(ValueError, match="does not fit tokens"):
        nn.embedding_grad(f(3), i(3), 7)
    with pytest.raises(ValueError, match="must not be negative"):
        nn.embedding_grad(f(3, 5), i(3), -1)
    with pytest.raises(TypeError, match="rows must be an integer"):
        nn.embedding_grad(f(3, 5), i(3), 2.0)
    with pytest.raises(TypeError, match="gate must be floating"):
        nn.gated_recurrence(i(2, 3, 4), f(2, 3, 4))
    with pytest.raises(ValueError, match="does not match gate"):
        nn.gated_recurrence(f(2, 3, 4), f(2, 3, 1))
    with pytest.raises(ValueError, match="axes for steps and channels"):
        nn.gated_recurrence(f(4), f(4))
    with pytest.raises(ValueError, match="initial of shape"):
        nn.gated_recurrence(f(2, 3, 4), f(2, 3, 4), f(2, 3))
    with pytest.raises(ValueError, match="h of shape"):
        nn.gated_recurrence_grad(f(2, 3, 4), f(2, 3, 4), f(2, 3, 4), f(2, 4, 4))
    with pytest.raises(ValueError, match="grad_final of shape"):
        nn.gated_recurrence_grad(*[f(2, 3, 4)] * 4, grad_final=f(3, 4))
    with pytest.raises(TypeError, match="logits must be floating"):
        nn.cross_entropy(i(2, 3), i(2))
    with pytest.raises(ValueError, match="do not fit targets"):
        nn.cross_entropy(f(2, 3), i(3))
    with pytest.raises(ValueError, match="no classes"):
        nn.cross_entropy(f(2, 0), i(2))
    with pytest.raises(ValueError, match="weight of shape"):
        nn.cross_entropy_grad(f(2, 3), i(2), f(3))
    with pytest.raises(TypeError, match="every array must be floating"):
        nn.global_norm([f(3), i(3)])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            nn.clip_by_global_norm([f(3)], bad)
    with pytest.raises(ValueError, match="out has 1 arrays for 2"):
        nn.clip_by_global_norm([f(3), f(3)], 1.0, out=[f(3)])
    with pytest.raises(ValueError, match="out of shape"):
        nn.clip_by_global_norm([f(3)], 1.0, out=[f(4)])
    with pytest.raises(ValueError, match="contiguous"):
        nn.clip_by_global_norm([f(3)], 1.0, out=[f(6)[::2]])
    with pytest.raises(TypeError, match="device arrays"):
        nn.clip_by_global_norm([f(3)], 1.0, out=[np.zeros(3, np.float32)])


def test_mixed_types():
    g = np.random.default_rng(40)
    gate, x = g.standard_normal((2, 5, 6)).astype(np.float16), g.standard_normal((2, 5, 6)).astype(np.float32)
    h, final = nn.gated_recurrence(cp.array(gate), cp.array(x))
    assert h.dtype == np.float32
    want, _, bound, _ = _recur(gate, x, np.zeros((2, 6)), True, E[np.float32])
    near(h, want, bound, np.float32)
    lazy = cp.array(x) * 2.0  # an expression not evaluated yet
    near(nn.gated_recurrence(cp.array(gate), lazy)[0], _recur(gate, 2 * x, np.zeros((2, 6)), True, 0)[0],
         2 * bound, np.float32)


def test_cross_entropy_many_short_rows():
    rows = 5_000_000
    x = cp.zeros((rows, 3), dtype=np.float32)
    t = cp.full((rows,), 1, dtype=np.int32)
    x[rows - 1, 1] = 2.0
    loss, grad = nn.cross_entropy_grad(x, t)
    loss = loss.get()
    assert np.allclose(loss[:-1], np.log(3), rtol=1e-6)
    assert np.isclose(loss[-1], np.log(2 + np.exp(2.0)) - 2, rtol=1e-6)
    assert np.allclose(grad[rows - 2].get(), [1 / 3, -2 / 3, 1 / 3], rtol=1e-6)


def test_embedding_many_tokens():
    """More tokens than the launch has workgroups for at once."""
    n, dim = (1 << 22) + 5, 1032
    tok = cp.array((np.arange(n) % 7).astype(np.int32))
    table = (np.arange(7 * dim) % 2003).astype(np.float16).reshape(7, dim)
    got = nn.embedding(cp.array(table), tok)
    for at in (0, n - 7, n - 6, n - 5, n - 4, n - 1):
        assert np.array_equal(got[at].get(), table[at % 7])
