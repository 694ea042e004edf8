"""``cp.nn`` at the limits of its plans and arguments, against plain NumPy in
64 bits."""
import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import nn

pytestmark = pytest.mark.gpu


def _sums(tok, grad, rows):
    """Sums of whole numbers by token, exact in any order."""
    want = np.zeros((rows, grad.shape[1]), np.float32)
    keep = (tok >= 0) & (tok < rows)
    np.add.at(want, tok[keep], grad[keep].astype(np.float32))
    return want


# ------------------------------------------------------------- embedding
@pytest.mark.parametrize("rows", [1 << 24, (1 << 24) + 1, (1 << 24) + 5, (1 << 25) + 3])
def test_embedding_grad_rows_beyond_24_bits(rows):
    """Rows that differ only in their bits from 24 on, the first and the last."""
    g = np.random.default_rng(rows)
    tok = g.integers(0, rows, 700)
    tok[:8] = [0, rows - 1, rows, -1, 5, min(rows - 1, (1 << 24) + 5 - 4), 1, rows - 1]
    tok[8:300] = g.integers(0, 3, 292) + (rows - 3)
    tok[300:400] = g.integers(0, 5, 100)
    grad = g.integers(-8, 9, (700, 1)).astype(np.float16)
    got = nn.embedding_grad(cp.array(grad), cp.array(tok), rows).get()
    assert np.array_equal(got.astype(np.float32), _sums(tok, grad, rows))


# ------------------------------------------------------------------ norm
def test_clip_refuses_outputs_that_overlap():
    """An output on another array's memory, or on a part of its own, would be
    scaled once or twice; arrays that only touch are others."""
    h = np.arange(1, 41, dtype=np.float32)
    a, b = cp.array(h), cp.array(h + 1)
    bad = [([a, a], [a, a]),                     # tied weights' gradients
           ([a, b], [b, a]),                     # two arrays that change places
           ([a[:15], b[:15]], [a[20:35], a[25:40]]),
           ([a[:20]], [a[1:21]]),                # a part of its own
           ([a[:20], b[:20]], [a[:20], a[10:30]]),
           ([a, b], [a, a]), ([a, a], [a, b])]
    for arrays, out in bad:
        with pytest.raises(ValueError, match="overlaps another array"):
            nn.clip_by_global_norm(arrays, 1.0, out=out)
    assert np.array_equal(a.get(), h) and np.array_equal(b.get(), h + 1)
    norm = np.sqrt(2 * (h.astype(np.float64) ** 2).sum())
    (c, d), n = nn.clip_by_global_norm([a, a], 1.0)  # read twice, written elsewhere
    assert np.isclose(n.get(), norm, rtol=1e-6)
    assert np.allclose(c.get(), h / norm, rtol=1e-6) and np.array_equal(c.get(), d.get())
    parts = [a[:10], a[10:10], a[10:11], a[11:]]     # side by side, one of them empty
    nn.clip_by_global_norm(parts, 1.0, out=parts)
    assert np.allclose(a.get(), h / np.linalg.norm(h), rtol=1e-6)


@pytest.mark.parametrize("dt,size,limits", [
    (np.float32, 1e38, (1.0, 1e-2, 1e-3, 1e-5, 1e-20, 3e-36)),
    (np.float64, 1e150, (1.0, 1e-150, 1e-160, 1e-200, 1e-290))],
    ids=["float32", "float64"])
def test_clip_factors_below_the_normal_range(dt, size, limits):
    """limit / norm has few bits or none as a number of the arrays' type, the
    results have all of theirs: a product of two factors of one rounding each."""
    g = np.random.default_rng(60)
    host = [(g.uniform(0.5, 1.0, n) * g.choice([-1, 1], n) * size).astype(dt) for n in (9001, 7, 1030)]
    host[1][3] = 0.0
    norm = np.sqrt(sum(((h.astype(np.float64) / size) ** 2).sum() for h in host))
    for limit in limits:
        clipped, got = nn.clip_by_global_norm([cp.array(h) for h in host], limit)
        same = [cp.array(h) for h in host]
        nn.clip_by_global_norm(same, limit, out=same)
        if dt == np.float64:
            assert np.isclose(float(got.get()), norm * size, rtol=1e-12)
        for c, s, h in zip(clipped, same, host):
            want = h.astype(np.float64) / size / norm * limit
            off = np.abs(c.get().astype(np.float64) - want)
            # the factor's rounding and the result's; the norm's sum of 10^4 squares
            assert (off <= (2.5 * np.finfo(dt).eps + 1e-13) * np.abs(want)).all(), limit
            assert np.array_equal(s.get(), c.get())


@pytest.mark.parametrize("rows", [1 << 18, (1 << 18) + 1, 1 << 19, (1 << 19) + 1, 1 << 20, (1 << 20) + 1])
@pytest.mark.parametrize("n", [129, 4096, 4097, 8192, 8193, 16_384, 16_385, 1 << 17, (1 << 17) + 1])
def test_embedding_grad_most_counters(rows, n):
    """Rows that fill the counters of a workgroup, and one more; tokens on both
    sides of what its waves keep and of the passes."""
    g = np.random.default_rng(rows + n)
    tok = g.integers(0, rows, n)
    tok[::9] = rows - 1 - tok[::9] % 300
    tok[::31] = 7
    tok[:4] = [0, rows - 1, rows, -1]
    grad = g.integers(-3, 4, (n, 2)).astype(np.float32)
    got = nn.embedding_grad(cp.array(grad), cp.array(tok), rows).get()
    assert np.array_equal(got, _sums(tok, grad, rows))


# ------------------------------------------------------------------ loss
@pytest.mark.parametrize("dt", [np.float16, np.float32, np.float64], ids=lambda t: t.__name__)
def test_loss_weight_on_the_device_is_not_waited_for(dt, monkeypatch):
    """A mean's weight that the device computed, as one number: used where it is."""
    g = np.random.default_rng(70)
    wide = np.float64 if dt == np.float64 else np.float32
    x, t = cp.array(g.standard_normal((4, 5, 33)).astype(dt)), g.integers(-1, 33, (4, 5))
    targets = cp.array(t)
    factor = wide(1024.0 / (t >= 0).sum())
    want = nn.cross_entropy_grad(x, targets, float(factor))
    weights = [cp.array(np.array(factor)), 1024.0 / cp.sum((targets >= 0).astype(wide)),
               cp.array(np.array(3, np.int32))]
    cp.materialize(*weights)

    def wait(self, *args):
        raise AssertionError("a device array was read on the host")

    with monkeypatch.context() as m:
        for name in ("get", "__float__", "item"):
            m.setattr(cp.ndarray, name, wait)
        got = [nn.cross_entropy_grad(x, targets, w) for w in weights]
        one = nn.cross_entropy_grad(x[0, 0], targets[0, 0], weights[0])
        assert nn.cross_entropy_grad(x[:0], targets[:0], weights[0])[1].shape == (0, 5, 33)
    for loss, grad in got[:2]:
        assert grad.dtype == dt
        assert np.array_equal(loss.get(), want[0].get()) and np.array_equal(grad.get(), want[1].get())
    assert np.array_equal(got[2][1].get(), nn.cross_entropy_grad(x, targets, 3)[1].get())
    assert np.array_equal(one[1].get(), want[1].get()[0, 0])


# -------------------------------------------------------------- refusals
@pytest.mark.parametrize("text", ["2", b"2", "nan", bytearray(b"2")])
def test_numbers_as_text_are_refused(text):
    f, i = cp.array(np.ones((3, 4), np.float32)), cp.array(np.zeros(3, np.int64))
    for call, name in ((lambda: nn.embedding(f, i, scale=text), "scale"),
                       (lambda: nn.embedding_grad(f, i, 5, scale=text), "scale"),
                       (lambda: nn.cross_entropy_grad(f, i, text), "weight"),
                       (lambda: nn.clip_by_global_norm([f], text), "max_norm")):
        with pytest.raises(TypeError, match=name + " must be a number"):
            call()


# ------------------------------------------------------------ recurrence
HALVES = np.arange(1 << 16, dtype=np.uint16).view(np.float16)


def _gates(dt, low, high):
    """Every float16 number between two, in type dt."""
    with np.errstate(invalid="ignore"):
        return HALVES[(HALVES >= low) & (HALVES <= high)].astype(dt)


@pytest.mark.parametrize("dt", [np.float16, np.float32, np.float64], ids=lambda t: t.__name__)
def test_recurrence_keeps_a_constant(dt):
    """A state of 1 and inputs of 1 stay 1 whatever the gate, but for rounding,
    however many calls follow each other.  With e the exponential, d = 1 + e is
    rounded by E / (1 + e) at most, its reciprocal by E (1 + e) / 2, the product
    of the two by E / 4 and the new state by E, together 2.75 E a step
    (an error of e itself leaves f + u as it is); a step keeps f of the error before."""
    e = 2.0 ** -53 if dt == np.float64 else 2.0 ** -24
    gate = _gates(dt, -4, 6)
    left = 1.0 / (1.0 + np.exp(gate.astype(np.float64)))  # 1 - f
    gates = cp.array(np.broadcast_to(gate, (16, gate.size)).copy())
    ones = cp.ones((16, gate.size), dtype=dt)
    state = cp.ones((gate.size,), dtype=np.float64 if dt == np.float64 else np.float32)
    for _ in range(64):
        _, state = nn.gated_recurrence(gates, ones, state)
    off = np.abs(state.get().astype(np.float64) - 1.0) * left / e
    assert off.max() <= 2.8, off.max()


@pytest.mark.parametrize("dt", [np.float32, np.float64], ids=lambda t: t.__name__)
def test_recurrence_state_of_one_step(dt):
    """From nothing and an input of 1 the state is 1 - f = e / (1 + e): e is rounded
    by 3 E (the device's exponential by a unit, 2 E, its correction by E), d by E, its
    reciprocal by E and the product by E."""
    gate = _gates(dt, -20, 20)
    want = 1.0 / (1.0 + np.exp(gate.astype(np.longdouble)))
    _, final = nn.gated_recurrence(cp.array(gate.reshape(1, -1)), cp.ones((1, gate.size), dtype=dt))
    off = np.abs(final.get() - want) / want / (2.0 ** -53 if dt == np.float64 else 2.0 ** -24)
    assert float(off.max()) <= 6.1, off.max()
