"""``cp.nn``'s gated delta rule against the recurrence itself, step by step in 64 bits."""
import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import nn

pytestmark = pytest.mark.gpu

FLOATS = [np.float16, np.float32, np.float64]
U = {np.float16: 2.0 ** -11, np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
# Half a unit of what states and sums are held in.
E = {np.float16: 2.0 ** -24, np.float32: 2.0 ** -24, np.float64: 2.0 ** -53}
by_name = {"ids": lambda v: getattr(v, "__name__", None) or str(v)}


def make(g, batch, steps, key_heads, heads, dk, dv, dt, anew=0.0, pad=0):
    unit = lambda *s: (lambda x: x / np.sqrt((x * x).sum(-1, keepdims=True)))(g.standard_normal(s))  # noqa: E731
    q, k = (unit(batch, steps, key_heads, dk).astype(dt) for _ in "qk")
    v = g.standard_normal((batch, steps, heads, dv)).astype(dt)
    gate = -np.exp(g.uniform(-6, 0.5, (batch, steps, heads)))
    gate[g.random((batch, steps, heads)) < anew] = -np.inf
    beta = g.random((batch, steps, heads))
    if pad:
        gate[:, -pad:], beta[:, -pad:] = 0.0, 0.0
    return q, k, v, gate.astype(dt), beta.astype(dt)


def rule(q, k, v, gate, beta, initial, scale):
    """o and final, step by step; the largest size of states that came by, head by head."""
    batch, steps, heads, dv = v.shape
    group = heads // k.shape[2]
    q, k, v, gate, beta = (x.astype(np.float64) for x in (q, k, v, gate, beta))
    q, k = np.repeat(q, group, 2), np.repeat(k, group, 2)
    S = np.zeros((batch, heads, k.shape[3], dv)) if initial is None else initial.astype(np.float64)
    o = np.zeros(v.shape)
    for t in range(steps):
        a = np.exp(gate[:, t])[..., None, None]
        S = np.where(a == 0, 0.0, a * S)
        u = beta[:, t, :, None] * (v[:, t] - (S * k[:, t, :, :, None]).sum(2))
        S = S + k[:, t, :, :, None] * u[:, :, None]
        o[:, t] = scale * (S * q[:, t, :, :, None]).sum(2)
    return o, S


def close(got, want, dt, rounding, parts):
    """The 2-norm of the difference over the result's: `parts` roundings of the state's type, which
    the recurrence (keys of length 1, beta at most 1: no step is longer than 1) does not enlarge,
    and the result's own rounding.  And each element within as many of the largest."""
    assert got.dtype == dt and got.shape == want.shape
    got = got.get().astype(np.float64)
    assert np.array_equal(np.isnan(got), np.isnan(want))
    size = np.sqrt(np.mean(want * want)) if want.size else 0.0
    off = np.abs(got - want)
    bound = rounding * 1.001 * np.abs(want) + parts * size + 2.0 ** -25 * (dt == np.float16)
    assert not off.size or np.max(off - bound) <= 0, (np.max(off - bound), np.max(off), size)


def parts_of(dt, steps, dk):
    """Relative error of states and outputs against their root mean square: sums of dk + chunk
    terms in the wide type (each term's rounding, added up as random ones, times 8 for the largest
    of all elements), over the steps that a state remembers.  float16's operands are pairs of
    float16 with 22 bits, or 2^-25 of 1 where the smaller one runs out of range; its P and T
    within a chunk have 22 and 11 bits, the latter for outputs alone."""
    n = np.sqrt(min(steps, 512) * (dk + 64)) * 8
    return n * E[dt] if dt != np.float16 else n * 2.0 ** -22


SIZES = [  # batch, steps, key heads, heads, dk, dv
    (1, 1, 1, 1, 1, 1), (2, 1, 2, 4, 33, 20), (3, 2, 1, 1, 128, 128), (1, 8, 2, 2, 256, 70), (2, 9, 1, 2, 16, 16),
    (1, 16, 1, 1, 64, 64), (1, 63, 2, 2, 40, 31), (2, 64, 1, 3, 128, 65), (1, 65, 2, 2, 129, 17), (2, 130, 3, 3, 72, 100),
    (1, 300, 1, 2, 200, 256), (1, 515, 2, 2, 8, 3)]


@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_delta_rule(dt, size):
    g = np.random.default_rng(sum(size))
    wide = np.float64 if dt == np.float64 else np.float32
    for start, anew in ((False, 0.0), (True, 0.05)):
        x = make(g, *size, dt, anew)
        batch, steps, key_heads, heads, dk, dv = size
        initial = g.standard_normal((batch, heads, dk, dv)).astype(wide) if start else None
        scale = dk ** -0.5
        o, S = rule(*x, initial, scale)
        got_o, got_s = nn.gated_delta_rule(*map(cp.array, x), None if initial is None else cp.array(initial))
        parts = parts_of(dt, steps, dk)
        # an output of float16 has P's and T's own roundings too
        close(got_o, o, dt, U[dt], parts + (8 * U[dt] if dt == np.float16 else 0))
        close(got_s, S, wide, U[wide], parts)


def rule_grad(grad, q, k, v, gate, beta, initial, grad_final, scale):
    """The gradients by the chain rule of one step, from the last to the first, in 64 bits."""
    batch, steps, heads, dv = v.shape
    shared = k.shape[2]
    group = heads // shared
    grad, q, k, v, gate, beta = (x.astype(np.float64) for x in (grad, q, k, v, gate, beta))
    q, k = np.repeat(q, group, 2), np.repeat(k, group, 2)
    S = np.zeros((batch, heads, k.shape[3], dv)) if initial is None else initial.astype(np.float64)
    seen = []
    for t in range(steps):
        a = np.exp(gate[:, t])[..., None, None]
        faded = np.where(a == 0, 0.0, a * S)
        miss = v[:, t] - (faded * k[:, t, :, :, None]).sum(2)
        u = beta[:, t, :, None] * miss
        S = faded + k[:, t, :, :, None] * u[:, :, None]
        seen.append((faded, miss, u, S))
    D = np.zeros_like(S) if grad_final is None else grad_final.astype(np.float64)
    gq, gk, gv, gg, gb = (np.zeros(x.shape) for x in (q, k, v, gate, beta))
    for t in reversed(range(steps)):
        faded, miss, u, S = seen.pop()
        go = scale * grad[:, t]
        gq[:, t] = (S * go[:, :, None]).sum(3)
        D = D + q[:, t, :, :, None] * go[:, :, None]
        du = (D * k[:, t, :, :, None]).sum(2)
        dm = beta[:, t, :, None] * du
        gb[:, t] = (du * miss).sum(2)
        gv[:, t] = dm
        gk[:, t] = (D * u[:, :, None]).sum(3) - (faded * dm[:, :, None]).sum(3)
        D = D - k[:, t, :, :, None] * dm[:, :, None]
        gg[:, t] = (D * faded).sum((2, 3))
        a = np.exp(gate[:, t])[..., None, None]
        D = np.where(a == 0, 0.0, a * D)
    join = lambda x: x.reshape(batch, steps, shared, group, -1).sum(3)  # noqa: E731
    return join(gq), join(gk), gv, gg, gb, D


def grads_close(got, want, dt, steps, dk, dv):
    """As the outputs; every gradient of float16 has operands rounded to it (states, their
    gradients, U and dR, P's and T's products): U each, of addends that are random in sign, 8 times
    the root mean square for the largest element.  A gate's gradient sums those of dk dv products
    and all later steps of its chunk and so may be larger than its parts' difference: their size
    is taken from the sums' largest."""
    wide = np.float64 if dt == np.float64 else np.float32
    parts = parts_of(dt, steps, max(dk, dv)) * 2
    loose = parts + (8 * 3 * U[dt] if dt == np.float16 else 0)
    for i, (a, b) in enumerate(zip(got[:5], want[:5])):
        close(a, b, dt, U[dt], loose * (8 if i == 3 else 2))
    close(got[5], want[5], wide, U[wide], parts)


@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("size", SIZES, ids=str)
def test_delta_rule_grad(dt, size):
    g = np.random.default_rng(sum(size) + 1)
    wide = np.float64 if dt == np.float64 else np.float32
    for start, anew in ((False, 0.0), (True, 0.05)):
        x = make(g, *size, dt, anew)
        batch, steps, key_heads, heads, dk, dv = size
        states = [g.standard_normal((batch, heads, dk, dv)).astype(wide) if start else None for _ in range(2)]
        grad = g.standard_normal(x[2].shape).astype(dt)
        want = rule_grad(grad, *x, *states, dk ** -0.5)
        got = nn.gated_delta_rule_grad(cp.array(grad), *map(cp.array, x), *(None if s is None else cp.array(s) for s in states))
        grads_close(got, want, dt, steps, dk, dv)


@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("size", [(1, 4160, 1, 1, 64, 33), (1, 2100, 2, 4, 130, 64), (2, 1500, 1, 1, 256, 16)], ids=str)
def test_long_sequences(dt, size):
    """Few heads and many chunks: segments that run at once, with and without fresh starts."""
    if dt == np.float64:
        size = (size[0], size[1] // 4) + size[2:]
    g = np.random.default_rng(size[1])
    wide = np.float64 if dt == np.float64 else np.float32
    batch, steps, key_heads, heads, dk, dv = size
    for anew in (0.0, 0.003):
        x = make(g, *size, dt, anew)
        # memories of some thousand steps: states pass many segments
        x = x[:3] + ((x[3].astype(np.float64) * 1e-2).astype(dt),) + x[4:]
        states = [g.standard_normal((batch, heads, dk, dv)).astype(wide) for _ in range(2)]
        o, S = rule(*x, states[0], dk ** -0.5)
        got_o, got_s = nn.gated_delta_rule(*map(cp.array, x), cp.array(states[0]))
        parts = parts_of(dt, steps, dk) * 4
        close(got_o, o, dt, U[dt], parts + (8 * U[dt] if dt == np.float16 else 0))
        close(got_s, S, wide, U[wide], parts)
        grad = g.standard_normal(x[2].shape).astype(dt)
        want = rule_grad(grad, *x, *states, dk ** -0.5)
        got = nn.gated_delta_rule_grad(cp.array(grad), *map(cp.array, x), *map(cp.array, states))
        loose = parts + (8 * 3 * U[dt] if dt == np.float16 else 0)
        for i in range(5):
            close(got[i], want[i], dt, U[dt], loose * (8 if i == 3 else 2))
        close(got[5], want[5], wide, U[wide], parts * 2)


@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("steps", [1, 6, 70])
def test_views(dt, steps):
    """Slices of one projection, reversed and broadcast arrays, gates of either type: the bits of
    contiguous copies."""
    g = np.random.default_rng(steps)
    b, h, kh, dk, dv = 2, 4, 2, 16, 24
    wide = np.float64 if dt == np.float64 else np.float32
    parts = cp.array((g.standard_normal((b, steps, 2 * kh * dk + h * dv + 5)) * 0.2).astype(dt))
    q = parts[..., :kh * dk].reshape((b, steps, kh, dk))
    k = parts[..., kh * dk:2 * kh * dk].reshape((b, steps, kh, dk))
    v = parts[..., 2 * kh * dk + 5:].reshape((b, steps, h, dv))
    both = cp.array(g.standard_normal((2, h, steps, b)).astype(wide))
    gate, beta = -cp.abs(both[0]).transpose((2, 1, 0)), cp.abs(both[1]).transpose((2, 1, 0)) * 0.3
    grad = cp.array(g.standard_normal((b, steps, h, 2 * dv)).astype(dt))[..., ::2]
    plain = lambda a: cp.array(np.ascontiguousarray(a.get()))  # noqa: E731
    cases = [(q, k, v, gate, beta, grad), (q[::-1], k[:, ::-1], v, gate, beta, grad),
             (cp.broadcast_to(q[:1], q.shape), k, cp.broadcast_to(v[:, :, :1], v.shape), gate, beta, grad)]
    for q_, k_, v_, gate_, beta_, grad_ in cases:
        got = nn.gated_delta_rule(q_, k_, v_, gate_, beta_)
        want = nn.gated_delta_rule(*map(plain, (q_, k_, v_, gate_, beta_)))
        for x, y in zip(got, want):
            assert x.dtype == y.dtype and np.array_equal(x.get(), y.get())
        got = nn.gated_delta_rule_grad(grad_, q_, k_, v_, gate_, beta_)
        want = nn.gated_delta_rule_grad(*map(plain, (grad_, q_, k_, v_, gate_, beta_)))
        assert [x.dtype for x in got] == [np.dtype(t) for t in (dt, dt, dt, wide, wide, wide)]
        for x, y in zip(got, want):
            assert np.array_equal(x.get(), y.get())


@pytest.mark.parametrize("dt", FLOATS, **by_name)
def test_steps_go_on(dt):
    """Token by token, in pieces and at once: the states agree to their own roundings."""
    g = np.random.default_rng(8)
    x = make(g, 2, 100, 1, 2, 32, 24, dt)
    parts = parts_of(dt, 100, 32) + (8 * U[dt] if dt == np.float16 else 0)
    o, S = rule(*x, None, 32 ** -0.5)
    for cuts in (range(0, 101), (0, 8, 17, 64, 100), (0, 99, 100)):
        state, rows = None, []
        for a, b in zip(cuts[:-1], cuts[1:]):
            row, state = nn.gated_delta_rule(*(cp.array(np.ascontiguousarray(v[:, a:b])) for v in x), state)
            rows.append(row.get())
        close(cp.array(np.concatenate(rows, 1)), o, dt, U[dt], parts)
        close(state, S, state.dtype.type, 0.0, parts)


def test_padding_and_fresh_starts():
    """Steps with a gate and a beta of 0 leave the state; a gate of -inf is as no state before."""
    g = np.random.default_rng(9)
    for dt in FLOATS:
        x = make(g, 1, 90, 1, 1, 16, 16, dt, pad=20)
        _, S = nn.gated_delta_rule(*map(cp.array, x))
        _, T = nn.gated_delta_rule(*(cp.array(np.ascontiguousarray(v[:, :70])) for v in x))
        wide = T.dtype.type
        close(S, T.get().astype(np.float64), wide, 0.0, parts_of(dt, 70, 16))
        x[3][:, 40] = -np.inf
        start = cp.array(g.standard_normal((1, 1, 16, 16)).astype(wide))
        o, S = nn.gated_delta_rule(*map(cp.array, x), start)
        p, T = nn.gated_delta_rule(*(cp.array(np.ascontiguousarray(v[:, 40:])) for v in x))
        close(S, T.get().astype(np.float64), wide, 0.0, parts_of(dt, 90, 16))
        close(cp.array(np.ascontiguousarray(o.get()[:, 40:])), p.get().astype(np.float64), dt, 2 * U[dt],
              parts_of(dt, 90, 16) + 8 * U[dt] * (dt == np.float16))
        # outputs from the fresh start on alone: nothing before it has a gradient
        grad = x[2].copy()
        grad[:, :40] = 0
        grads = nn.gated_delta_rule_grad(cp.array(grad), *map(cp.array, x), start)
        assert not np.any(grads[0].get()[:, :40]) and not np.any(grads[2].get()[:, :40])
        assert float(grads[3].get()[0, 40, 0]) == 0.0 and not np.any(grads[5].get())


def test_empty():
    for dt in FLOATS:
        wide = np.float64 if dt == np.float64 else np.float32
        z = lambda *s: cp.zeros(s, dtype=dt)  # noqa: E731
        one = cp.ones((2, 3, 4, 5), dtype=wide)
        o, S = nn.gated_delta_rule(z(2, 0, 1, 4), z(2, 0, 1, 4), z(2, 0, 3, 5), z(2, 0, 3), z(2, 0, 3), one)
        assert o.shape == (2, 0, 3, 5) and np.array_equal(S.get(), one.get())
        grads = nn.gated_delta_rule_grad(z(2, 0, 3, 5), z(2, 0, 1, 4), z(2, 0, 1, 4), z(2, 0, 3, 5), z(2, 0, 3), z(2, 0, 3), one, one)
        assert np.array_equal(grads[5].get(), one.get())
        for steps in (3, 20):
            o, S = nn.gated_delta_rule(z(2, steps, 1, 0), z(2, steps, 1, 0), z(2, steps, 3, 5), z(2, steps, 3), z(2, steps, 3))
            assert S.shape == (2, 3, 0, 5) and not np.any(o.get())
            grads = nn.gated_delta_rule_grad(z(2, steps, 3, 5), z(2, steps, 1, 0), z(2, steps, 1, 0), z(2, steps, 3, 5), z(2, steps, 3), z(2, steps, 3))
            assert not any(np.any(g.get()) for g in grads)
            k = cp.ones((2, steps, 1, 4), dtype=dt)
            o, S = nn.gated_delta_rule(k, k, z(2, steps, 3, 0), z(2, steps, 3), z(2, steps, 3))
            assert o.shape == (2, steps, 3, 0) and S.shape == (2, 3, 4, 0)
            grads = nn.gated_delta_rule_grad(z(2, steps, 3, 0), k, k, z(2, steps, 3, 0), z(2, steps, 3), z(2, steps, 3))
            assert not any(np.any(g.get()) for g in grads)
            o, S = nn.gated_delta_rule(k, k, z(2, steps, 0, 5), z(2, steps, 0), z(2, steps, 0))
            assert o.shape == (2, steps, 0, 5)
            grads = nn.gated_delta_rule_grad(z(2, steps, 0, 5), k, k, z(2, steps, 0, 5), z(2, steps, 0), z(2, steps, 0))
            assert not np.any(grads[0].get()) and not np.any(grads[1].get())
            assert nn.gated_delta_rule(z(0, steps, 1, 4), z(0, steps, 1, 4), z(0, steps, 2, 5), z(0, steps, 2), z(0, steps, 2))[0].size == 0


def test_differences():
    """The gradient against differences of the operator itself, in 64 bits."""
    g = np.random.default_rng(11)
    x = [a.astype(np.float64) for a in make(g, 1, 37, 1, 2, 6, 5, np.float64)]
    states = [g.standard_normal((1, 2, 6, 5)) for _ in range(2)]
    grad = g.standard_normal(x[2].shape)

    def value(args):
        o, S = nn.gated_delta_rule(*map(cp.array, args))
        return float((o.get() * grad).sum() + (S.get() * states[1]).sum())

    args = x + [states[0]]
    grads = nn.gated_delta_rule_grad(cp.array(grad), *map(cp.array, args), cp.array(states[1]))
    step = 1e-5
    for i, a in enumerate(args):
        d = g.standard_normal(a.shape)
        move = lambda by: [b + by * d if j == i else b for j, b in enumerate(args)]  # noqa: E731
        slope = (value(move(step)) - value(move(-step))) / (2 * step)
        want = float((grads[i].get() * d).sum())
        # third derivatives of order 1e4 times step^2 / 6, and 2^-53 of values of some 1e2 over step
        assert abs(slope - want) <= 1e4 * step ** 2 + 1e2 * 2.0 ** -53 / step * 10


def test_repeats():
    """The same bits every time."""
    g = np.random.default_rng(12)
    for dt in FLOATS:
        x = [cp.array(a) for a in make(g, 2, 700, 2, 4, 48, 40, dt, 0.01)]
        first = nn.gated_delta_rule(*x) + nn.gated_delta_rule_grad(x[2], *x)
        again = nn.gated_delta_rule(*x) + nn.gated_delta_rule_grad(x[2], *x)
        assert all(np.array_equal(a.get(), b.get(), equal_nan=True) for a, b in zip(first, again))


def test_refusals():
    z = lambda *s, dt=np.float32: cp.zeros(s, dtype=dt)  # noqa: E731
    q, v, g = z(2, 3, 2, 4), z(2, 3, 4, 5), z(2, 3, 4)
    for bad, error in (((z(2, 3, 8), q, v, g, g), ValueError), ((q, z(2, 3, 2, 5), v, g, g), ValueError),
                       ((q, q, z(2, 4, 4, 5), g, g), ValueError), ((q, q, z(2, 3, 3, 5), z(2, 3, 3), z(2, 3, 3)), ValueError),
                       ((q, q, v, z(2, 3, 2), g), ValueError), ((q, q, v, g, z(2, 3)), ValueError),
                       ((z(2, 3, 2, 257), z(2, 3, 2, 257), v, g, g), ValueError),
                       ((q, q, v, g, cp.zeros((2, 3, 4), dtype=np.int32)), TypeError),
                       ((z(2, 3, 0, 4), z(2, 3, 0, 4), v, g, g), ValueError),
                       ((q, q, v, g, g, z(2, 4, 5, 4)), ValueError), ((q, q, v, g, g, None), None)):
        if error is None:
            nn.gated_delta_rule(*bad)
            continue
        with pytest.raises(error):
            nn.gated_delta_rule(*bad)
        with pytest.raises(error):
            nn.gated_delta_rule_grad(v, *bad)
    with pytest.raises(TypeError):
        nn.gated_delta_rule(q, q, v, g, g, scale="1")
    with pytest.raises(ValueError):
        nn.gated_delta_rule_grad(q, q, q, v, g, g)
    with pytest.raises(ValueError):
        nn.gated_delta_rule_grad(v, q, q, v, g, g, None, z(2, 4, 4, 4))
