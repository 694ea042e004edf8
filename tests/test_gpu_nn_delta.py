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
