"""How far a NaN reaches in ``cp.nn``'s block operators, and that none comes from memory
that an earlier call left."""
import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import nn

pytestmark = pytest.mark.gpu

FLOATS = [np.float16, np.float32, np.float64]
by_name = {"ids": lambda v: getattr(v, "__name__", None) or str(v)}


def _rule(g, batch, steps, key_heads, heads, dk, dv, dt):
    unit = lambda *s: (lambda x: x / np.sqrt((x * x).sum(-1, keepdims=True)))(g.standard_normal(s))  # noqa: E731
    x = [unit(batch, steps, key_heads, dk), unit(batch, steps, key_heads, dk), g.standard_normal((batch, steps, heads, dv)),
         -g.random((batch, steps, heads)), g.random((batch, steps, heads)), g.standard_normal((batch, steps, heads, dv))]
    return [a.astype(dt) for a in x]


def _run(x):
    *inputs, grad = (cp.array(a) for a in x)
    out = nn.gated_delta_rule(*inputs) + nn.gated_delta_rule_grad(grad, *inputs)
    return dict(zip(("o", "final", "q", "k", "v", "gate", "beta", "initial"), (a.get() for a in out)))


@pytest.mark.parametrize("bad", [np.nan, np.inf])
@pytest.mark.parametrize("dt", FLOATS, **by_name)
@pytest.mark.parametrize("size", [(2, 6, 40, 70), (2, 200, 40, 70), (2, 200, 64, 64), (1, 2000, 64, 32)], ids=str)
def test_delta_rule(size, dt, bad):
    """In a value: other heads have the same bits, and its own outputs those of
    the chunks (at most 64 steps) before."""
    batch, steps, dk, dv = size
    x = _rule(np.random.default_rng(steps + dk), batch, steps, 2, 4, dk, dv, dt)
    clean = _run(x)
    at = steps * 3 // 4
    x[2][0, at, 1, dv // 2] = bad
    got = _run(x)
    assert np.array_equal(got["o"][0, :at // 64 * 64], clean["o"][0, :at // 64 * 64])
    assert not np.isfinite(got["final"][0, 1]).all()
    for name in got:
        axis = 1 if name in ("final", "initial") else 2
        of = [1] if got[name].shape[axis] == 2 else [0, 2, 3]  # q's and k's heads are shared by two
        a, b = (np.take(r[name][0], of, axis=axis - 1) for r in (got, clean))
        assert np.array_equal(a, b), name
        assert np.array_equal(got[name][1:], clean[name][1:]), name


@pytest.mark.parametrize("dt", FLOATS, **by_name)
def test_memory_of_earlier_calls(dt):
    """The same bits when freed memory holds NaN."""
    g = np.random.default_rng(7)
    calls = {}
    for size in ((2, 5, 1, 2, 33, 20), (1, 70, 1, 3, 40, 31), (1, 1500, 1, 2, 72, 100), (3, 130, 2, 2, 200, 16)):
        calls[f"delta {size}"] = lambda x=_rule(g, *size, dt): list(_run(x).values())
    for rows, dim, hidden in ((3, 37, 23), (9, 2050, 300), (300, 130, 77)):
        x, w, d = (cp.array(g.standard_normal(s).astype(dt)) for s in ((rows, dim), (dim, 2 * hidden), (rows, hidden)))
        calls[f"feed-forward {rows, dim, hidden}"] = lambda x=x, w=w, d=d: [
            a.get() for a in (nn.gated_feed_forward(x, w), *nn.gated_feed_forward_grad(d, x, w))]
    x = cp.array(g.standard_normal(1003).astype(dt))
    calls["dropout"] = lambda: [nn.dropout(x, 0.3, 1, 2).get()]
    want = {n: call() for n, call in calls.items()}
    for name, call in calls.items():
        spoiled = [cp.full(2 ** k * m // 16, np.nan, dtype=np.float32) for k in range(8, 26) for m in (4, 5, 6, 7) for _ in range(3)]
        cp.materialize(*spoiled)
        del spoiled
        got = call()
        assert all(np.isfinite(a).all() for a in got), name
        assert all(np.array_equal(a, b) for a, b in zip(got, want[name])), name
