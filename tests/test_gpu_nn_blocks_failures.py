"""``cp.nn``'s block operators (delta rule, feed-forward, dropout) while the stream
is captured, when an allocation or a launch fails, and from several host threads
at once.  Failures are injected by the library's test hook: no kernel runs
wrong, faults or hangs."""
import ctypes
import threading

import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import _abi, nn
from macmetalpy_amd._backend import HipBackend, HipError
from test_gpu_nn_capture import _captured, _Data
from test_gpu_nn_failures import ALLOCATION, LAUNCH, _equal, _in_use, be  # noqa: F401

pytestmark = pytest.mark.gpu

CODE = {np.float16: _abi.DTYPE_CODES[np.dtype(np.float16)], np.float32: _abi.DTYPE_CODES[np.dtype(np.float32)]}


def _normal(g, shape, dt):
    return g.standard_normal(shape).astype(dt)


# -------------------------------------------------------------- captured
def _dropout(g):
    n = 4099
    d = _Data(x=((n,), np.float16), r=((n,), np.float16), at=((), np.int64), y=((n,), np.float16))
    new = lambda: (d.put("x", _normal(g, n, np.float16)), d.put("r", _normal(g, n, np.float16)),  # noqa: E731
                   d.put("at", np.array(g.integers(0, 1 << 40))))
    call = lambda: HipBackend().dropout(CODE[np.float16], n, d.x, d.r, 0.3, 7, 5, d.at, d.y)  # noqa: E731
    return d, new, call, ["y"]


def _delta(steps, dt):
    def case(g):
        b, kh, h, dk, dv = 2, 1, 2, 40, 33
        d = _Data(q=((b, steps, kh, dk), dt), k=((b, steps, kh, dk), dt), v=((b, steps, h, dv), dt),
                  gate=((b, steps, h), dt), beta=((b, steps, h), dt), o=((b, steps, h, dv), dt),
                  s=((b, h, dk, dv), np.float32), end=((b, h, dk, dv), np.float32))

        def new():
            for n, shape in (("q", (b, steps, kh, dk)), ("k", (b, steps, kh, dk)), ("v", (b, steps, h, dv))):
                d.put(n, _normal(g, shape, dt) * dt(0.1))
            d.put("gate", -np.abs(_normal(g, (b, steps, h), dt)))
            d.put("beta", np.abs(_normal(g, (b, steps, h), dt)))
            d.put("s", _normal(g, (b, h, dk, dv), np.float32))

        keys, values, gates = (steps * kh * dk, kh * dk, dk), (steps * h * dv, h * dv, dv), (0, steps * h, h, 1)
        call = lambda: HipBackend().delta_rule(  # noqa: E731
            CODE[dt], b, steps, kh, h, dk, dv, d.q, *keys, d.k, *keys, d.v, *values, d.gate, *gates, d.beta, *gates,
            d.s, 1.0, d.o, d.end)
        return d, new, call, ["o", "end"]
    return case


def _ffn(rows, dim, hidden, dt, grad=False):
    def case(g):
        d = _Data(x=((rows, dim), dt), w=((dim, 2 * hidden), dt), h=((rows, hidden), dt), gx=((rows, dim), dt),
                  gw=((dim, 2 * hidden), dt))
        new = lambda: (d.put("x", _normal(g, (rows, dim), dt)), d.put("w", _normal(g, (dim, 2 * hidden), dt)),  # noqa: E731
                       d.put("h", _normal(g, (rows, hidden), dt)) if grad else None)
        if grad:
            call = lambda: HipBackend().gated_feed_forward_grad(CODE[dt], 0, rows, dim, hidden, d.h, hidden, d.x, dim,  # noqa: E731
                                                                d.w, 2 * hidden, d.gx, d.gw)
            return d, new, call, ["gx", "gw"]
        call = lambda: HipBackend().gated_feed_forward(CODE[dt], 1, rows, dim, hidden, d.x, dim, d.w, 2 * hidden, d.h)  # noqa: E731
        return d, new, call, ["h"]
    return case


REPLAY = {"dropout": _dropout, "delta_token": _delta(1, np.float16), "delta_8": _delta(8, np.float32),
          "ffn": _ffn(70, 96, 64, np.float16), "ffn_few": _ffn(3, 512, 264, np.float16),
          "ffn32": _ffn(5, 8, 8, np.float32), "ffn32_few": _ffn(3, 512, 264, np.float32)}
REFUSED = {"delta": _delta(9, np.float16), "delta_long": _delta(700, np.float32),
           "ffn_odd": _ffn(5, 9, 8, np.float16), "ffn_grad": _ffn(5, 8, 8, np.float16, True),
           "ffn_grad32": _ffn(5, 8, 8, np.float32, True)}


@pytest.mark.parametrize("name", REPLAY)
def test_replays_follow_the_inputs(name):
    """Four replays, each with new inputs and eager work in between, against the eager call.  A
    feed-forward product may be cut into ranges of k when eager: sums of `dim` terms in another
    order, within dim units of 2^-24 of their size, and float16's rounding."""
    d, new, call, outs = REPLAY[name](np.random.default_rng(60))
    new()
    stats = HipBackend().memory_stats()
    hip, stream, graph, error = _captured(call)
    assert error is None and HipBackend().memory_stats() == stats
    exe = ctypes.c_void_p()
    try:
        assert hip.hipGraphInstantiate(ctypes.byref(exe), graph, None, None, 0) == 0
        for _ in range(4):
            new()
            assert hip.hipGraphLaunch(exe, stream) == 0
            got = [d.get(k) for k in outs]
            call()
            for k, a in zip(outs, got):
                b = d.get(k)
                if name.endswith("_few"):
                    assert np.allclose(a.astype(float), b.astype(float), rtol=2.0 ** -9, atol=512 * 2.0 ** -24 * 512)
                else:
                    assert np.array_equal(a, b)
                assert np.isfinite(a).all() and a.any()
    finally:
        if exe.value:
            hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


@pytest.mark.parametrize("name", REFUSED)
def test_scratch_memory_is_not_captured(name):
    d, new, call, outs = REFUSED[name](np.random.default_rng(61))
    new()
    call()
    want = [d.get(k) for k in outs]
    stats = HipBackend().memory_stats()
    hip, _, graph, error = _captured(call)
    hip.hipGraphDestroy(graph)
    assert error is not None and "cannot be captured" in str(error)
    assert HipBackend().memory_stats() == stats
    call()  # and goes on as before
    assert all(np.array_equal(d.get(k), w) for k, w in zip(outs, want))


# -------------------------------------------------------------- failures
def _operators(seed, scale=1):
    g = np.random.default_rng(seed)
    f = lambda dt, *s: cp.array((g.standard_normal(s) * 0.3).astype(dt))  # noqa: E731
    made = {}
    for dt in (np.float16, np.float32):
        for name, steps in (("short", 5), ("chunks", 70 * scale), ("segments", 1100)):
            x = [f(dt, 1, steps, 1, 24), f(dt, 1, steps, 1, 24), f(dt, 1, steps, 2, 20), -cp.abs(f(dt, 1, steps, 2)),
                 cp.abs(f(dt, 1, steps, 2))]
            cp.materialize(*x[3:])
            key = f"{name}_{np.dtype(dt).name}"
            made["delta_" + key] = lambda x=x: nn.gated_delta_rule(*x)
            made["delta_grad_" + key] = lambda x=x: nn.gated_delta_rule_grad(x[2], *x)
        for name, (rows, dim, hidden) in (("odd", (33 * scale, 41, 27)), ("even", (64, 512 * scale, 40))):
            x, w, d = f(dt, rows, dim), f(dt, dim, 2 * hidden), f(dt, rows, hidden)
            key = f"{name}_{np.dtype(dt).name}"
            made["ffn_" + key] = lambda x=x, w=w: [nn.gated_feed_forward(x, w)]
            made["ffn_grad_" + key] = lambda x=x, w=w, d=d: nn.gated_feed_forward_grad(d, x, w)
    x = f(np.float32, 1000 * scale)
    made["dropout"] = lambda: [nn.dropout(x, 0.5, seed)]
    return made


@pytest.fixture(scope="module")
def calls():
    return _operators(80)


@pytest.mark.parametrize("kind", [ALLOCATION, LAUNCH], ids=["allocation", "launch"])
@pytest.mark.parametrize("name", [
    f"{op}_{size}_{dt}" for op, sizes in (("delta", ("short", "chunks", "segments")), ("delta_grad", ("short", "chunks", "segments")),
                                          ("ffn", ("odd", "even")), ("ffn_grad", ("odd", "even")))
    for size in sizes for dt in ("float16", "float32")] + ["dropout"])
def test_failures_are_raised_and_leave_nothing(be, calls, name, kind):  # noqa: F811
    """The first, second, ... allocation or launch of a call fails, until the call
    has no more of them: an error each time, no memory kept, the next call right."""
    call = calls[name]
    out = call()
    want = [a.get() for a in out]
    del out
    before = _in_use()
    for k in range(1, 40):
        be.debug_fail_next(kind, k)
        out = None
        try:
            out = call()
        except HipError as e:
            assert "injected" in str(e)
        if out is None:  # what the error's traceback held is free by now
            assert _in_use() == before, k
            out = call()
            assert _equal(out, want), k
            continue
        be.debug_fail_next(0, 0)
        if kind == LAUNCH:
            assert k > 1
        # (a product does without ranges of k where their memory is missing)
        assert name.startswith("ffn") or _equal(out, want)
        return
    raise AssertionError("the call never got through")


def test_threads():
    """Each thread with arrays of its own."""
    works = [_operators(90 + k, scale=1 + 2 * k) for k in range(3)]
    wants = [{n: [a.get() for a in call()] for n, call in w.items()} for w in works]
    errors = []

    def work(k):
        try:
            for turn in range(3):
                for j in range(len(works[k])):
                    name = list(works[k])[(j + 3 * k + turn) % len(works[k])]
                    assert _equal(works[k][name](), wants[k][name]), (k, turn, name)
        except BaseException as e:  # reported by the main thread
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(3)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not any(t.is_alive() for t in threads), "a worker thread did not finish"
    assert not errors, errors
    cp.synchronize()
