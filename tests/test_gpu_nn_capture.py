"""The operators of ``cp.nn`` while the library's stream is captured into a
graph: what keeps nothing in the library's memory replays with new inputs, the
rest is refused."""
import ctypes

import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import _abi
from macmetalpy_amd._backend import HipBackend, HipUnsupportedError, load_library
from test_zz_no_alloc import HIP_STREAM_CAPTURE_MODE_RELAXED, _hip_runtime

pytestmark = pytest.mark.gpu

F32, I64 = (_abi.DTYPE_CODES[np.dtype(t)] for t in (np.float32, np.int64))


def _captured(call):
    """The graph of ``call()`` and what it raised, if it did."""
    hip, lib = _hip_runtime(), load_library()
    HipBackend().synchronize()
    stream, graph = ctypes.c_void_p(), ctypes.c_void_p()
    assert lib.mmp_stream(ctypes.byref(stream)) == 0 and stream.value
    assert hip.hipStreamBeginCapture(stream, HIP_STREAM_CAPTURE_MODE_RELAXED) == 0
    error = None
    try:
        call()
    except HipUnsupportedError as e:
        error = e
    finally:
        end = hip.hipStreamEndCapture(stream, ctypes.byref(graph))
    assert end == 0 and graph.value
    return hip, stream, graph, error


class _Data:
    """Named device arrays; new values go into the same memory."""

    def __init__(self, **shapes):
        self.a = {k: cp.zeros(s, dtype=d) for k, (s, d) in shapes.items()}
        cp.materialize(*self.a.values())
        for v in self.a.values():
            v._ensure_gpu()

    def __getattr__(self, name):
        return self.a[name]._ptr

    def put(self, name, host):
        v = self.a[name]
        assert host.shape == v.shape and host.dtype == v.dtype
        HipBackend().write_buffer(v._buffer, 0, host.ravel())

    def get(self, name):
        HipBackend().synchronize()
        return self.a[name].copy().get()


def _rand(g, *shape):
    return g.standard_normal(shape).astype(np.float32)


def _embed(g):
    n, rows, dim = 90, 50, 33
    d = _Data(tok=((n,), np.int64), table=((rows, dim), np.float32), out=((n, dim), np.float32))
    new = lambda: (d.put("tok", g.integers(-1, rows, n)), d.put("table", _rand(g, rows, dim)))  # noqa: E731
    call = lambda: HipBackend().embedding(F32, I64, n, d.tok, rows, dim, d.table, dim, 1.5, d.out)  # noqa: E731
    return d, new, call, ["out"]


def _embed_grad(g):
    n, rows, dim = 128, 50, 33
    d = _Data(tok=((n,), np.int64), grad=((n, dim), np.float32), out=((rows, dim), np.float32))
    new = lambda: (d.put("tok", g.integers(-1, rows, n)), d.put("grad", _rand(g, n, dim)))  # noqa: E731
    call = lambda: HipBackend().embedding_grad(F32, I64, n, d.tok, d.grad, dim, rows, dim, 1.5, d.out)  # noqa: E731
    return d, new, call, ["out"]


def _recur(steps):
    def case(g):
        b, dim = 3, 37
        s = ((b, steps, dim), np.float32)
        d = _Data(gate=s, x=s, h=s, final=((b, dim), np.float32))
        at = lambda p: (p, steps * dim, dim)  # noqa: E731
        new = lambda: [d.put(k, _rand(g, b, steps, dim)) for k in ("gate", "x")]  # noqa: E731
        call = lambda: HipBackend().recurrence(F32, 1, b, steps, dim, at(d.gate), at(d.x), None,  # noqa: E731
                                               d.h, d.final)
        return d, new, call, ["h", "final"]
    return case


def _recur_grad(steps):
    def case(g):
        b, dim = 3, 37
        s = ((b, steps, dim), np.float32)
        d = _Data(grad=s, gate=s, x=s, h=s, og=s, ox=s, oi=((b, dim), np.float32))
        at = lambda p: (p, steps * dim, dim)  # noqa: E731
        new = lambda: [d.put(k, _rand(g, b, steps, dim)) for k in ("grad", "gate", "x", "h")]  # noqa: E731
        call = lambda: HipBackend().recurrence_grad(  # noqa: E731
            F32, 1, b, steps, dim, at(d.grad), at(d.gate), at(d.x), at(d.h), None, None, d.og, d.ox, d.oi)
        return d, new, call, ["og", "ox", "oi"]
    return case


def _loss(rows, classes, grad):
    def case(g):
        d = _Data(x=((rows, classes), np.float32), t=((rows,), np.int64), loss=((rows,), np.float32),
                  grad=((rows, classes), np.float32))
        new = lambda: (d.put("x", _rand(g, rows, classes)), d.put("t", g.integers(-1, classes, rows)))  # noqa: E731
        call = lambda: HipBackend().cross_entropy(F32, I64, rows, classes, d.x, classes, d.t, None,  # noqa: E731
                                                  1.0, d.loss, d.grad if grad else None)
        return d, new, call, ["loss", "grad"] if grad else ["loss"]
    return case


def _clip(g):
    d = _Data(x=((5000,), np.float32), out=((5000,), np.float32), norm=((), np.float32))
    new = lambda: d.put("x", _rand(g, 5000))  # noqa: E731
    call = lambda: HipBackend().clip_norm([F32], [5000], [d.x], [d.out], 1.0, F32, d.norm)  # noqa: E731
    return d, new, call, ["out", "norm"]


def _many_tokens(g):
    n, rows, dim = 129, 50, 33
    d = _Data(tok=((n,), np.int64), grad=((n, dim), np.float32), out=((rows, dim), np.float32))
    new = lambda: (d.put("tok", g.integers(-1, rows, n)), d.put("grad", _rand(g, n, dim)))  # noqa: E731
    call = lambda: HipBackend().embedding_grad(F32, I64, n, d.tok, d.grad, dim, rows, dim, 1.5, d.out)  # noqa: E731
    return d, new, call, ["out"]


REPLAY = {"embed": _embed, "embed_grad": _embed_grad, "recur_step": _recur(1), "recur_16": _recur(16),
          "recur_one_tile": _recur(60), "recur_grad_16": _recur_grad(16), "loss": _loss(7, 300, False),
          "loss_grad": _loss(7, 300, True), "loss_long": _loss(2, 270_001, False),
          "loss_grad_long": _loss(2, 270_001, True)}
REFUSED = {"recur": _recur(1500), "recur_grad": _recur_grad(1500), "embed_grad": _many_tokens,
           "clip": _clip}


@pytest.mark.parametrize("name", REPLAY)
def test_replays_follow_the_inputs(name):
    """Four replays, each with new inputs and eager work in between, against the
    eager call.  A long row's parts are summed in another order when eager."""
    d, new, call, outs = REPLAY[name](np.random.default_rng(50))
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
                if "long" in name:
                    assert np.allclose(a, b, rtol=1e-5, atol=1e-9)
                else:
                    assert np.array_equal(a, b)
                assert np.isfinite(a).all() and a.any()
    finally:
        if exe.value:
            hip.hipGraphExecDestroy(exe)
        hip.hipGraphDestroy(graph)


@pytest.mark.parametrize("name", REFUSED)
def test_scratch_memory_is_not_captured(name):
    d, new, call, outs = REFUSED[name](np.random.default_rng(51))
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
