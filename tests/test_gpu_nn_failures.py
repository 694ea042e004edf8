"""``cp.nn`` when an allocation or a launch fails, and from several host threads
at once.  Failures are injected by the library's test hook: no kernel runs
wrong, faults or hangs."""
import gc
import threading

import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import nn
from macmetalpy_amd._backend import HipBackend, HipError

pytestmark = pytest.mark.gpu

ALLOCATION, LAUNCH = 1, 3


def _operators(seed, scale=1):
    """Calls that take memory and launch several kernels, by name: each returns
    what it made, from inputs of its own."""
    g = np.random.default_rng(seed)
    f = lambda *s: cp.array(g.standard_normal(s).astype(np.float32))  # noqa: E731
    i = lambda hi, *s: cp.array(g.integers(-1, hi, s))  # noqa: E731
    steps = 700 * scale
    table, tok = f(500, 40), i(500, 20_000 * scale)
    grad = f(20_000 * scale, 40)
    few, few_grad = i(500, 100), f(100, 40)
    passes, passes_grad = i(70_000, 140_000), f(140_000, 3)
    gate, x, h = f(3, steps, 70), f(3, steps, 70), f(3, steps, 70)
    short = f(5, 7, 33)
    logits, t = f(60, 900), i(900, 60)
    row, rt = f(1, 200_000), i(200_000, 1)
    arrays = [f(n) for n in (5, 70_000 * scale, 1001)]
    return {
        "embedding": lambda: [nn.embedding(table, tok)],
        "embedding_grad": lambda: [nn.embedding_grad(grad, tok, 500)],
        "embedding_grad_few": lambda: [nn.embedding_grad(few_grad, few, 500)],
        "embedding_grad_passes": lambda: [nn.embedding_grad(passes_grad, passes, 70_000)],
        "recurrence": lambda: nn.gated_recurrence(gate, x),
        "recurrence_short": lambda: nn.gated_recurrence(short, short),
        "recurrence_grad": lambda: nn.gated_recurrence_grad(x, gate, x, h),
        "recurrence_grad_short": lambda: nn.gated_recurrence_grad(short, short, short, short),
        "loss": lambda: [nn.cross_entropy(logits, t)],
        "loss_grad": lambda: nn.cross_entropy_grad(logits, t),
        "loss_parts": lambda: [nn.cross_entropy(row, rt)],
        "loss_grad_parts": lambda: nn.cross_entropy_grad(row, rt),
        "norm": lambda: [nn.global_norm(arrays)],
        "clip": lambda: nn.clip_by_global_norm(arrays, 1.0)[0],
    }


def _in_use():
    gc.collect()
    cp.synchronize()
    return HipBackend().memory_stats()[0]


def _equal(got, want):
    return len(got) == len(want) and all(np.array_equal(a.get(), b) for a, b in zip(got, want))


@pytest.fixture(scope="module")
def calls():
    return _operators(80)


@pytest.fixture
def be():
    b = HipBackend()
    yield b
    b.debug_fail_next(0, 0)  # disarm whatever a failed test left armed


@pytest.mark.parametrize("kind", [ALLOCATION, LAUNCH], ids=["allocation", "launch"])
@pytest.mark.parametrize("name", [
    "embedding", "embedding_grad", "embedding_grad_few", "embedding_grad_passes", "recurrence",
    "recurrence_short", "recurrence_grad", "recurrence_grad_short", "loss", "loss_grad",
    "loss_parts", "loss_grad_parts", "norm", "clip"])
def test_failures_are_raised_and_leave_nothing(be, calls, name, kind):
    """The first, second, ... allocation or launch of a call fails, until the call
    has no more of them: an error each time, no memory kept, the next call right."""
    call = calls[name]
    out = call()
    want = [a.get() for a in out]
    del out
    before = _in_use()
    for k in range(1, 20):
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
        assert k > 1 and _equal(out, want)
        return
    raise AssertionError("the call never got through")


def test_threads():
    """Recurrences of lengths that make the tiles' memory grow under each
    other's calls, and the other operators, each thread with arrays of its own."""
    works = [_operators(90 + k, scale=1 + 3 * k) for k in range(4)]
    wants = [{n: [a.get() for a in call()] for n, call in w.items()} for w in works]
    errors = []

    def work(k):
        try:
            for turn in range(6):
                for j in range(len(works[k])):
                    name = list(works[k])[(j + 3 * k + turn) % len(works[k])]
                    assert _equal(works[k][name](), wants[k][name]), (k, turn, name)
        except BaseException as e:  # reported by the main thread
            errors.append(repr(e))

    threads = [threading.Thread(target=work, args=(k,)) for k in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join(timeout=100)
    assert not any(t.is_alive() for t in threads), "a worker thread did not finish"
    assert not errors, errors
    cp.synchronize()
