"""The matrix state language model: its loss and gradients against the whole model in plain
NumPy in 64 bits, and answers a token at a time against the whole text's."""
import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import nn
from macmetalpy_amd.delta_lm import DeltaLM, paired_text

pytestmark = pytest.mark.gpu


def plain_loss(model, weights, tokens, targets, keep):
    """The model step by step; ``keep``: the dropouts' factors in order."""
    batch, steps = tokens.shape
    h, dk, dv = model.heads, model.dk, model.dv
    sigmoid = lambda x: 1.0 / (1.0 + np.exp(-x))  # noqa: E731
    y = weights[0][tokens] * model.scale
    for i in range(model.layers):
        into, back, ffn, down = weights[1 + 4 * i:5 + 4 * i]
        q, k, v, a, b = np.split(y @ into, np.cumsum([h * dk, h * dk, h * dv, h]), -1)
        q, k, v = (x.reshape(batch, steps, h, -1) for x in (q, k, v))
        q, k = (x / np.sqrt((x * x).sum(-1, keepdims=True) + 1e-12) for x in (q, k))
        decay, beta = sigmoid(a + 3.0), sigmoid(b)
        state, out = np.zeros((batch, h, dk, dv)), []
        for t in range(steps):
            state = decay[:, t, :, None, None] * state
            u = beta[:, t, :, None] * (v[:, t] - (state * k[:, t, :, :, None]).sum(2))
            state = state + k[:, t, :, :, None] * u[:, :, None]
            out.append((state * q[:, t, :, :, None]).sum(2))
        o = np.stack(out, 1).reshape(batch, steps, h * dv)
        y = y + keep[2 * i] * (o @ back)
        g, up = np.split(y @ ffn, 2, -1)
        y = y + keep[2 * i + 1] * ((g * sigmoid(g) * up) @ down)
    logits = y @ weights[-1]
    top = logits.max(-1, keepdims=True)
    lse = np.log(np.exp(logits - top).sum(-1)) + top[..., 0]
    loss = lse - np.take_along_axis(logits, np.maximum(targets, 0)[..., None], -1)[..., 0]
    return (loss * (targets >= 0)).sum() / (targets >= 0).sum()


def test_gradients():
    rng = np.random.default_rng(3)
    model = DeltaLM(11, 24, layers=2, heads=3, dk=5, dv=7, hidden=20, rate=0.2, seed=9,
                    dtype=np.float64)
    text = paired_text(rng, 4, 11, 5, 6)
    tokens, targets = text[:, :-1], text[:, 1:].astype(np.int64)
    targets[1, 5:] = -1
    first = model.drawn
    loss, grads = model.gradients(cp.array(tokens), targets)
    size = tokens.size * model.dim
    keep = [nn.dropout(cp.ones(tokens.shape + (24,), dtype=np.float64), 0.2, 9, first + j * size).get()
            for j in range(4)]
    assert model.drawn == first + 4 * size
    weights = [w.get() for w in model.weights]
    # sums of some thousand terms of order 1 in 64 bits, through a few products
    assert abs(float(loss) - plain_loss(model, weights, tokens, targets, keep)) < 1e-11
    # each weight's gradient along a few directions of length 1, against differences of the plain
    # model: third derivatives of order 1e2 times step^2 / 6, and 2^-53 of some units over step
    step = 1e-5
    for i, g in enumerate(grads):
        for _ in range(3):
            d = rng.standard_normal(g.shape)
            d /= np.linalg.norm(d)
            at = lambda by: plain_loss(model, weights[:i] + [weights[i] + by * d] + weights[i + 1:], tokens, targets, keep)  # noqa: E731
            slope = (at(step) - at(-step)) / (2 * step)
            assert abs(slope - float((g.get() * d).sum())) < 1e2 * step ** 2 + 16 * 2.0 ** -53 / step, i


def test_answers_token_by_token():
    """Each token's logits from the states alone are those of the whole text: float32, states
    handed on unrounded, so only the order of sums differs (some hundred terms of order 1)."""
    rng = np.random.default_rng(4)
    model = DeltaLM(16, 32, layers=2)
    text = cp.array(paired_text(rng, 5, 40, 8, 8))
    whole = model.forward(text)[0].get()
    states, rows = None, []
    for t in range(80):
        logits, states, _ = model.forward(text[:, t:t + 1], states)
        rows.append(logits.get())
    assert np.abs(np.concatenate(rows, 1) - whole).max() < 2e-3 * np.abs(whole).max()
    first = model.forward(text[:, :50])
    rest = model.forward(text[:, 50:], first[1])[0].get()
    assert np.abs(rest - whole[:, 50:]).max() < 2e-3 * np.abs(whole).max()


def test_training_runs():
    rng = np.random.default_rng(5)
    model = DeltaLM(16, 32)
    for _ in range(3):
        loss, norm = model.train_step(paired_text(rng, 8, 12, 8, 8))
        assert np.isfinite(float(loss)) and np.isfinite(float(norm))
    assert model.answer(paired_text(rng, 3, 6, 8, 8), 4).shape == (3, 4)
