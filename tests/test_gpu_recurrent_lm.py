"""The small recurrent language model: its gradients, its training and its
answers one token at a time."""
import numpy as np
import pytest

import macmetalpy_amd as cp
from macmetalpy_amd import nn
from macmetalpy_amd.recurrent_lm import RecurrentLM, counting_text

pytestmark = pytest.mark.gpu


def test_gradients():
    """Against central differences of the loss in 64 bits."""
    rng = np.random.default_rng(0)
    model = RecurrentLM(7, 4, layers=2, seed=1)
    host = [w.get().astype(np.float64) for w in model.weights]
    text = counting_text(rng, 3, 6, 7)
    text[1, 4:] = -1  # a shorter sequence
    tokens, targets = cp.array(text[:, :-1].copy()), text[:, 1:].copy()

    def loss_of(weights):
        model.weights = [cp.array(w) for w in weights]
        logits, _, _ = model.forward(tokens)
        return float(nn.cross_entropy(logits, cp.array(targets)).get().sum() / (targets >= 0).sum())

    model.weights = [cp.array(w) for w in host]
    loss, grads = model.gradients(tokens, targets)
    grads = [g.get() for g in grads]
    assert abs(float(loss) - loss_of(host)) < 1e-12
    step = 1e-5
    for k, g in enumerate(grads):
        for i in rng.choice(g.size, min(g.size, 12), replace=False):
            ends = []
            for s in (step, -step):
                moved = [w.copy() for w in host]
                moved[k].reshape(-1)[i] += s
                ends.append(loss_of(moved))
            assert abs((ends[0] - ends[1]) / (2 * step) - g.reshape(-1)[i]) < 1e-7


def test_trains_and_answers():
    rng = np.random.default_rng(2)
    model = RecurrentLM(29, 64)
    losses = [float(model.train_step(counting_text(rng, 32, 40, 29))[0]) for _ in range(150)]
    assert losses[-1] < 0.3 * losses[0]
    # the states that single tokens go on from are those of the whole text
    text = counting_text(rng, 5, 30, 29)
    whole, _, _ = model.forward(cp.array(text[:, :-1].copy()))
    states, rows = None, []
    for t in range(30):
        logits, states, _ = model.forward(cp.array(text[:, t:t + 1].copy()), states)
        rows.append(logits.get())
    whole = whole.get()
    assert np.abs(np.concatenate(rows, 1) - whole).max() < 1e-4 * np.abs(whole).max()
    assert model.answer(text[:, :9], 4).shape == (5, 4)
