"""The matrix state language model: its gradients against the whole model's in 64
bits on the CPU, and answers a token at a time against the whole text's."""
import numpy as np
import pytest
import torch

import macmetalpy_amd as cp
from macmetalpy_amd import nn
from macmetalpy_amd.delta_lm import DeltaLM, paired_text

pytestmark = pytest.mark.gpu


def plain_loss(model, weights, tokens, targets, keep):
    """The model in elementary torch operations; ``keep``: the dropouts' factors in order."""
    batch, steps = tokens.shape
    h, dk, dv = model.heads, model.dk, model.dv
    y = weights[0][tokens] * model.scale
    for i in range(model.layers):
        into, back, ffn, down = weights[1 + 4 * i:5 + 4 * i]
        parts = y @ into
        q, k, v, a, b = parts.split([h * dk, h * dk, h * dv, h, h], -1)
        q, k, v = (x.reshape(batch, steps, h, -1) for x in (q, k, v))
        q, k = (x / (x.square().sum(-1, keepdim=True) + 1e-12).sqrt() for x in (q, k))
        decay, beta = torch.sigmoid(a + 3.0), torch.sigmoid(b)
        state, out = torch.zeros(batch, h, dk, dv, dtype=y.dtype), []
        for t in range(steps):
            state = decay[:, t, :, None, None] * state
            u = beta[:, t, :, None] * (v[:, t] - (state * k[:, t, :, :, None]).sum(2))
            state = state + k[:, t, :, :, None] * u[:, :, None]
            out.append((state * q[:, t, :, :, None]).sum(2))
        o = torch.stack(out, 1).reshape(batch, steps, h * dv)
        y = y + keep[2 * i] * (o @ back)
        both = y @ ffn
        half = both.shape[-1] // 2
        g = both[..., :half]
        y = y + keep[2 * i + 1] * ((g * torch.sigmoid(g) * both[..., half:]) @ down)
    logits = y @ weights[-1]
    at = targets >= 0
    loss = torch.logsumexp(logits, -1) - logits.gather(-1, targets.clamp(min=0)[..., None])[..., 0]
    return (loss * at).sum() / at.sum()


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
    keep = [torch.from_numpy(nn.dropout(cp.ones(tokens.shape + (24,), dtype=np.float64), 0.2, 9,
                                        first + j * size).get()) for j in range(4)]
    assert model.drawn == first + 4 * size
    weights = [torch.from_numpy(w.get()).requires_grad_() for w in model.weights]
    want = plain_loss(model, weights, torch.from_numpy(tokens.astype(np.int64)),
                      torch.from_numpy(targets), keep)
    want.backward()
    # sums of some thousand terms of order 1 in 64 bits, through a few products
    assert abs(float(loss) - want.item()) < 1e-11
    for g, w in zip(grads, weights):
        assert np.abs(g.get() - w.grad.numpy()).max() < 1e-11


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
