"""A small recurrent language model on ``cp.nn``: training, and answering.

    python -m macmetalpy_amd.recurrent_lm

Tokens -> ``embedding`` -> a block (a product makes gates and inputs of one
array, ``gated_recurrence`` runs along the sequence, a product goes back, its
input is added) -> a product with the classes -> ``cross_entropy_grad``, then
the gradients in reverse, ``clip_by_global_norm`` and a step of descent.
Answers are drawn one token a call from the blocks' states, float32
throughout.  The text is synthetic: a number that counts up by a step of its
own, so the next token follows from the last two.
"""
from __future__ import annotations

import numpy as np

import macmetalpy_amd as cp
from macmetalpy_amd import nn

__all__ = ["RecurrentLM", "counting_text"]


def counting_text(rng, batch, steps, classes):
    """(batch, steps + 1) tokens; every sequence starts anywhere and goes up
    by 1, 2 or 3 modulo ``classes``."""
    start, by = rng.integers(0, classes, (batch, 1)), rng.integers(1, 4, (batch, 1))
    return ((start + by * np.arange(steps + 1)) % classes).astype(np.int32)


class RecurrentLM:
    def __init__(self, classes, dim, layers=2, seed=0):
        g = np.random.default_rng(seed)

        def weight(*shape):
            return cp.array((g.standard_normal(shape) / shape[0] ** 0.5).astype(np.float32))

        self.classes, self.dim, self.layers = classes, dim, layers
        # the table's rows are scaled by sqrt(dim) when they are looked up
        self.scale = dim ** 0.5
        self.weights = [cp.array((g.standard_normal((classes, dim)) / dim ** 0.5)
                                 .astype(np.float32))]
        for _ in range(layers):
            self.weights += [weight(dim, 2 * dim), weight(dim, dim)]
        self.weights.append(weight(dim, classes))

    def forward(self, tokens, states=None):
        """Logits (batch, steps, classes), the blocks' states after the last
        step, and what the gradients need."""
        d = self.dim
        y = nn.embedding(self.weights[0], tokens, scale=self.scale)
        kept, after = [], []
        for i in range(self.layers):
            into, back = self.weights[1 + 2 * i], self.weights[2 + 2 * i]
            both = y.reshape((-1, d)) @ into
            both = both.reshape(y.shape[:-1] + (2 * d,))
            gate, x = both[..., :d], both[..., d:]
            h, final = nn.gated_recurrence(gate, x, None if states is None else states[i])
            kept.append((y, gate, x, h))
            after.append(final)
            y = y + (h.reshape((-1, d)) @ back).reshape(y.shape)
        logits = (y.reshape((-1, d)) @ self.weights[-1]).reshape(y.shape[:-1] + (self.classes,))
        return logits, after, (kept, y)

    def gradients(self, tokens, targets):
        """The mean loss and the gradient of every weight.  Targets of -1 are
        not counted."""
        d = self.dim
        logits, _, (kept, y) = self.forward(tokens)
        count = max(1, int((np.asarray(targets) >= 0).sum()))
        loss, grad = nn.cross_entropy_grad(logits, cp.array(targets), 1.0 / count)
        grads = [None] * len(self.weights)
        grad = grad.reshape((-1, self.classes))
        grads[-1] = y.reshape((-1, d)).T @ grad
        grad = grad @ self.weights[-1].T
        for i in reversed(range(self.layers)):
            into, back = self.weights[1 + 2 * i], self.weights[2 + 2 * i]
            y, gate, x, h = kept[i]
            grads[2 + 2 * i] = h.reshape((-1, d)).T @ grad
            grad_h = (grad @ back.T).reshape(y.shape)
            grad_gate, grad_x, _ = nn.gated_recurrence_grad(grad_h, gate, x, h)
            both = cp.concatenate([grad_gate.reshape((-1, d)), grad_x.reshape((-1, d))], axis=1)
            grads[1 + 2 * i] = y.reshape((-1, d)).T @ both
            grad = grad + both @ into.T
        grads[0] = nn.embedding_grad(grad.reshape(y.shape), tokens, self.classes, scale=self.scale)
        return cp.sum(loss) / count, grads

    def train_step(self, text, rate=0.5, max_norm=1.0):
        """One step of descent on (batch, steps + 1) tokens; the mean loss and
        the gradients' norm, as device arrays."""
        tokens = cp.array(np.maximum(text[:, :-1], -1))
        loss, grads = self.gradients(tokens, np.ascontiguousarray(text[:, 1:]))
        grads, norm = nn.clip_by_global_norm(grads, max_norm)
        self.weights = [w - rate * g for w, g in zip(self.weights, grads)]
        cp.materialize(*self.weights)
        return loss, norm

    def answer(self, text, steps):
        """The likeliest ``steps`` tokens after each of (batch, n) texts, one
        token a call from the states."""
        logits, states, _ = self.forward(cp.array(text))
        out = []
        for _ in range(steps):
            token = cp.argmax(logits[:, -1], axis=-1).reshape((-1, 1))
            out.append(token)
            logits, states, _ = self.forward(token, states)
        return cp.concatenate(out, axis=1).get()


def main(train_steps=300, batch=32, steps=48, classes=61, dim=96):
    rng = np.random.default_rng(1)
    model = RecurrentLM(classes, dim)
    for step in range(train_steps):
        loss, norm = model.train_step(counting_text(rng, batch, steps, classes))
        if step % 50 == 0 or step == train_steps - 1:
            print(f"step {step}: loss {float(loss):.4f}, gradient norm {float(norm):.3f}", flush=True)
    text = counting_text(rng, 4, 28, classes)
    got = model.answer(text[:, :9], 20)
    for row, more in zip(text, got):
        print(" ".join(map(str, row[:9])), "->", " ".join(map(str, more)))
    print(f"right: {np.mean(got == text[:, 9:29]):.2f}")


if __name__ == "__main__":
    main()
