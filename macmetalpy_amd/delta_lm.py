"""A small language model of matrix states on ``cp.nn``: training, and answering.

    python -m macmetalpy_amd.delta_lm

Tokens -> ``embedding`` -> blocks -> a product with the classes ->
``cross_entropy_grad``, then the gradients in reverse, ``clip_by_global_norm`` and a
step of descent.  A block is a product that makes queries, keys, values and gates
of its input, ``gated_delta_rule`` over keys and queries of length 1, a product
back, then ``gated_feed_forward`` and a product back; both results go through
``dropout``, which adds the block's input.  Answers are drawn one token a call from
the blocks' states.  The text is synthetic: pairs of a name and a number, of
which some come again, so that what follows a name a second time is known from
the first.
"""
from __future__ import annotations

import numpy as np

import macmetalpy_amd as cp
from macmetalpy_amd import nn

__all__ = ["DeltaLM", "paired_text"]


def paired_text(rng, batch, pairs, names, numbers):
    """(batch, 2 * pairs) tokens: names from 0 on, each followed by a number from
    ``names`` on, the same one in all of a sequence."""
    of = rng.integers(0, numbers, (batch, names))
    name = rng.integers(0, names, (batch, pairs))
    number = np.take_along_axis(of, name, 1) + names
    return np.stack([name, number], 2).reshape(batch, 2 * pairs).astype(np.int32)


def _unit(x):
    """x / |x| along the last axis, and 1 / |x|."""
    by = 1.0 / cp.sqrt(cp.sum(x * x, axis=-1, keepdims=True) + 1e-12)
    return x * by, by


def _unit_grad(grad, unit, by):
    return (grad - unit * cp.sum(grad * unit, axis=-1, keepdims=True)) * by


class DeltaLM:
    def __init__(self, classes, dim, layers=2, heads=2, dk=16, dv=16, hidden=64, rate=0.1, seed=0,
                 dtype=np.float32):
        g = np.random.default_rng(seed)

        def weight(*shape):
            return cp.array((g.standard_normal(shape) / shape[0] ** 0.5).astype(dtype))

        self.classes, self.dim, self.layers = classes, dim, layers
        self.heads, self.dk, self.dv, self.rate, self.seed = heads, dk, dv, rate, seed
        self.scale = dim ** 0.5  # of the table's rows, when they are looked up
        self.drawn = 0           # words of the dropout's stream used by now
        self.weights = [cp.array((g.standard_normal((classes, dim)) / dim ** 0.5).astype(dtype))]
        for _ in range(layers):
            self.weights += [weight(dim, heads * (2 * dk + dv + 2)), weight(heads * dv, dim),
                             weight(dim, 2 * hidden), weight(hidden, dim)]
        self.weights.append(weight(dim, classes))

    def _layer(self, i):
        return self.weights[1 + 4 * i:5 + 4 * i]

    def forward(self, tokens, states=None, train=False):
        """Logits (batch, steps, classes), the blocks' states after the last
        step, and what the gradients need."""
        batch, steps = tokens.shape
        h, dk, dv, d = self.heads, self.dk, self.dv, self.dim
        rate, at = self.rate if train else 0.0, self.drawn
        y = nn.embedding(self.weights[0], tokens, scale=self.scale).reshape((-1, d))
        kept, after = [], []
        for i in range(self.layers):
            into, back, ffn, down = self._layer(i)
            parts = (y @ into).reshape((batch, steps, -1))
            cut = np.cumsum([0, h * dk, h * dk, h * dv, h, h])
            q, k, v, a, b = (parts[..., cut[j]:cut[j + 1]] for j in range(5))
            q, q_by = _unit(q.reshape((batch, steps, h, dk)))
            k, k_by = _unit(k.reshape((batch, steps, h, dk)))
            v = v.reshape((batch, steps, h, dv))
            # the decay's logarithm is that of a sigmoid that starts near 1
            gate, beta = -cp.log1p(cp.exp(-a - 3.0)), 1.0 / (1.0 + cp.exp(-b))
            o, final = nn.gated_delta_rule(q, k, v, gate, beta,
                                           None if states is None else states[i], scale=1.0)
            mid = nn.dropout(o.reshape((-1, h * dv)) @ back, rate, self.seed, at, residual=y)
            wide = nn.gated_feed_forward(mid, ffn)
            kept.append((y, q, q_by, k, k_by, v, gate, beta, o, mid, wide, at))
            after.append(final)
            y = nn.dropout(wide @ down, rate, self.seed, at + y.size, residual=mid)
            at += 2 * y.size
        if train:
            self.drawn = at
        return (y @ self.weights[-1]).reshape((batch, steps, self.classes)), after, (kept, y)

    def gradients(self, tokens, targets):
        """The mean loss and the gradient of every weight.  Targets of -1 are
        not counted."""
        batch, steps = tokens.shape
        h, dk, dv = self.heads, self.dk, self.dv
        logits, _, (kept, y) = self.forward(tokens, train=True)
        count = max(1, int((np.asarray(targets) >= 0).sum()))
        loss, grad = nn.cross_entropy_grad(logits, cp.array(targets), 1.0 / count)
        grads = [None] * len(self.weights)
        grad = grad.reshape((-1, self.classes))
        grads[-1] = y.T @ grad
        grad = grad @ self.weights[-1].T
        for i in reversed(range(self.layers)):
            into, back, ffn, down = self._layer(i)
            y, q, q_by, k, k_by, v, gate, beta, o, mid, wide, at = kept[i]
            own = nn.dropout(grad, self.rate, self.seed, at + y.size)
            g_down = wide.T @ own
            own, g_ffn = nn.gated_feed_forward_grad(own @ down.T, mid, ffn)
            grad = grad + own
            own = nn.dropout(grad, self.rate, self.seed, at)
            g_back = o.reshape((-1, h * dv)).T @ own
            gq, gk, gv, g_gate, g_beta, _ = nn.gated_delta_rule_grad(
                (own @ back.T).reshape(o.shape), q, k, v, gate, beta, scale=1.0)
            # d gate / d a = 1 - exp(gate), d beta / d b = beta (1 - beta)
            parts = cp.concatenate([x.reshape((batch * steps, -1)) for x in (
                _unit_grad(gq, q, q_by), _unit_grad(gk, k, k_by), gv,
                g_gate * (1.0 - cp.exp(gate)), g_beta * beta * (1.0 - beta))], axis=1)
            grads[1 + 4 * i:5 + 4 * i] = [y.T @ parts, g_back, g_ffn, g_down]
            grad = grad + parts @ into.T
        grads[0] = nn.embedding_grad(grad.reshape((batch, steps, self.dim)), tokens, self.classes,
                                     scale=self.scale)
        return cp.sum(loss) / count, grads

    def train_step(self, text, rate=0.5, max_norm=1.0, targets=None):
        """One step of descent on (batch, steps + 1) tokens; the mean loss and
        the gradients' norm, as device arrays.  ``targets`` are the following
        tokens if None."""
        if targets is None:
            targets = text[:, 1:]
        tokens = cp.array(np.maximum(text[:, :-1], -1))
        loss, grads = self.gradients(tokens, np.ascontiguousarray(targets))
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


def main(train_steps=800, batch=64, pairs=24, names=8, numbers=8, dim=64):
    rng = np.random.default_rng(1)
    model = DeltaLM(names + numbers, dim)
    for step in range(train_steps):
        text = paired_text(rng, batch, pairs, names, numbers)
        targets = text[:, 1:].copy()
        targets[:, 1::2] = -1  # names are drawn: only numbers are learnt
        loss, norm = model.train_step(text, targets=targets)
        if step % 100 == 0 or step == train_steps - 1:
            print(f"step {step}: loss {float(loss):.4f}, gradient norm {float(norm):.3f}", flush=True)
    text = paired_text(rng, 200, pairs, names, numbers)
    known = (text[:, :-2:2] == text[:, -2:-1]).any(1)
    got = model.answer(text[:, :-1], 1)[:, 0]
    print(f"right after a name that came before: {np.mean(got[known] == text[known, -1]):.2f}")


if __name__ == "__main__":
    main()
