"""The operators of a block of a language model whose states are matrices, as
measurable cases: training steps and single tokens.

Three operators.  The gated delta rule, a recurrence whose state is a matrix
that keys write to and queries read from, and its gradient; the gated
feed-forward product (both projections, the activation and the product) and its
gradient; dropout by a counter-based generator, with or without the addition of
the block's input.  ``listed`` names twelve cases, ``draw`` gives others of the
same ranges.

``own`` says whose operators run: the library's (``macmetalpy_amd.nn`` on the
library's arrays), or their plain form, elementary torch operations in 32 bits
rounded once at the end.  The inputs' values are the same for both; a program
on the library holds them as the library's arrays, so that is what ``prepare``
puts them in when ``own`` is set.  Library results are returned as torch views
of the library's own memory, so that returning them copies nothing.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

_TORCH = {"float16": torch.float16, "float32": torch.float32}
_ITEM = {"float16": 2, "float32": 4}
_NUMPY = {torch.float16: np.float16, torch.float32: np.float32}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # Serving: one token of 48 sequences against their states.
        {"name": "delta_token", "kind": "delta", "batch": 48, "steps": 1, "key_heads": 8,
         "heads": 16, "dk": 128, "dv": 128, "dtype": "float16", "start": True, "packed": False},
        # A training batch of packed documents, keys and queries shared by two heads.
        {"name": "delta_batch", "kind": "delta", "batch": 8, "steps": 2048, "key_heads": 8,
         "heads": 16, "dk": 128, "dv": 128, "dtype": "float16", "start": False, "packed": True},
        # One long document is read on from a state.
        {"name": "delta_long", "kind": "delta", "batch": 1, "steps": 32_768, "key_heads": 8,
         "heads": 8, "dk": 128, "dv": 128, "dtype": "float16", "start": True, "packed": False},
        # A training batch's gradient.
        {"name": "delta_grad_batch", "kind": "delta_grad", "batch": 4, "steps": 2048,
         "key_heads": 8, "heads": 16, "dk": 128, "dv": 128, "dtype": "float16", "start": False,
         "packed": True},
        # Sizes that no tile divides, single precision, the last piece of a longer text.
        {"name": "delta_grad_ragged", "kind": "delta_grad", "batch": 3, "steps": 777,
         "key_heads": 5, "heads": 5, "dk": 72, "dv": 100, "dtype": "float32", "start": True,
         "packed": False},
        # Serving: a token of 8 sequences; the weights are what has to be read.
        {"name": "ffn_token", "kind": "ffn", "rows": 8, "dim": 2048, "hidden": 5632,
         "activation": "silu", "dtype": "float16"},
        # A short batch over widths that no vector divides.
        {"name": "ffn_ragged", "kind": "ffn", "rows": 1999, "dim": 1001, "hidden": 2503,
         "activation": "gelu", "dtype": "float16"},
        # A training batch, and its gradient.
        {"name": "ffn_batch", "kind": "ffn", "rows": 8192, "dim": 2048, "hidden": 5632,
         "activation": "silu", "dtype": "float16"},
        {"name": "ffn_grad_batch", "kind": "ffn_grad", "rows": 8192, "dim": 2048, "hidden": 5632,
         "activation": "silu", "dtype": "float16"},
        # The gradient of a small model in single precision.
        {"name": "ffn_grad_ragged", "kind": "ffn_grad", "rows": 515, "dim": 771, "hidden": 1030,
         "activation": "gelu", "dtype": "float32"},
        # Dropout of a few rows, where the latency of a call counts.
        {"name": "dropout_few", "kind": "dropout", "rows": 61, "dim": 1001, "rate": 0.1,
         "dtype": "float16", "residual": False},
        # A training batch's block output, dropped out and added to the block's input.
        {"name": "dropout_batch", "kind": "dropout", "rows": 65_536, "dim": 2048, "rate": 0.1,
         "dtype": "float16", "residual": True},
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("delta", "delta_grad", "ffn", "ffn_grad", "dropout"))
    dtype = rng.choice(("float16", "float32"))
    less = 1 if dtype == "float16" else 8
    if kind in ("delta", "delta_grad"):
        dk, dv = _log(rng, 16, 256), _log(rng, 16, 256)
        key_heads = _log(rng, 1, 12)
        heads = key_heads * rng.choice((1, 1, 2, 3))
        most = min(200_000 * (2 if kind == "delta" else 1),
                   3_000_000_000 // less // (dk * dv)) // heads
        batch = _log(rng, 1, min(64, most))
        # one in four is a single token or a short piece of text
        steps = _log(rng, 1, 16) if rng.random() < 0.25 else _log(rng, 16, 32_768)
        return {"kind": kind, "batch": batch, "steps": max(1, min(steps, most // batch)),
                "key_heads": key_heads, "heads": heads, "dk": dk, "dv": dv, "dtype": dtype,
                "start": rng.random() < 0.5, "packed": rng.random() < 0.5}
    if kind in ("ffn", "ffn_grad"):
        dim, hidden = _log(rng, 64, 4096), _log(rng, 64, 12_000)
        rows = _log(rng, 1, min(16_384, 90_000_000_000 // less // (dim * hidden)))
        return {"kind": kind, "rows": rows, "dim": dim, "hidden": hidden,
                "activation": rng.choice(("silu", "gelu", "sigmoid")), "dtype": dtype}
    dim = _log(rng, 33, 8192)
    return {"kind": kind, "rows": _log(rng, 1, 60_000_000 // dim), "dim": dim,
            "rate": rng.choice((0.05, 0.1, 0.2, 0.5)), "dtype": dtype,
            "residual": rng.random() < 0.5}


# ----------------------------------------------------------------- inputs
def _inputs(case, seed):
    """The case's inputs by name, as torch tensors on the GPU (numbers of the
    host for dropout's seed and offset)."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, dt = case["kind"], _TORCH[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if kind in ("delta", "delta_grad"):
        b, t, h, dk, dv = (case[k] for k in ("batch", "steps", "heads", "dk", "dv"))

        def unit(*shape):
            x = torch.randn(*shape, generator=g, device="cuda")
            return (x / x.square().sum(-1, keepdim=True).sqrt()).to(dt)

        s = {"q": unit(b, t, case["key_heads"], dk), "k": unit(b, t, case["key_heads"], dk),
             "v": normal(b, t, h, dv)}
        # Logarithms of decay factors, each head with a memory of its own: from
        # a few steps to thousands.
        rate = torch.exp(torch.linspace(math.log(1e-3), math.log(0.5), h, device="cuda"))
        gate = -rate * torch.log1p(torch.exp(torch.randn(b, t, h, generator=g, device="cuda")))
        beta = torch.sigmoid(torch.randn(b, t, h, generator=g, device="cuda"))
        if case["packed"]:
            # A document begins about every 500 steps: the state starts anew.
            new = torch.rand(b, t, 1, generator=g, device="cuda") < 0.002
            gate = torch.where(new, -math.inf, gate)
            # Every other sequence ends early: what fills it up leaves the state as it is.
            pad = torch.arange(t, device="cuda") >= t - t // 16
            pad = pad[None, :, None] & (torch.arange(b, device="cuda") % 2 == 1)[:, None, None]
            gate, beta = gate.masked_fill(pad, 0.0), beta.masked_fill(pad, 0.0)
        s["gate"], s["beta"] = gate.to(dt), beta.to(dt)
        if case["start"]:
            s["initial"] = normal(b, h, dk, dv, dtype=torch.float32, scale=0.3)
        if kind == "delta_grad":
            s["grad"] = normal(b, t, h, dv)
            if case["start"]:
                s["grad_final"] = normal(b, h, dk, dv, dtype=torch.float32, scale=0.3)
        return s
    if kind in ("ffn", "ffn_grad"):
        n, d, m = case["rows"], case["dim"], case["hidden"]
        s = {"x": normal(n, d), "weights": normal(d, 2 * m, scale=1.3 / d ** 0.5)}
        if kind == "ffn_grad":
            s["grad"] = normal(n, m)
        return s
    s = {"x": normal(case["rows"], case["dim"]), "seed": 1_000_003 * seed + 12_345,
         "offset": (seed % 977) * case["rows"] * case["dim"]}
    if case["residual"]:
        s["residual"] = normal(case["rows"], case["dim"])
    return s


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        # The same values in the arrays that a program on the library keeps.
        import macmetalpy_amd as cp
        arrays = {}
        for name, t in state.items():
            if isinstance(t, int):
                arrays[name] = t
                continue
            arrays[name] = cp.empty(tuple(t.shape), dtype=_NUMPY[t.dtype])
            arrays[name]._ensure_gpu()
        cp.synchronize()
        for name, t in state.items():
            if not isinstance(t, int):
                _out(arrays[name]).copy_(t)
        torch.cuda.synchronize()
        state = arrays
    state["case"] = case
    return state


# ------------------------------------------------------- the plain forms
# The delta rule of a head, with a state S (dk x dv):
#
#   S_t = a_t S_{t-1} + k_t u_t^T,  u_t = beta_t (v_t - a_t S_{t-1}^T k_t),  a_t = exp(gate_t)
#   o_t = scale S_t^T q_t
#
# In chunks of C steps, with the decay D_ij from step j to step i, c_i from
# before the chunk to step i and e_j from step j to the chunk's end:
#
#   (1 + A) U = R,  A_ij = beta_i D_ij k_i.k_j (j < i),  R = beta (V - c K S)
#   O = scale (c Q S + P U),  P_ij = D_ij q_i.k_j (j <= i)
#   S' = c_C S + (e K)^T U
_C = 64


def _chunks(x, steps):
    """(batch, steps, heads, ...) as (chunks, batch, heads, C, ...) in 32 bits, filled up with zeros."""
    n = -(-steps // _C)
    x = x.float()
    pad = x.new_zeros((x.shape[0], n * _C - steps) + tuple(x.shape[2:]))
    x = torch.cat([x, pad], 1).reshape((x.shape[0], n, _C) + tuple(x.shape[2:]))
    return x.movedim(3, 1).movedim(2, 0).contiguous()


def _unchunk(x, steps, dtype):
    """_chunks' inverse."""
    x = x.movedim(0, 2).movedim(1, 3)
    return x.reshape((x.shape[0], -1) + tuple(x.shape[3:]))[:, :steps].to(dtype).contiguous()


def _shared(x, heads):
    """(chunks, batch, key heads, C, dk) repeated for the heads that share a key head."""
    return x.repeat_interleave(heads // x.shape[2], 2)


def _inverse(a):
    """(1 + a)^-1 of strictly lower triangular a: (1 - a)(1 + a^2)(1 + a^4)..."""
    one = torch.eye(_C, device=a.device)
    inv, a = one - a, a @ a
    for _ in range(int(math.log2(_C)) - 1):
        inv, a = inv + inv @ a, a @ a
    return inv


def _delta_parts(s):
    """What the chunks need of the inputs alone."""
    case = s["case"]
    steps, heads = case["steps"], case["heads"]
    q, k = (_shared(_chunks(s[x], steps), heads) for x in "qk")
    v, gate, beta = (_chunks(s[x], steps) for x in ("v", "gate", "beta"))
    # A gate of -inf is counted apart: nothing passes it.
    anew = gate.isinf()
    count = anew.cumsum(-1)
    total = gate.masked_fill(anew, 0.0).double().cumsum(-1)
    lower = torch.ones(_C, _C, dtype=torch.bool, device=gate.device).tril()
    same = (count[..., :, None] == count[..., None, :]) & lower
    far = torch.where(same, total[..., :, None] - total[..., None, :], -math.inf)
    decay = far.float().exp()
    c = torch.where(count == 0, total, -math.inf).float().exp()
    e = torch.where(count == count[..., -1:], total[..., -1:] - total, -math.inf).float().exp()
    kk = decay.tril(-1) * (k @ k.mT)
    p = decay * (q @ k.mT)
    return q, k, v, beta, c, e, decay, kk, p, _inverse(beta[..., None] * kk)


def _scale(case):
    return case["dk"] ** -0.5


def _initial(s, name="initial"):
    case = s["case"]
    shape = (case["batch"], case["heads"], case["dk"], case["dv"])
    return s[name] if name in s else torch.zeros(shape, device="cuda")


def _delta_states(s, parts):
    """The state before each chunk and after the last, and each chunk's U."""
    q, k, v, beta, c, e, decay, kk, p, inv = parts
    states, us = [_initial(s)], []
    for i in range(len(q)):
        r = beta[i][..., None] * (v[i] - c[i][..., None] * (k[i] @ states[-1]))
        us.append(inv[i] @ r)
        states.append(c[i][..., -1:, None] * states[-1] + (e[i][..., None] * k[i]).mT @ us[-1])
    return torch.stack(states), torch.stack(us)


def _plain_delta(s):
    case, dt = s["case"], _TORCH[s["case"]["dtype"]]
    parts = _delta_parts(s)
    q, k, v, beta, c, e, decay, kk, p, inv = parts
    states, u = _delta_states(s, parts)
    o = _scale(case) * (c[..., None] * (q @ states[:-1]) + p @ u)
    return {"o": _unchunk(o, case["steps"], dt), "final": states[-1].clone()}


def _plain_delta_grad(s):
    case, dt = s["case"], _TORCH[s["case"]["dtype"]]
    steps, heads, shared = case["steps"], case["heads"], case["key_heads"]
    parts = _delta_parts(s)
    q, k, v, beta, c, e, decay, kk, p, inv = parts
    states, u = _delta_states(s, parts)
    before = states[:-1]
    go = _chunks(s["grad"], steps) * _scale(case)
    b_, c_, e_ = beta[..., None], c[..., None], e[..., None]
    local = p.mT @ go
    grad, after, dr = _initial(s, "grad_final"), [], []
    for i in reversed(range(len(q))):
        after.append(grad)
        dr.append(inv[i].mT @ (local[i] + (e_[i] * k[i]) @ grad))
        grad = c_[i][..., -1:, :] * grad + (c_[i] * q[i]).mT @ go[i] \
            - (b_[i] * c_[i] * k[i]).mT @ dr[-1]
    after, dr = torch.stack(after[::-1]), torch.stack(dr[::-1])
    dp = (go @ u.mT).tril()
    da = -(dr @ u.mT).tril(-1)
    # to the products of keys and queries, through the decays
    to_p, to_a = dp * decay, b_ * da * decay
    q_state = c_ * (go @ before.mT)
    k_state = -c_ * (dr @ before.mT)
    k_after = e_ * (u @ after.mT)
    dq = q_state + to_p @ k
    dk = b_ * k_state + k_after + to_p.mT @ q + (to_a + to_a.mT) @ k
    dbeta = (dr * v).sum(-1) + (k * k_state).sum(-1) + (da * kk).sum(-1)
    m = dp * p + b_ * da * kk
    w = (k * k_after).sum(-1)
    dg = (q * q_state).sum(-1) + beta * (k * k_state).sum(-1) - w + m.sum(-1) - m.sum(-2)
    dg[..., -1] += w.sum(-1) + c[..., -1] * (before * after).sum((-1, -2))
    dg = dg.flip(-1).cumsum(-1).flip(-1)  # every later step's logarithm holds this one's
    dg = torch.where(_chunks(s["gate"], steps).isinf(), 0.0, dg)

    def heads_joined(x):
        x = x.reshape(x.shape[:2] + (shared, heads // shared) + x.shape[3:]).sum(3)
        return _unchunk(x, steps, dt)

    return {"q": heads_joined(dq), "k": heads_joined(dk), "v": _unchunk(b_ * dr, steps, dt),
            "gate": _unchunk(dg, steps, dt), "beta": _unchunk(dbeta, steps, dt),
            "initial": grad.clone()}


def _activation(name, g):
    """The activation and its derivative."""
    if name == "gelu":
        phi = 0.5 * (1.0 + torch.erf(g * 0.5 ** 0.5))
        return g * phi, phi + g * torch.exp(-0.5 * g * g) * (0.5 / math.pi) ** 0.5
    f = torch.sigmoid(g)
    rest = torch.sigmoid(-g)
    return (g * f, f * (1.0 + g * rest)) if name == "silu" else (f, f * rest)


def _plain_ffn(s):
    case, dt = s["case"], _TORCH[s["case"]["dtype"]]
    x, w, m = s["x"].float(), s["weights"].float(), case["hidden"]
    both = x @ w
    a, da = _activation(case["activation"], both[:, :m])
    if case["kind"] == "ffn":
        return (a * both[:, m:]).to(dt)
    grad = s["grad"].float()
    both = torch.cat([grad * both[:, m:] * da, grad * a], 1)
    return {"x": (both @ w.T).to(dt), "weights": (x.T @ both).to(dt)}


_M = 0xFFFFFFFF


def _random_words(first, count, seed):
    """Words first .. first + count of the stream that ``seed`` names, of
    Philox4x32-10 (Salmon, Moraes, Dror, Shaw 2011): block i holds words 4 i to
    4 i + 3, its counter is (i, 0) and its key the seed, 64 bits each."""
    block = torch.arange(first // 4, (first + count + 3) // 4, device="cuda")
    c = [block & _M, block >> 32 & _M, torch.zeros_like(block), torch.zeros_like(block)]
    key = [seed & _M, seed >> 32 & _M]
    for _ in range(10):
        a, b = c[0] * 0xD2511F53, c[2] * 0xCD9E8D57
        c = [b >> 32 & _M ^ c[1] ^ key[0], b & _M, a >> 32 & _M ^ c[3] ^ key[1], a & _M]
        key = [key[0] + 0x9E3779B9 & _M, key[1] + 0xBB67AE85 & _M]
    return torch.stack(c, 1).reshape(-1)[first % 4:][:count]


def _plain_dropout(s):
    case, dt = s["case"], _TORCH[s["case"]["dtype"]]
    x = s["x"].float()
    word = _random_words(s["offset"], x.numel(), s["seed"]).reshape(x.shape)
    y = torch.where(word >= round(case["rate"] * 2 ** 32), x * (1.0 / (1.0 - case["rate"])), 0.0)
    return (y + s["residual"].float() if case["residual"] else y).to(dt)


_PLAIN = {"delta": _plain_delta, "delta_grad": _plain_delta_grad, "ffn": _plain_ffn,
          "ffn_grad": _plain_ffn, "dropout": _plain_dropout}


# ------------------------------------------------------------------ a pass
class _View:
    """A device array as torch.as_tensor reads one; it keeps the array alive."""

    __slots__ = ("array", "__cuda_array_interface__")

    def __init__(self, a):
        self.array = a
        self.__cuda_array_interface__ = {"shape": a.shape, "typestr": a.dtype.str, "strides": None,
                                         "data": (a._ptr, False), "version": 2}


def _out(a):
    return torch.as_tensor(_View(a), device="cuda")


def run(state):
    case = state["case"]
    kind = case["kind"]
    if not own:
        return _PLAIN[kind](state)
    from macmetalpy_amd import nn
    s = state
    if kind == "delta":
        o, final = nn.gated_delta_rule(s["q"], s["k"], s["v"], s["gate"], s["beta"],
                                       s.get("initial"))
        return {"o": _out(o), "final": _out(final)}
    if kind == "delta_grad":
        grads = nn.gated_delta_rule_grad(s["grad"], s["q"], s["k"], s["v"], s["gate"], s["beta"],
                                         s.get("initial"), s.get("grad_final"))
        return dict(zip(("q", "k", "v", "gate", "beta", "initial"), map(_out, grads)))
    if kind == "ffn":
        return _out(nn.gated_feed_forward(s["x"], s["weights"], case["activation"]))
    if kind == "ffn_grad":
        grads = nn.gated_feed_forward_grad(s["grad"], s["x"], s["weights"], case["activation"])
        return {"x": _out(grads[0]), "weights": _out(grads[1])}
    return _out(nn.dropout(s["x"], case["rate"], s["seed"], s["offset"], s.get("residual")))


# -------------------------------------------------------- what a pass needs
def work(case):
    kind, z = case["kind"], _ITEM[case["dtype"]]
    if kind in ("delta", "delta_grad"):
        n = case["batch"] * case["steps"]
        qk = 2 * n * case["key_heads"] * case["dk"] * z
        v, gates = n * case["heads"] * case["dv"] * z, 2 * n * case["heads"] * z
        size = case["batch"] * case["heads"] * case["dk"] * case["dv"]
        state = size * 4 * (2 if case["start"] else 1)
        # a step decays the state and multiplies it with a key, a query and its change
        if kind == "delta":
            return {"bytes": qk + 2 * v + gates + state, "flops": 7 * size * case["steps"]}
        # the gradient works the states out and goes through them backwards:
        # five such products more
        state = size * 4 * (3 if case["start"] else 1)
        return {"bytes": 2 * qk + 3 * v + 2 * gates + state, "flops": 18 * size * case["steps"]}
    if kind in ("ffn", "ffn_grad"):
        n, d, m = case["rows"], case["dim"], case["hidden"]
        if kind == "ffn":
            return {"bytes": (n * d + 2 * d * m + n * m) * z, "flops": 4 * n * d * m}
        return {"bytes": (2 * n * d + 4 * d * m + n * m) * z, "flops": 12 * n * d * m}
    n = case["rows"] * case["dim"]
    return {"bytes": n * z * (3 if case["residual"] else 2), "flops": 2 * n}


# ------------------------------------------------ the definitions in 64 bits
def _exact_delta(s, case):
    """Step after step, as the operator is defined; the gradient by the chain
    rule of one step, from states kept every so often."""
    steps, heads, shared = case["steps"], case["heads"], case["key_heads"]
    group = heads // shared

    def at(x, t):  # (batch, heads, ...) of step t
        x = x[:, t].double()
        return x.repeat_interleave(group, 1) if x.shape[1] != heads else x

    def step(state, t):
        a, k = at(s["gate"], t).exp()[..., None, None], at(s["k"], t)
        faded = torch.where(a == 0.0, 0.0, a * state)
        miss = at(s["v"], t) - (k[..., None] * faded).sum(-2)
        u = at(s["beta"], t)[..., None] * miss
        return faded + k[..., None] * u[..., None, :], faded, miss, u

    state = _initial({**s, "case": case}).double()
    if case["kind"] == "delta":
        o = torch.empty(s["v"].shape, dtype=torch.float64, device="cuda")
        for t in range(steps):
            state = step(state, t)[0]
            o[:, t] = _scale(case) * (at(s["q"], t)[..., None] * state).sum(-2)
        return {"o": o, "final": state}
    every = max(1, int(steps ** 0.5))
    kept = []
    for t in range(steps):
        if t % every == 0:
            kept.append(state)
        state = step(state, t)[0]
    grad = _initial({**s, "case": case}, "grad_final").double()
    out = {n: torch.zeros(s[n].shape, dtype=torch.float64, device="cuda")
           for n in ("q", "k", "v", "gate", "beta")}

    def joined(x):
        return x.reshape(x.shape[0], shared, group, x.shape[2]).sum(2)

    for first in range((steps - 1) // every * every, -1, -every):
        state, seen = kept.pop(), []
        for t in range(first, min(first + every, steps)):
            seen.append((state,) + step(state, t))
            state = seen[-1][1]
        for t in range(first + len(seen) - 1, first - 1, -1):
            old, new, faded, miss, u = seen.pop()
            q, k, go = at(s["q"], t), at(s["k"], t), at(s["grad"], t) * _scale(case)
            beta = at(s["beta"], t)[..., None]
            out["q"][:, t] = joined((new * go[..., None, :]).sum(-1))
            grad = grad + q[..., None] * go[..., None, :]
            du = (grad * k[..., None]).sum(-2)
            dm = beta * du
            out["beta"][:, t] = (du * miss).sum(-1)
            out["v"][:, t] = dm
            out["k"][:, t] = joined((grad * u[..., None, :]).sum(-1)
                                    - (faded * dm[..., None, :]).sum(-1))
            grad = grad - k[..., None] * dm[..., None, :]
            out["gate"][:, t] = (grad * faded).sum((-1, -2))
            a = at(s["gate"], t).exp()[..., None, None]
            grad = torch.where(a == 0.0, 0.0, a * grad)
    return {**out, "initial": grad}


def _exact_words(first, count, seed):
    """_random_words on the host, the 64 bit products as they are."""
    low = np.uint64(0xFFFFFFFF)
    half = np.uint64(32)
    got = np.empty((first % 4 + count + 3) // 4 * 4, dtype=np.uint32).reshape(-1, 4)
    for i in range(0, len(got), 1 << 20):
        block = np.arange(first // 4 + i, first // 4 + min(i + (1 << 20), len(got)),
                          dtype=np.uint64)
        x0, x1, x2, x3 = block & low, block >> half, 0 * block, 0 * block
        for r in range(10):
            k0 = np.uint64((seed % 2 ** 32 + r * 0x9E3779B9) % 2 ** 32)
            k1 = np.uint64((seed // 2 ** 32 % 2 ** 32 + r * 0xBB67AE85) % 2 ** 32)
            p, t = np.uint64(0xD2511F53) * x0, np.uint64(0xCD9E8D57) * x2
            x0, x1, x2, x3 = (t >> half) ^ x1 ^ k0, t & low, (p >> half) ^ x3 ^ k1, p & low
        got[i:i + len(block)] = np.stack([x0, x1, x2, x3], 1)
    return got.reshape(-1)[first % 4:first % 4 + count]


def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind in ("delta", "delta_grad"):
        return _exact_delta(s, case)
    if kind in ("ffn", "ffn_grad"):
        x, w, m = s["x"].double(), s["weights"].double(), case["hidden"]
        gate, up = x @ w[:, :m].contiguous(), x @ w[:, m:].contiguous()
        name = case["activation"]
        if name in ("silu", "sigmoid"):
            f = 1.0 / (1.0 + torch.exp(-gate))
            a = gate * f if name == "silu" else f
            da = f + a * (1.0 - f) if name == "silu" else f * (1.0 - f)
        else:
            da = 0.5 * torch.special.erfc(-gate / math.sqrt(2.0))
            a = gate * da
            da = da + gate * torch.exp(-gate * gate / 2.0) / math.sqrt(2.0 * math.pi)
        if kind == "ffn":
            return a * up
        grad = s["grad"].double()
        gate, up = grad * up * da, grad * a
        xt = x.T.contiguous()
        return {"x": gate @ w[:, :m].T.contiguous() + up @ w[:, m:].T.contiguous(),
                "weights": torch.cat([xt @ gate, xt @ up], 1)}
    words = torch.from_numpy(_exact_words(s["offset"], s["x"].numel(), s["seed"]).astype(np.int64))
    keep = (words.cuda() >= round(case["rate"] * 2 ** 32)).reshape(s["x"].shape)
    y = torch.where(keep, s["x"].double() / (1.0 - case["rate"]), 0.0)
    return y + s["residual"].double() if case["residual"] else y
