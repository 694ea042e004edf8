"""The operators of a training step, and of single tokens, of a recurrent
language model, as measurable cases.

Five kinds of pass: the embedding of tokens and its gradient, a gated linear
recurrence over sequences and its gradient, the softmax cross entropy of a
vocabulary with or without its gradient, and the clipping of many gradient
arrays by their global norm.  ``listed`` names twelve cases, ``draw`` gives
others of the same ranges.

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

_TORCH = {"float16": torch.float16, "float32": torch.float32, "int32": torch.int32,
          "int64": torch.int64}
_ITEM = {"float16": 2, "float32": 4, "int32": 4, "int64": 8}
_NUMPY = {torch.float16: np.float16, torch.float32: np.float32, torch.int32: np.int32,
          torch.int64: np.int64}


# ------------------------------------------------------------------ cases
def listed():
    return [
        # One new token for each of 200 sequences: the latency of a lookup.
        {"name": "embed_token", "kind": "embed", "tokens": 200, "rows": 32_000, "dim": 1024,
         "dtype": "float16", "index": "int64"},
        # A training batch's lookup: 64 sequences of 1024 tokens.
        {"name": "embed_batch", "kind": "embed", "tokens": 65_536, "rows": 50_021, "dim": 2048,
         "dtype": "float32", "index": "int32"},
        # The same batch's gradient in half precision, twice the tokens.
        {"name": "embed_grad_batch", "kind": "embed_grad", "tokens": 131_072, "rows": 64_000,
         "dim": 1024, "dtype": "float16", "index": "int64"},
        # Serving: one token of 200 sequences against their states.
        {"name": "recur_token", "kind": "recur", "batch": 200, "steps": 1, "dim": 2048,
         "dtype": "float16", "logits": True},
        # One long document: few channels, a long axis.
        {"name": "recur_long", "kind": "recur", "batch": 1, "steps": 65_536, "dim": 1024,
         "dtype": "float16", "logits": True},
        # A training batch's gradient.
        {"name": "recur_grad_batch", "kind": "recur_grad", "batch": 16, "steps": 2048, "dim": 2048,
         "dtype": "float16", "logits": True},
        # Sizes that no tile divides, single precision, decay factors that the
        # program computed itself.
        {"name": "recur_grad_ragged", "kind": "recur_grad", "batch": 3, "steps": 1999,
         "dim": 1001, "dtype": "float32", "logits": False},
        # A few rows of logits, as a last short batch has them.
        {"name": "loss_grad_few", "kind": "loss_grad", "rows": 50, "classes": 32_000,
         "dtype": "float16"},
        # The loss alone of held-out text, over an odd vocabulary.
        {"name": "loss_eval", "kind": "loss", "rows": 2047, "classes": 100_003,
         "dtype": "float32"},
        # A training batch's loss and gradient.
        {"name": "loss_grad_batch", "kind": "loss_grad", "rows": 16_384, "classes": 50_021,
         "dtype": "float16"},
        # The gradients of a small model: many little arrays of odd lengths.
        {"name": "clip_small", "kind": "clip", "arrays": 40, "total": 60_001, "dtype": "float32"},
        # The gradients of a large one.
        {"name": "clip_large", "kind": "clip", "arrays": 60, "total": 600_000_011,
         "dtype": "float16"},
    ]


def _log(rng, lo, hi):
    """An integer spread evenly over the logarithm of [lo, hi]."""
    return max(lo, min(hi, int(round(lo * (hi / lo) ** rng.random()))))


def draw(rng):
    kind = rng.choice(("embed", "embed_grad", "recur", "recur_grad", "loss", "loss_grad", "clip"))
    dtype = rng.choice(("float16", "float32"))
    if kind in ("embed", "embed_grad"):
        dim = _log(rng, 32, 4096)
        return {"kind": kind, "tokens": _log(rng, 1, 100_000_000 // dim),
                "rows": _log(rng, 100, 60_000_000 // dim), "dim": dim, "dtype": dtype,
                "index": rng.choice(("int32", "int64"))}
    if kind in ("recur", "recur_grad"):
        dim = _log(rng, 33, 4096)
        batch = _log(rng, 1, 300)
        # one in four is a single token or a short piece of text
        most = max(40, min(65_536, 60_000_000 // (dim * batch)))
        steps = _log(rng, 1, 32) if rng.random() < 0.25 else _log(rng, 32, most)
        return {"kind": kind, "batch": batch, "steps": steps, "dim": dim, "dtype": dtype,
                "logits": rng.random() < 0.7}
    if kind in ("loss", "loss_grad"):
        classes = _log(rng, 50, 260_000)
        return {"kind": kind, "rows": _log(rng, 1, min(60_000, 400_000_000 // classes)),
                "classes": classes, "dtype": dtype}
    arrays = rng.randint(1, 60)
    return {"kind": "clip", "arrays": arrays, "total": _log(rng, 100 * arrays, 300_000_000),
            "dtype": dtype}


# ----------------------------------------------------------------- inputs
def _lengths(arrays, total):
    """``arrays`` lengths from about total / 2 down to a few elements (the
    weights, biases and gains of a model), ``total`` in all."""
    part = [2.0 ** -(1 + 12 * i / max(arrays, 2)) for i in range(arrays)]
    n = [max(1, int(total * p / sum(part))) for p in part]
    n[0] += total - sum(n)
    return n


def _recurrence64(a, b, initial):
    """h_t = a_t h_{t-1} + b_t of (B, T, D) arrays, one step after another."""
    h = torch.empty_like(b)
    last = initial
    for t in range(b.shape[1]):
        last = torch.addcmul(b[:, t], a[:, t], last)
        h[:, t] = last
    return h


def _inputs(case, seed):
    """The case's inputs by name, as torch tensors on the GPU."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    kind, dt = case["kind"], _TORCH[case["dtype"]]

    def normal(*shape, dtype=dt, scale=1.0):
        return (torch.randn(*shape, generator=g, device="cuda") * scale).to(dtype)

    if kind in ("embed", "embed_grad"):
        n, v = case["tokens"], case["rows"]
        # Words' frequencies fall with their rank: uniform in the rank's logarithm.
        rank = torch.exp(torch.rand(n, generator=g, device="cuda") * math.log(v + 1.0)) - 1.0
        word = torch.randperm(v, generator=g, device="cuda")
        tokens = word[rank.long().clamp_(0, v - 1)]
        # Ragged sequences are filled up with -1.
        tokens[torch.rand(n, generator=g, device="cuda") < 0.02] = -1
        tokens = tokens.to(_TORCH[case["index"]])
        return ({"table": normal(v, case["dim"]), "tokens": tokens} if kind == "embed"
                else {"grad": normal(n, case["dim"]), "tokens": tokens})
    if kind in ("recur", "recur_grad"):
        shape = (case["batch"], case["steps"], case["dim"])
        # Gates that keep most of the state, each channel with a memory of its own.
        gate = torch.randn(*shape, generator=g, device="cuda") + torch.linspace(
            0.0, 6.0, shape[2], device="cuda")
        if not case["logits"]:
            gate = torch.sigmoid(gate)
        s = {"gate": gate.to(dt), "x": normal(*shape),
             "initial": normal(shape[0], shape[2], dtype=torch.float32)}
        if kind == "recur_grad":
            a, b = _factors(s["gate"], s["x"], case["logits"])
            s["h"] = _scan(a, _with_initial(a, b, s["initial"])).to(dt)
            s["grad"] = normal(*shape)
        return s
    if kind in ("loss", "loss_grad"):
        n, v = case["rows"], case["classes"]
        logits = torch.randn(n, v, generator=g, device="cuda").mul_(2.5)
        targets = torch.randint(0, v, (n,), generator=g, device="cuda")
        # A trained model gives the answer some weight; some rows are padding.
        logits[torch.arange(n, device="cuda"), targets] += 8.0
        targets[torch.rand(n, generator=g, device="cuda") < 0.02] = -1
        s = {"logits": logits.to(dt), "targets": targets}
        if kind == "loss_grad":
            # A mean's weights; half precision scales the loss, as its small
            # gradients would vanish.
            w = torch.rand(n, generator=g, device="cuda") + 0.5
            s["weight"] = w * ((65_536.0 if dt == torch.float16 else 1.0) / n)
        return s
    return {"g%02d" % i: normal(n, scale=0.05 / (1 + 0.1 * i))
            for i, n in enumerate(_lengths(case["arrays"], case["total"]))}


def prepare(case, seed):
    state = _inputs(case, seed)
    if own:
        # The same values in the arrays that a program on the library keeps.
        import macmetalpy_amd as cp
        arrays = {}
        for name, t in state.items():
            arrays[name] = cp.empty(tuple(t.shape), dtype=_NUMPY[t.dtype])
            arrays[name]._ensure_gpu()
        cp.synchronize()
        for name, t in state.items():
            _out(arrays[name]).copy_(t)
        torch.cuda.synchronize()
        state = arrays
    state["case"] = case
    return state


# ------------------------------------------------------- the plain forms
def _factors(gate, x, logits):
    """a and b of h_t = a_t h_{t-1} + b_t, in 32 bits."""
    gate, x = gate.float(), x.float()
    if not logits:
        return gate, x
    return torch.sigmoid(gate), torch.sigmoid(-gate) * x


def _with_initial(a, b, initial):
    b = b.clone()
    b[:, 0] += a[:, 0] * initial
    return b


def _scan(a, b):
    """h_t = a_t h_{t-1} + b_t over axis 1: neighbours are joined, half as
    many steps scanned, and the steps between filled in."""
    n = a.shape[1]
    if n == 1:
        return b
    a1 = a[:, 1::2]
    odd = _scan(a[:, 0:n - 1:2] * a1, a1 * b[:, 0:n - 1:2] + b[:, 1::2])
    h = torch.empty_like(b)
    h[:, 1::2] = odd
    h[:, :1] = b[:, :1]
    h[:, 2::2] = a[:, 2::2] * odd[:, :(n - 1) // 2] + b[:, 2::2]
    return h


def _plain(s):
    case = s["case"]
    kind, dt = case["kind"], _TORCH[case["dtype"]]
    if kind == "embed":
        tok = s["tokens"].long()
        rows = s["table"][tok.clamp(min=0)].float() * _scale(case)
        return torch.where((tok >= 0)[:, None], rows, 0.0).to(dt)
    if kind == "embed_grad":
        tok = s["tokens"].long()
        grad = torch.where((tok >= 0)[:, None], s["grad"].float(), 0.0)
        total = torch.zeros(case["rows"], case["dim"], device="cuda")
        return (total.index_add_(0, tok.clamp(min=0), grad) * _scale(case)).to(dt)
    if kind == "recur":
        a, b = _factors(s["gate"], s["x"], case["logits"])
        h = _scan(a, _with_initial(a, b, s["initial"]))
        return {"h": h.to(dt), "final": h[:, -1].clone()}
    if kind == "recur_grad":
        gate, x, h = s["gate"].float(), s["x"].float(), s["h"].float()
        before = torch.cat([s["initial"][:, None], h[:, :-1]], 1)
        a = torch.sigmoid(gate) if case["logits"] else gate
        # c_t = a_t c_{t+1} + a_t grad_t is the same scan from the last step on
        grad = s["grad"].float()
        c = _scan(a.flip(1), (a * grad).flip(1)).flip(1)
        d = grad.clone()
        d[:, :-1] += c[:, 1:]
        if case["logits"]:
            rest = torch.sigmoid(-gate)
            return {"gate": (d * (before - x) * a * rest).to(dt), "x": (d * rest).to(dt),
                    "initial": c[:, 0].clone()}
        return {"gate": (d * before).to(dt), "x": d.to(dt), "initial": c[:, 0].clone()}
    if kind in ("loss", "loss_grad"):
        x, t = s["logits"].float(), s["targets"]
        keep = t >= 0
        at = t.clamp(min=0)[:, None]
        x = x - x.amax(1, keepdim=True)
        e = x.exp()
        total = e.sum(1, keepdim=True)
        loss = torch.where(keep, (total.log() - x.gather(1, at))[:, 0], 0.0)
        if kind == "loss":
            return loss
        grad = e / total
        grad.scatter_add_(1, at, torch.full_like(total, -1.0))
        grad *= torch.where(keep, s["weight"], 0.0)[:, None]
        return {"loss": loss, "grad": grad.to(dt)}
    grads = [s[k] for k in sorted(s) if k != "case"]
    norm = torch.stack([(g.float() * g.float()).sum() for g in grads]).sum().sqrt()
    by = _max_norm(case) / torch.clamp(norm, min=_max_norm(case))
    return {"norm": norm, "clipped": [(g.float() * by).to(dt) for g in grads]}


def _max_norm(case):
    """A limit that these gradients pass, as in a step that needs one."""
    return 0.02 * float(case["total"]) ** 0.5


def _scale(case):
    """Embeddings are scaled by the square root of their width."""
    return float(case["dim"]) ** 0.5


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
    if not own:
        return _plain(state)
    from macmetalpy_amd import nn
    case = state["case"]
    kind = case["kind"]
    if kind == "embed":
        return _out(nn.embedding(state["table"], state["tokens"], scale=_scale(case)))
    if kind == "embed_grad":
        return _out(nn.embedding_grad(state["grad"], state["tokens"], case["rows"],
                                      scale=_scale(case)))
    if kind == "recur":
        h, final = nn.gated_recurrence(state["gate"], state["x"], state["initial"],
                                       logits=case["logits"])
        return {"h": _out(h), "final": _out(final)}
    if kind == "recur_grad":
        gate, x, initial = nn.gated_recurrence_grad(state["grad"], state["gate"], state["x"],
                                                    state["h"], state["initial"],
                                                    logits=case["logits"])
        return {"gate": _out(gate), "x": _out(x), "initial": _out(initial)}
    if kind == "loss":
        return _out(nn.cross_entropy(state["logits"], state["targets"]))
    if kind == "loss_grad":
        loss, grad = nn.cross_entropy_grad(state["logits"], state["targets"], state["weight"])
        return {"loss": _out(loss), "grad": _out(grad)}
    clipped, norm = nn.clip_by_global_norm([state[k] for k in sorted(state) if k != "case"],
                                           _max_norm(case))
    return {"norm": _out(norm), "clipped": [_out(g) for g in clipped]}


# -------------------------------------------------------- what a pass needs
def work(case):
    kind, s = case["kind"], _ITEM[case["dtype"]]
    if kind in ("embed", "embed_grad"):
        n, v, d = case["tokens"], case["rows"], case["dim"]
        index = n * _ITEM[case["index"]]
        if kind == "embed":  # at most every row of the table once
            return {"bytes": index + (n + min(n, v)) * d * s, "flops": n * d}
        return {"bytes": index + (n + v) * d * s, "flops": n * d}
    if kind in ("recur", "recur_grad"):
        n, state = case["batch"] * case["steps"] * case["dim"], case["batch"] * case["dim"] * 4
        if kind == "recur":
            return {"bytes": 3 * n * s + 2 * state, "flops": (8 if case["logits"] else 2) * n}
        return {"bytes": (6 if case["logits"] else 5) * n * s + 2 * state,
                "flops": (12 if case["logits"] else 4) * n}
    if kind in ("loss", "loss_grad"):
        n, v = case["rows"], case["classes"]
        if kind == "loss":
            return {"bytes": n * v * s + 12 * n, "flops": 4 * n * v}
        return {"bytes": 2 * n * v * s + 16 * n, "flops": 7 * n * v}
    return {"bytes": 2 * case["total"] * s + 4, "flops": 3 * case["total"]}


# ------------------------------------------------ the definitions in 64 bits
def exact(case, seed):
    s = _inputs(case, seed)
    kind = case["kind"]
    if kind in ("embed", "embed_grad"):
        tok, scale = s["tokens"].long(), math.sqrt(case["dim"])
        kept = torch.nonzero(tok >= 0)[:, 0]
        if kind == "embed":
            out = torch.zeros(case["tokens"], case["dim"], dtype=torch.float64, device="cuda")
            out[kept] = s["table"][tok[kept]].double() * scale
            return out
        out = torch.zeros(case["rows"], case["dim"], dtype=torch.float64, device="cuda")
        return out.index_put_((tok[kept],), s["grad"][kept].double() * scale, accumulate=True)
    if kind in ("recur", "recur_grad"):
        gate, x, initial = s["gate"].double(), s["x"].double(), s["initial"].double()
        f = 1.0 / (1.0 + torch.exp(-gate)) if case["logits"] else gate
        u = 1.0 / (1.0 + torch.exp(gate)) if case["logits"] else torch.ones_like(gate)
        if kind == "recur":
            h = _recurrence64(f, u * x, initial)
            return {"h": h, "final": h[:, -1]}
        d = torch.empty_like(x)
        c = torch.zeros_like(initial)
        for t in range(case["steps"] - 1, -1, -1):
            d[:, t] = s["grad"][:, t].double() + c
            c = f[:, t] * d[:, t]
        before = torch.cat([initial[:, None], s["h"][:, :-1].double()], 1)
        to_gate = (before - x) * f * u if case["logits"] else before
        return {"gate": d * to_gate, "x": d * u, "initial": c}
    if kind in ("loss", "loss_grad"):
        n, v = case["rows"], case["classes"]
        loss = torch.zeros(n, dtype=torch.float64, device="cuda")
        # gradients go as far as 32 bits hold them, to keep the memory in bounds
        grad = torch.zeros(n, v, device="cuda") if kind == "loss_grad" else None
        step = max(1, 100_000_000 // v)
        for i in range(0, n, step):
            x, t = s["logits"][i:i + step].double(), s["targets"][i:i + step]
            rows = torch.nonzero(t >= 0)[:, 0]
            lse = torch.logsumexp(x, 1)
            loss[i + rows] = lse[rows] - x[rows, t[rows]]
            if grad is not None:
                p = torch.exp(x - lse[:, None])
                p[rows, t[rows]] -= 1.0
                w = torch.zeros(len(t), dtype=torch.float64, device="cuda")
                w[rows] = s["weight"][i + rows].double()
                grad[i:i + step] = p * w[:, None]
        return loss if grad is None else {"loss": loss, "grad": grad}
    grads = [s[k].double() for k in sorted(s)]
    norm = torch.linalg.vector_norm(torch.cat(grads))
    most = _max_norm(case)
    return {"norm": norm, "clipped": [g * (most / max(float(norm), most)) for g in grads]}
