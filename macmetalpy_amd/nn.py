"""``cp.nn``: the operators of sequence models, with their gradients.

Embedding rows by tokens, a gated linear recurrence, the softmax cross
entropy and the clipping of gradients by their global norm: with ``matmul``
the parts of a training step of a recurrent language model, and, one step at a
time, of its answers (``python -m macmetalpy_amd.recurrent_lm`` runs both).
The reference has none of them.  Each is one call on device arrays, most of
which read their inputs once (the norm's limit needs a second pass over the
arrays, and so does the gradient of a loss for rows too long for a workgroup's
registers, or few and cut into parts); nothing is recorded or differentiated
automatically, a gradient is a call of its own.

float16, float32 and float64; sums, states and softmax statistics are held in
float32 (float64 for float64), and results are rounded to the inputs' type
once.  Nothing waits for the device: tokens and targets out of range are not
errors but no tokens (zeros, no gradient), so batches can be filled up with
-1.  (``scale`` and ``max_norm`` are numbers of the host: one that is on the device
is read, which waits.)  A call repeated gives the same bits, nothing depends on
timing; losses and norms of the same values at another address modulo 16 may be
added in another order.
"""
from __future__ import annotations

import math

import numpy as np

from . import _elementwise as ew
from ._abi import DTYPE_CODES as _CODE
from ._backend import HipBackend
from ._native import empty as _empty
from .manipulation import broadcast_to
from .ndarray import ndarray, _c_contiguous_strides, _prod

__all__ = ["embedding", "embedding_grad", "gated_recurrence", "gated_recurrence_grad",
           "cross_entropy", "cross_entropy_grad", "global_norm", "clip_by_global_norm"]

_F32, _F64, _I32, _I64 = (np.dtype(t) for t in (np.float32, np.float64, np.int32, np.int64))
_FLOATS = frozenset((np.dtype(np.float16), _F32, _F64))
# The type that sums and states are held in.
_WIDE = {dt: _F64 if dt == _F64 else _F32 for dt in _FLOATS}


def _device(a) -> ndarray:
    if type(a) is ndarray:
        if a._fusion_node is None and a._np_data is None:
            return a
    elif not isinstance(a, ndarray):
        from .creation import asarray
        a = asarray(a)
    return a._ensure_gpu()


def _floating(a, what) -> ndarray:
    a = _device(a)
    if a._dtype not in _FLOATS:
        raise TypeError(f"{what} must be floating, not {a._dtype}")
    return a


def _contiguous(a, dtype) -> ndarray:
    if a._dtype != dtype:
        return a._contiguous_copy(dtype)
    return a if a._strides == _c_contiguous_strides(a._shape) else a._contiguous_copy()


def _integers(a, what) -> ndarray:
    """Contiguous int32 or int64 indices."""
    a = _device(a)
    dtype = a._dtype
    if dtype.kind not in "iu":
        raise TypeError(f"{what} must be integers, not {dtype}")
    return _contiguous(a, dtype if dtype == _I32 or dtype == _I64 else _I64)


def _collapsed(a, axes):
    """The one stride that steps through the first ``axes`` axes of ``a`` in
    order, or None if there is none."""
    stride, size = 0, 1
    for n, s in zip(reversed(a._shape[:axes]), reversed(a._strides[:axes])):
        if n == 1:
            continue
        if size == 1:
            stride = s
        elif s != stride * size:
            return None
        size *= n
    return stride


def _rows(a):
    """(array, row stride) of ``a`` as rows of adjacent elements: ``a`` itself
    where its strides allow it, else a contiguous copy."""
    shape, strides = a._shape, a._strides
    if strides != _c_contiguous_strides(shape):
        if shape[-1] <= 1 or strides[-1] == 1:
            stride = _collapsed(a, len(shape) - 1)
            if stride is not None:
                return a, stride
        a = a._contiguous_copy()
    return a, shape[-1]


def _steps(a):
    """(array, (pointer, sequence stride, step stride)) of a (..., steps,
    channels) array with adjacent channels, ``a`` itself where possible."""
    shape, strides = a._shape, a._strides
    if strides != _c_contiguous_strides(shape):
        if shape[-1] <= 1 or strides[-1] == 1:
            stride = _collapsed(a, len(shape) - 2)
            if stride is not None:
                return a, (a._ptr, stride, strides[-2])
        a = a._contiguous_copy()
    return a, (a._ptr, shape[-2] * shape[-1], shape[-1])


def _scalar(v, what) -> float:
    try:
        if not isinstance(v, (str, bytes, bytearray)):  # float() reads those too
            return float(v)
    except (TypeError, ValueError):
        pass
    raise TypeError(f"{what} must be a number, not {type(v).__name__}")


# ------------------------------------------------------------- embedding
def embedding(table, tokens, scale=1.0) -> ndarray:
    """``scale * table[tokens]``: the rows of a (rows, dim) table, of shape
    ``tokens.shape + (dim,)`` and the table's type.  A token outside
    ``[0, rows)`` gives a row of zeros."""
    table, tokens = _floating(table, "table"), _integers(tokens, "tokens")
    if table.ndim != 2:
        raise ValueError(f"table must have two axes, not {table.ndim}")
    scale = _scalar(scale, "scale")
    rows, dim = table._shape
    table, stride = _rows(table)
    out = _empty(tokens._shape + (dim,), table._dtype)
    n = tokens.size
    if n and dim:
        HipBackend().embedding(_CODE[table._dtype], _CODE[tokens._dtype], n, tokens._ptr,
                               rows, dim, table._ptr, stride, scale, out._ptr)
    return out


def embedding_grad(grad, tokens, rows, scale=1.0) -> ndarray:
    """The gradient of :func:`embedding` with respect to its (rows, dim)
    table, whole: row v is ``scale`` times the sum of ``grad`` over the tokens
    equal to v, added in an order that the tokens, the width and the type decide.
    ``grad`` has shape ``tokens.shape + (dim,)`` and gives the type."""
    grad, tokens = _floating(grad, "grad"), _integers(tokens, "tokens")
    if grad.ndim == 0 or grad._shape[:-1] != tokens._shape:
        raise ValueError(f"grad of shape {grad._shape} does not fit tokens of shape "
                         f"{tokens._shape}: expected {tokens._shape} and the table's width")
    if not isinstance(rows, (int, np.integer)) or isinstance(rows, bool):
        raise TypeError(f"rows must be an integer, not {type(rows).__name__}")
    rows = int(rows)
    if rows < 0:
        raise ValueError(f"rows must not be negative: {rows}")
    scale = _scalar(scale, "scale")
    dim = grad._shape[-1]
    grad, stride = _rows(grad)
    out = _empty((rows, dim), grad._dtype)
    if rows and dim:
        HipBackend().embedding_grad(_CODE[grad._dtype], _CODE[tokens._dtype],
                                    tokens.size, tokens._ptr, grad._ptr, stride, rows, dim, scale,
                                    out._ptr)
    return out


# ------------------------------------------------------------ recurrence
def _sequences(named):
    """Floating arrays of one shape (..., steps, channels), in one type."""
    arrays = [_floating(a, name) for name, a in named]
    first = arrays[0]
    for (name, _), a in zip(named, arrays):
        if a.ndim < 2:
            raise ValueError(f"{name} must have axes for steps and channels: shape {a._shape}")
        if a._shape != first._shape:
            raise ValueError(f"{name} of shape {a._shape} does not match {named[0][0]} of shape "
                             f"{first._shape}")
    dtype = first._dtype
    if any(a._dtype != dtype for a in arrays):
        dtype = np.result_type(*(a._dtype for a in arrays))
        arrays = [_contiguous(a, dtype) for a in arrays]
    return arrays, dtype


def _state(a, shape, dtype, name):
    """A state (..., channels) of ``shape`` as a contiguous array, or None."""
    if a is None:
        return None
    a = _floating(a, name)
    if a._shape != shape:
        raise ValueError(f"{name} of shape {a._shape}: expected {shape}")
    return _contiguous(a, dtype)


def _ptr(a):
    return None if a is None else a._ptr


def gated_recurrence(gate, x, initial=None, *, logits=True):
    """``(h, final)`` of a linear recurrence along the last axis but one of
    (..., steps, channels) arrays, each channel by itself::

        logits=True   f = 1 / (1 + exp(-gate)),  h_t = f_t h_{t-1} + (1 - f_t) x_t
        logits=False                             h_t = gate_t h_{t-1} + x_t

    ``initial`` is the state before the first step (..., channels), zeros if
    None; ``final`` the state after the last, in float32 (float64 for float64)
    and not rounded to the type of ``h``, to go on from: one new token a call
    is ``steps == 1``.  A gate of ``-inf`` (a factor of 0) starts a channel
    anew from any finite state.  Factors are multiplied up along many steps,
    so the products of neighbouring ones have to stay in the type's range: use
    ones of at most 1 in size.  A state that has become infinite may go on as
    NaN, where such a product has become 0."""
    (gate, x), dtype = _sequences((("gate", gate), ("x", x)))
    steps, dim = x._shape[-2:]
    wide = _WIDE[dtype]
    state_shape = x._shape[:-2] + (dim,)
    initial = _state(initial, state_shape, wide, "initial")
    h = _empty(x._shape, dtype)
    final = _empty(state_shape, wide)
    if final.size:
        gate, at_gate = _steps(gate)
        x, at_x = _steps(x)
        HipBackend().recurrence(_CODE[dtype], 1 if logits else 0, _prod(x._shape[:-2]), steps,
                                dim, at_gate, at_x, _ptr(initial), h._ptr, final._ptr)
    return h, final


def gated_recurrence_grad(grad, gate, x, h, initial=None, grad_final=None, *, logits=True):
    """``(grad_gate, grad_x, grad_initial)`` of :func:`gated_recurrence`, from
    ``grad`` (of ``h``), its inputs, the ``h`` that it returned and, where
    the final state was used too, ``grad_final``.  The gradients of gate and x
    have the sequences' type, ``grad_initial`` the states'."""
    (grad, gate, x, h), dtype = _sequences((("grad", grad), ("gate", gate), ("x", x), ("h", h)))
    steps, dim = x._shape[-2:]
    wide = _WIDE[dtype]
    state_shape = x._shape[:-2] + (dim,)
    initial = _state(initial, state_shape, wide, "initial")
    grad_final = _state(grad_final, state_shape, wide, "grad_final")
    grad_gate = _empty(x._shape, dtype)
    grad_x = _empty(x._shape, dtype)
    grad_initial = _empty(state_shape, wide)
    if grad_initial.size:
        grad, at_grad = _steps(grad)
        gate, at_gate = _steps(gate)
        x, at_x = _steps(x)
        h, at_h = _steps(h)
        HipBackend().recurrence_grad(_CODE[dtype], 1 if logits else 0, _prod(x._shape[:-2]),
                                     steps, dim, at_grad, at_gate, at_x, at_h, _ptr(initial),
                                     _ptr(grad_final), grad_gate._ptr, grad_x._ptr,
                                     grad_initial._ptr)
    return grad_gate, grad_x, grad_initial


# ------------------------------------------------------------------ loss
def _loss(logits, targets, weight, want_grad):
    logits, targets = _floating(logits, "logits"), _integers(targets, "targets")
    if logits.ndim == 0 or logits._shape[:-1] != targets._shape:
        raise ValueError(f"logits of shape {logits._shape} do not fit targets of shape "
                         f"{targets._shape}: expected {targets._shape} and the classes")
    classes, dtype = logits._shape[-1], logits._dtype
    if classes == 0:
        raise ValueError("logits have no classes")
    wide, scale, each = _WIDE[dtype], 1.0, None
    if isinstance(weight, ndarray) and weight.ndim == 0:
        # one number on the device, for every row: reading it here would wait
        each = _contiguous(broadcast_to(_device(weight), targets._shape), wide)
    elif isinstance(weight, (ndarray, np.ndarray)) and weight.ndim:
        each = _floating(weight, "weight")
        if each._shape != targets._shape:
            raise ValueError(f"weight of shape {each._shape}: expected a number or "
                             f"{targets._shape}")
        each = _contiguous(each, wide)
    else:
        scale = _scalar(weight, "weight")
    loss = _empty(targets._shape, wide)
    grad = _empty(logits._shape, dtype) if want_grad else None
    n = targets.size
    if n:
        logits, stride = _rows(logits)
        HipBackend().cross_entropy(_CODE[dtype], _CODE[targets._dtype], n, classes,
                                   logits._ptr, stride, targets._ptr, _ptr(each), scale, loss._ptr,
                                   _ptr(grad))
    return loss, grad


def cross_entropy(logits, targets) -> ndarray:
    """``log(sum(exp(x))) - x[target]`` of each row of (..., classes) logits,
    in float32 (float64 for float64).  A target outside ``[0, classes)`` gives
    0.  A logit of ``-inf`` is a class that cannot be; a row with nothing else,
    or with a logit of ``+inf``, gives NaN."""
    return _loss(logits, targets, 1.0, False)[0]


def cross_entropy_grad(logits, targets, weight=1.0):
    """``(loss, grad)``: the losses of :func:`cross_entropy`, and the gradient
    of ``sum(weight * loss)`` with respect to the logits, in their type.
    ``weight`` is a number (``1 / n`` for a mean, times the factor by which
    float16 training scales its loss), also as a device array of no axes, or
    one for each target."""
    return _loss(logits, targets, weight, True)


# ------------------------------------------------------------------ norm
def _clip(arrays, limit, out):
    given, codes, sizes, ptrs, outs = [], [], [], [], None
    for a in arrays:
        a = _floating(a, "every array")
        shape, dtype = a._shape, a._dtype
        if a._strides != _c_contiguous_strides(shape):
            a = a._contiguous_copy()
        given.append(a)
        codes.append(_CODE[dtype])
        sizes.append(_prod(shape))
        ptrs.append(a._buffer.ptr + a._offset * dtype.itemsize)
    wide = _F64 if _CODE[_F64] in codes else _F32
    norm = _empty((), wide)
    if limit is None:
        limit, out_ptrs = 0.0, None
    elif out is None:
        outs = [_empty(a._shape, a._dtype) for a in given]
        out_ptrs = [o._buffer.ptr for o in outs]
    else:
        outs = list(out)
        if len(outs) != len(given):
            raise ValueError(f"out has {len(outs)} arrays for {len(given)}")
        for a, o in zip(given, outs):
            if not isinstance(o, ndarray):
                raise TypeError(f"out must hold device arrays, not {type(o).__name__}")
            if o._shape != a._shape or o._dtype != a._dtype:
                raise ValueError(f"out of shape {o._shape} and type {o._dtype} for an array of "
                                 f"shape {a._shape} and type {a._dtype}")
            o._ensure_gpu()
            if not o._is_c_contiguous():
                raise ValueError("out must be contiguous")
            ew.flush_lazy(o._buffer)
        out_ptrs = [o._ptr for o in outs]
    HipBackend().clip_norm(codes, sizes, ptrs, out_ptrs, limit, _CODE[wide], norm._ptr)
    return outs, norm


def global_norm(arrays) -> ndarray:
    """The square root of the sum of the squares of every element of every
    array, as a float32 scalar array (float64 if one of them is); squares are
    summed in float64, where those of float64 elements from 1e154 on are
    infinite."""
    return _clip(arrays, None, None)[1]


def clip_by_global_norm(arrays, max_norm, out=None):
    """``(clipped, norm)``: the arrays scaled by ``min(1, max_norm / norm)``,
    a list in their order and types, and their :func:`global_norm` before.
    ``out`` is a list of arrays to write (the same arrays, to clip them in
    place; one that overlaps another array, as tied weights' gradients given
    twice do, is an error).  A norm of NaN makes everything NaN."""
    limit = _scalar(max_norm, "max_norm")
    if not limit >= 0 or math.isnan(limit):
        raise ValueError(f"max_norm must not be negative or NaN: {max_norm}")
    return _clip(arrays, limit, out)
