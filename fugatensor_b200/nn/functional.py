"""Row graphs written in primitives (reference: src/fugatensor/nn/functional.py:82-198).

The decompositions are the reference's, op for op: f16/bf16 inputs are
upcast to f32 for statistics and cast back, the affine ``* weight`` and
``+ bias`` run after the cast back in the input dtype, softmax's max is under
stop_gradient, mean is sum / count. The backend fuses each of these (and
their VJPs) into one row kernel.

``embedding``, ``cross_entropy`` and ``adjust_logits`` are operators with
native kernels of their own (operators.py): lazy like everything else, and
differentiable by ``ft.grad`` (``adjust_logits`` is for choosing tokens and
has no derivative).
"""
from __future__ import annotations

from .. import dtypes as _dt
from .. import operators as _operators
from .. import ops as _ops
from ..autograd import stop_gradient
from ..tensor import Tensor as _Tensor

_FLOAT, _INDEX = ("f32", "f16", "bf16"), ("i32", "i64")
_F32_OVER, _F32_ZERO = 2.0 ** 128 - 2.0 ** 103, 2.0 ** -150  # f32: infinite from here on; zero down from here


def _norm_axes(x, normalized_shape, axis):
    rank = x.ndim
    if normalized_shape is not None and axis is not None:
        raise ValueError("specify either normalized_shape or axis, not both")
    if axis is not None:
        axes = _ops._axes(axis, rank)
        return axes, tuple(x.shape[a] for a in axes)
    if normalized_shape is None:
        if rank == 0:
            raise ValueError("normalization requires at least 1D input when normalized_shape is omitted")
        norm_shape = (x.shape[-1],)
    elif isinstance(normalized_shape, int):
        norm_shape = (normalized_shape,)
    else:
        norm_shape = tuple(normalized_shape)
    if not norm_shape or len(norm_shape) > rank or x.shape[-len(norm_shape):] != norm_shape:
        raise ValueError(f"normalized_shape {norm_shape} does not match trailing shape {x.shape}")
    return tuple(range(rank - len(norm_shape), rank)), norm_shape


def _apply_affine(x, normalized_shape, weight=None, bias=None):
    target = x.shape
    if weight is not None:
        w = weight.astype(x.dtype) if weight.dtype is not x.dtype else weight
        x = x * _ops.broadcast_to(w, target)
    if bias is not None:
        b = bias.astype(x.dtype) if bias.dtype is not x.dtype else bias
        x = x + _ops.broadcast_to(b, target)
    return x


def _work(x):
    return x.astype(_dt.fp32) if x.dtype in (_dt.fp16, _dt.bf16) else x


def softmax(x, axis=-1):
    """Numerically stable softmax along ``axis`` (f16/bf16 statistics in f32)."""
    work = _work(x)
    m = stop_gradient(_ops.amax(work, axis=axis, keepdims=True))
    shifted = work - _ops.broadcast_to(m, work.shape)
    ex = _ops.exp(shifted)
    denom = _ops.broadcast_to(_ops.sum(ex, axis=axis, keepdims=True), work.shape)
    out = ex / denom
    return out.astype(x.dtype) if work is not x else out


def log_softmax(x, axis=-1):
    work = _work(x)
    m = stop_gradient(_ops.amax(work, axis=axis, keepdims=True))
    shifted = work - _ops.broadcast_to(m, work.shape)
    lse = _ops.log(_ops.sum(_ops.exp(shifted), axis=axis, keepdims=True))
    out = shifted - _ops.broadcast_to(lse, work.shape)
    return out.astype(x.dtype) if work is not x else out


def layer_norm(x, normalized_shape=None, weight=None, bias=None, *, eps=1e-5, axis=None):
    axes, norm_shape = _norm_axes(x, normalized_shape, axis)
    work = _work(x)
    mean = _ops.broadcast_to(_ops.mean(work, axis=axes, keepdims=True), work.shape)
    diff = work - mean
    var = _ops.mean(diff * diff, axis=axes, keepdims=True)
    inv_std = _ops.broadcast_to(1 / _ops.sqrt(var + eps), work.shape)
    normed = diff * inv_std
    out = normed.astype(x.dtype) if work is not x else normed
    return _apply_affine(out, norm_shape, weight=weight, bias=bias)


def rms_norm(x, normalized_shape=None, weight=None, *, eps=1e-6, axis=None):
    axes, norm_shape = _norm_axes(x, normalized_shape, axis)
    work = _work(x)
    ms = _ops.mean(work * work, axis=axes, keepdims=True)
    inv_rms = _ops.broadcast_to(1 / _ops.sqrt(ms + eps), work.shape)
    out = work * inv_rms
    out = out.astype(x.dtype) if work is not x else out
    return _apply_affine(out, norm_shape, weight=weight, bias=None)


def _tensor(x, what, kinds, like=None):
    if not isinstance(x, _Tensor):
        raise TypeError(f"{what} must be a Tensor")
    if like is not None and x._engine is not like._engine:
        raise ValueError("tensors belong to different engines")
    if x._dtype.ir not in kinds:
        raise TypeError(f"{what} must have dtype {' or '.join(kinds)}, not {x._dtype.ir}")
    return x


def _number(x, what):
    if type(x) not in (int, float):
        raise TypeError(f"{what} must be a number")
    if not -_F32_OVER < x < _F32_OVER:
        raise ValueError(f"{what} must be finite in f32")
    return float(x)


def embedding(table, indices, *, scale=1.0, padding_idx=None):
    """``scale * table[indices]``: a row of ``table`` [vocab, dim] for every index.

    Indices outside [0, vocab) read a row of zeros and take no part in the
    gradient (as in ``gather``). The gradient of ``table`` adds the cotangent's
    rows in f32 and rounds once: in the order of their indices, for an index that
    occurs more than 64 times in fixed pieces of 64 whose sums are then added in
    order. The row ``padding_idx`` gets none.
    """
    _tensor(table, "embedding table", _FLOAT)
    _tensor(indices, "embedding indices", _INDEX, table)
    if table.ndim != 2:
        raise ValueError(f"embedding table must be [vocab, dim], got shape {table._shape}")
    scale = _number(scale, "scale")
    if padding_idx is not None:
        if type(padding_idx) is not int:
            raise TypeError("padding_idx must be an int")
        if not 0 <= padding_idx < table._shape[0]:
            raise ValueError("padding_idx is out of range")
    return _operators.node("embedding", (table, indices), (scale, padding_idx), table._dtype,
                           indices._shape + (table._shape[1],))


def cross_entropy(logits, targets, *, ignore_index=-100, label_smoothing=0.0, z_loss=0.0, reduction="mean"):
    """Cross-entropy of ``logits`` [..., vocab] against the token ids ``targets`` [...], in f32.

    A row's loss is ``lse - (1 - e) * x[t] - e / vocab * sum(x) + z_loss * lse**2``
    with ``lse = log(sum(exp(x)))`` and ``e = label_smoothing``. Rows whose
    target is ``ignore_index`` or outside [0, vocab) have loss 0 and gradient 0
    and do not count in the mean (0 when no row counts). A counted row whose
    logits are all -inf has no distribution: its loss and gradient are NaN.
    Evaluated together with its ``ft.grad``, loss and gradient are one launch
    that reads the logits from memory once.
    """
    _tensor(logits, "cross_entropy logits", _FLOAT)
    _tensor(targets, "cross_entropy targets", _INDEX, logits)
    if not logits._shape or logits._shape[-1] == 0:
        raise ValueError("cross_entropy logits must be [..., vocab] with a vocabulary")
    if targets._shape != logits._shape[:-1]:
        raise ValueError(f"cross_entropy targets must have shape {logits._shape[:-1]}, got {targets._shape}")
    if type(ignore_index) is not int:
        raise TypeError("ignore_index must be an int")
    if not -2 ** 63 <= ignore_index < 2 ** 63:
        raise ValueError("ignore_index must fit 64 bits")
    if reduction not in _operators.REDUCTIONS:
        raise ValueError(f"reduction must be one of {', '.join(_operators.REDUCTIONS)}")
    smoothing, z = _number(label_smoothing, "label_smoothing"), _number(z_loss, "z_loss")
    if not 0.0 <= smoothing <= 1.0:
        raise ValueError("label_smoothing must be in [0, 1]")
    if z < 0.0:
        raise ValueError("z_loss must not be negative")
    return _operators.node("cross_entropy", (logits, targets), (ignore_index, smoothing, z, reduction), _dt.fp32,
                           targets._shape if reduction == "none" else ())


def adjust_logits(logits, tokens=None, lengths=None, *, prompt_lengths=None, repetition=1.0, presence=0.0, frequency=0.0,
                  bias_tokens=None, bias=None, allowed=None):
    """``logits`` [..., vocab] edited for choosing the next token; in this order:

    - tokens of the row's history (``tokens`` [..., length]; the first
      ``lengths`` [...] of them, of which the first ``prompt_lengths`` [...] are the
      prompt): ``x / repetition`` where x > 0, ``x * repetition`` elsewhere;
    - tokens that occur c > 0 times after the prompt: ``x - frequency * c - presence``;
    - ``x + bias[k]`` for every k with ``bias_tokens[k]`` == token (``bias`` f32, both [..., k]);
    - -inf, whatever x was, where the token's bit in ``allowed`` is clear
      ([..., ceil(vocab / 32)] int32; bit v % 32 of word v // 32 is token v).

    ``repetition`` (> 0), ``presence`` and ``frequency`` are numbers or f32
    Tensors [...]. Tokens outside [0, vocab) are skipped, so histories may be
    padded with -1. Computed in f32 and rounded once to the logits' dtype. A
    row that allows nothing is all -inf.
    """
    _tensor(logits, "logits", _FLOAT)
    if not logits._shape:
        raise ValueError("logits must be [..., vocab]")
    batch, vocab = logits._shape[:-1], logits._shape[-1]
    names, args = ["logits"], [logits]

    def take(name, x, kinds, shape=None):  # None: the batch's, with a length of its own
        _tensor(x, name, kinds, logits)
        if shape is None:
            if not x._shape:
                raise ValueError(f"{name} must have shape {batch} and a length of its own, got ()")
            shape = batch + x._shape[-1:]
        if x._shape != shape:
            raise ValueError(f"{name} must have shape {shape}, got {x._shape}")
        if 0 not in shape:  # nothing in it: as if it had not been given
            names.append(name)
            args.append(x)

    if tokens is not None:
        take("tokens", tokens, _INDEX)
        for name, x in (("lengths", lengths), ("prompt_lengths", prompt_lengths)):
            if x is not None:
                take(name, x, _INDEX, batch)
        if lengths is not None and prompt_lengths is not None and lengths._dtype is not prompt_lengths._dtype:
            raise TypeError("lengths and prompt_lengths must have the same dtype")
        if 0 in tokens._shape:  # no history
            names, args = ["logits"], [logits]
    elif lengths is not None or prompt_lengths is not None:
        raise ValueError("lengths and prompt_lengths need tokens")
    numbers = []
    for name, x in (("repetition", repetition), ("presence", presence), ("frequency", frequency)):
        if isinstance(x, _Tensor):
            take(name, x, ("f32",), batch)
            numbers.append(1.0)
        else:
            numbers.append(_number(x, name))
    if numbers[0] <= _F32_ZERO:
        raise ValueError("repetition must be positive")
    if (bias is None) != (bias_tokens is None):
        raise ValueError("bias and bias_tokens are given together")
    if bias is not None:
        take("bias_tokens", bias_tokens, _INDEX)
        take("bias", bias, ("f32",), bias_tokens._shape)
    if allowed is not None:
        take("allowed", allowed, ("i32",), batch + (-(-vocab // 32),))
    return _operators.node("adjust_logits", tuple(args), (tuple(names), *numbers), logits._dtype, logits._shape)
