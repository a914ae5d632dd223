"""Operators of the vocabulary: nodes of the lazy graph that run as native kernels of their own.

A partition (one fused kernel list) covers the Fuga primitives; an operator
is a pending tensor whose expression names an entry point of the C ABI
(include/fgt.h) instead: embedding rows and their gradient, cross-entropy and
its gradient, the rules that edit logits. ``Engine.evaluate`` cuts the graph
at them: whatever an operator reads is evaluated first (as partitions and
operators), and partitions take operator results as inputs. A loss and its
gradient that are evaluated together run as one launch that reads the logits
from memory once.

The public functions are in ``nn.functional``; this module types the nodes,
gives their VJPs and launches them. Like partitions they run on the current
stream, with outputs and workspaces from torch's allocator, and have no CPU
path.
"""
from __future__ import annotations

import numpy as np

from .tensor import Tensor

NAMES = frozenset(("embedding", "embedding_grad", "cross_entropy", "cross_entropy_grad", "adjust_logits"))
_DIRECT = ("embedding", "cross_entropy")  # differentiable in their first operand alone
REDUCTIONS = {"none": 0, "sum": 1, "mean": 2}
_DT = {"bool": 0, "i32": 1, "i64": 2, "f32": 3, "f16": 4, "bf16": 5}
_native = _fgt = torch = _TORCH = None  # loaded with the first launch


def node(op, args, attrs, dtype, shape):
    """A pending tensor for operator ``op`` (dtype and shape are already in their final form)."""
    t = Tensor.__new__(Tensor)
    t._engine, t._dtype, t._shape = args[0]._engine, dtype, shape
    t._data, t._expr, t._ops = None, (op, args, attrs), True
    return t


def _scalar(t, depth=4):
    """The value of a rank-0 f32 expression of a few constants (a loss scale), or None."""
    if t._expr is None or t._shape != () or not depth:
        return None
    op, args, attrs = t._expr
    if op == "constant":
        return float(np.float32(attrs[0]))
    if op in ("mul", "div"):
        a, b = (_scalar(x, depth - 1) for x in args)
        if a is not None and b is not None:
            with np.errstate(all="ignore"):  # as the f32 partition would compute it
                return float(np.float32(a) * np.float32(b) if op == "mul" else np.float32(a) / np.float32(b))
    return None


# ------------------------------------------------------------- gradients ---
def vjp(t, g, active):
    """Cotangents of an operator's operands given its cotangent ``g`` (None: the number one)."""
    op, args, attrs = t._expr
    if op == "embedding":
        table, indices = args
        scale, padding = attrs
        grad = node("embedding_grad", (indices, g), (table._shape[0], scale, padding), table._dtype, table._shape)
        return [grad if active[0] else None, None]
    if op == "cross_entropy":
        logits, targets = args
        value = 1.0 if g is None else _scalar(g)
        seed, scale = ((), value) if value is not None else ((g,), 1.0)
        return [node("cross_entropy_grad", (logits, targets) + seed, attrs + (scale,), logits._dtype, logits._shape), None]
    from .autograd import DifferentiationError
    raise DifferentiationError(f"{op} has no derivative rule")


def vjp_direct(out, leaf, seed):
    """``vjp`` of an operator that reads ``leaf`` and no pending tensor (there is no other path
    between the two); None where that is not so."""
    expr = out._expr
    if expr is None or expr[0] not in _DIRECT or expr[1][0] is not leaf:
        return None
    for a in expr[1]:
        if a._expr is not None:
            return None
    return vjp(out, seed, (True, False))[0]


# ------------------------------------------------------------ scheduling ---
def _pending_order(roots):
    """The pending tensors under ``roots``, operands first."""
    order, seen = [], set()
    stack = [(r, False) for r in reversed(roots)]
    while stack:
        t, done = stack.pop()
        if done:
            order.append(t)
            continue
        if t._expr is None or id(t) in seen:
            continue
        seen.add(id(t))
        stack.append((t, True))
        for a in t._expr[1]:
            if a._expr is not None and id(a) not in seen:
                stack.append((a, False))
    return order


_NONE = frozenset()


def units(roots):
    """The operators under ``roots`` as launches with the launches they wait for.

    Returns a list of (members, needs): ``members`` are one operator, or a
    loss with its gradient; ``needs`` the indices of the launches whose results
    they read, directly or through partitions. A pair is only formed when the
    launches stay free of cycles (a seed computed from the loss itself keeps
    the two apart)."""
    order = _pending_order(roots)
    found = [t for t in order if t._expr[0] in NAMES]
    if len(found) == 1:
        return [(found, _NONE)]
    reads, below = {}, {}  # operators that an operator reads; that a tensor is or is computed from
    for t in order:
        got = _NONE
        for a in t._expr[1]:
            more = below.get(id(a), _NONE)
            got = got | more if got else more
        if t._expr[0] in NAMES:
            reads[id(t)] = got
            got = frozenset((id(t),))
        below[id(t)] = got

    group = {id(t): i for i, t in enumerate(found)}  # operator -> launch
    losses = {}
    for t in found:
        if t._expr[0] == "cross_entropy":
            losses[_pair_key(t)] = t
    for t in found:
        if t._expr[0] != "cross_entropy_grad":
            continue
        loss = losses.pop(_pair_key(t), None)  # one gradient per loss is paired
        if loss is None:
            continue
        alone = group[id(loss)]
        group[id(loss)] = group[id(t)]
        if _levels(found, group, reads) is None:
            group[id(loss)] = alone
    ordered = _levels(found, group, reads)
    at = {g: i for i, g in enumerate(ordered)}
    out = [([], set()) for _ in ordered]
    for t in found:
        i = at[group[id(t)]]
        out[i][0].append(t)
        out[i][1].update(at[group[r]] for r in reads[id(t)])
    return out


def _pair_key(t):
    return id(t._expr[1][0]), id(t._expr[1][1]), t._expr[2][:4]


def _levels(found, group, reads):
    """The launches in an order that respects ``reads``, or None if there is a cycle."""
    needs = {}
    for t in found:
        needs.setdefault(group[id(t)], set()).update(group[r] for r in reads[id(t)])
    ordered, done = [], set()
    while len(ordered) < len(needs):
        ready = [g for g, n in needs.items() if g not in done and n <= done]
        if not ready:
            return None
        ordered += ready
        done.update(ready)
    return ordered


def direct(roots):
    """``units`` where no root reads a pending tensor: no graph to order, or None if there is one."""
    groups, losses = [], {}
    for t in roots:
        if t._expr[0] not in NAMES:
            return None
        for a in t._expr[1]:
            if a._expr is not None:
                return None
        if t._expr[0] != "cross_entropy_grad":
            groups.append([t])
            if t._expr[0] == "cross_entropy":
                losses[_pair_key(t)] = groups[-1]
    for t in roots:
        if t._expr[0] == "cross_entropy_grad":
            group = losses.pop(_pair_key(t), None)
            if group is None:
                groups.append([t])
            else:
                group.append(t)
    return groups


# -------------------------------------------------------------- launches ---
def launch(members, data, stream):
    """Run one launch on raw ``stream``; ``data(tensor)`` gives an operand's buffer, which is kept until
    the launch is enqueued, and its address. Returns the members' results."""
    if _native is None:
        _load()
    return _LAUNCH[members[-1]._expr[0]](members, data, stream)


def _load():
    global _native, _fgt, torch, _TORCH
    import torch
    from . import _fgt, _native
    _TORCH = {ir: _fgt.torch_dtype(ir) for ir in _DT}


def _empty(t, like):
    return like.new_empty(t._shape, dtype=_TORCH[t._dtype.ir])


def _workspace(size, like):
    return like.new_empty((size,), dtype=torch.uint8) if size else None


def _check(status):
    if status:
        _fgt.check(status)


def _embedding(members, data, stream):
    (t,) = members
    (table, indices), (scale, padding) = t._expr[1:]
    (tb, table_at), (ib, ids_at) = data(table), data(indices)
    out = _empty(t, tb)
    _check(_native.embedding(_DT[t._dtype.ir], _DT[indices._dtype.ir], table._shape[0], table._shape[1], ib.numel(),
                             scale, table_at, ids_at, out.data_ptr(), stream))
    return (out,)


def _embedding_grad(members, data, stream):
    (t,) = members
    (indices, g), (vocab, scale, padding) = t._expr[1:]
    (ib, ids_at), (gb, g_at) = data(indices), data(g)
    out = _empty(t, gb)
    desc = (_DT[t._dtype.ir], _DT[indices._dtype.ir], vocab, t._shape[1], ib.numel(), scale,
            -1 if padding is None else padding)
    size = _native.embedding_grad_workspace(*desc)
    ws = _workspace(size, gb)
    _check(_native.embedding_grad(*desc, ids_at, g_at, out.data_ptr(), ws.data_ptr() if size else 0, size, stream))
    return (out,)


def _cross_entropy(members, data, stream):
    loss = grad = None
    for t in members:
        if t._expr[0] == "cross_entropy":
            loss = t
        else:
            grad = t
    args, attrs = (loss if grad is None else grad)._expr[1:]
    logits, targets = args[:2]
    ignore, smoothing, z, reduction = attrs[:4]
    (xb, logits_at), (tb, targets_at) = data(logits), data(targets)
    seed, seed_at = data(args[2]) if len(args) == 3 else (None, 0)
    loss_out = None if loss is None else _empty(loss, xb)
    grad_out = None if grad is None else torch.empty_like(xb)
    desc = (_DT[logits._dtype.ir], _DT[targets._dtype.ir], REDUCTIONS[reduction], smoothing, z,
            1.0 if grad is None else attrs[4], tb.numel(), logits._shape[-1], ignore)
    size = _native.cross_entropy_workspace(*desc)
    ws = _workspace(size, xb)
    _check(_native.cross_entropy(*desc, logits_at, targets_at, seed_at, 0 if loss is None else loss_out.data_ptr(),
                                 0 if grad is None else grad_out.data_ptr(), ws.data_ptr() if size else 0, size, stream))
    return [loss_out if t is loss else grad_out for t in members]


# the operands' places in the native call
_RULES = {name: i for i, name in enumerate(("logits", "tokens", "lengths", "prompt_lengths", "repetition", "presence",
                                            "frequency", "bias_tokens", "bias", "allowed"))}


def _adjust_logits(members, data, stream):
    (t,) = members
    args, (names, repetition, presence, frequency) = t._expr[1:]
    at, kept = [0] * len(_RULES), []
    token = length = bias_token = 1  # dtypes of what is not given: any
    history = biases = 0
    for name, a in zip(names, args):
        i = _RULES[name]
        buffer, at[i] = data(a)
        kept.append(buffer)
        if i == 1:
            token, history = _DT[a._dtype.ir], a._shape[-1]
        elif i in (2, 3):
            length = _DT[a._dtype.ir]
        elif i == 7:
            bias_token, biases = _DT[a._dtype.ir], a._shape[-1]
    x = kept[0]
    out = torch.empty_like(x)
    vocab = t._shape[-1]
    _check(_native.adjust_logits(_DT[t._dtype.ir], token, length, bias_token, x.numel() // vocab if vocab else 0, vocab,
                                 history, biases, repetition, presence, frequency, *at, out.data_ptr(), stream))
    return (out,)


_LAUNCH = {"embedding": _embedding, "embedding_grad": _embedding_grad, "cross_entropy": _cross_entropy,
           "cross_entropy_grad": _cross_entropy, "adjust_logits": _adjust_logits}
