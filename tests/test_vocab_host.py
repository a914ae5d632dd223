"""Vocabulary operators on the host: typing, refusals, scheduling of launches, ABI validation."""
import pytest
import torch

import fugatensor_b200 as ft
import fugatensor_b200.nn.functional as F
from fugatensor_b200 import _fgt, _native, operators


def leaf(shape, dtype=ft.fp32, engine=None):
    return ft.Tensor(engine or ft.current_engine(), dtype, shape, data=torch.empty(0))


TABLE, IDS = ((10, 4), ft.fp32), ((3, 2), ft.int64)
LOGITS, TARGETS = ((5, 7), ft.bf16), ((5,), ft.int32)


def test_results_are_typed_before_anything_runs():
    y = F.embedding(leaf(*TABLE), leaf(*IDS), scale=2)
    assert (y.shape, y.dtype, y.is_pending) == ((3, 2, 4), ft.fp32, True)
    assert F.cross_entropy(leaf(*LOGITS), leaf(*TARGETS)).shape == ()
    rows = F.cross_entropy(leaf((2, 5, 7)), leaf((2, 5), ft.int64), reduction="none")
    assert rows.shape == (2, 5) and rows.dtype is ft.fp32
    d = ft.grad(rows, rows._expr[1][0], seed=leaf((2, 5)))
    assert d.shape == (2, 5, 7) and d.is_pending
    a = F.adjust_logits(leaf(*LOGITS), leaf((5, 9), ft.int32), leaf((5,), ft.int32))
    assert a.shape == (5, 7) and a.dtype is ft.bf16


@pytest.mark.parametrize("error,match,call", [
    (TypeError, "must be a Tensor", lambda: F.embedding([1.0], leaf(*IDS))),
    (TypeError, "embedding table must have dtype", lambda: F.embedding(leaf((3, 4), ft.int32), leaf(*IDS))),
    (TypeError, "embedding indices must have dtype", lambda: F.embedding(leaf(*TABLE), leaf((3,)))),
    (ValueError, r"\[vocab, dim\]", lambda: F.embedding(leaf((3,)), leaf(*IDS))),
    (ValueError, "different engines", lambda: F.embedding(leaf(*TABLE), leaf(*IDS, engine=ft.Engine("cuda:0")))),
    (ValueError, "padding_idx is out of range", lambda: F.embedding(leaf(*TABLE), leaf(*IDS), padding_idx=10)),
    (TypeError, "padding_idx", lambda: F.embedding(leaf(*TABLE), leaf(*IDS), padding_idx=True)),
    (ValueError, "scale must be finite", lambda: F.embedding(leaf(*TABLE), leaf(*IDS), scale=float("inf"))),
    (ValueError, "targets must have shape", lambda: F.cross_entropy(leaf(*LOGITS), leaf((4,), ft.int32))),
    (TypeError, "targets must have dtype", lambda: F.cross_entropy(leaf(*LOGITS), leaf((5,)))),
    (ValueError, "with a vocabulary", lambda: F.cross_entropy(leaf((5, 0)), leaf(*TARGETS))),
    (ValueError, "reduction must be", lambda: F.cross_entropy(leaf(*LOGITS), leaf(*TARGETS), reduction="max")),
    (ValueError, "label_smoothing must be in", lambda: F.cross_entropy(leaf(*LOGITS), leaf(*TARGETS), label_smoothing=1.5)),
    (ValueError, "z_loss must not be", lambda: F.cross_entropy(leaf(*LOGITS), leaf(*TARGETS), z_loss=-1.0)),
    (TypeError, "ignore_index", lambda: F.cross_entropy(leaf(*LOGITS), leaf(*TARGETS), ignore_index=1.0)),
    (ValueError, "64 bits", lambda: F.cross_entropy(leaf(*LOGITS), leaf(*TARGETS), ignore_index=2 ** 63)),
    (ValueError, "need tokens", lambda: F.adjust_logits(leaf(*LOGITS), lengths=leaf((5,), ft.int32))),
    (ValueError, "tokens must have shape", lambda: F.adjust_logits(leaf(*LOGITS), leaf((4, 9), ft.int32))),
    (ValueError, "lengths must have shape", lambda: F.adjust_logits(leaf(*LOGITS), leaf((5, 9), ft.int32), leaf((5, 1), ft.int32))),
    (TypeError, "same dtype", lambda: F.adjust_logits(leaf(*LOGITS), leaf((5, 9), ft.int32), leaf((5,), ft.int32),
                                                     prompt_lengths=leaf((5,), ft.int64))),
    (ValueError, "repetition must be positive", lambda: F.adjust_logits(leaf(*LOGITS), repetition=0.0)),
    (TypeError, "presence must have dtype", lambda: F.adjust_logits(leaf(*LOGITS), presence=leaf((5,), ft.bf16))),
    (TypeError, "frequency must be a number", lambda: F.adjust_logits(leaf(*LOGITS), frequency="1")),
    (ValueError, "given together", lambda: F.adjust_logits(leaf(*LOGITS), bias=leaf((5, 2)))),
    (ValueError, "bias must have shape", lambda: F.adjust_logits(leaf(*LOGITS), bias=leaf((5, 2)), bias_tokens=leaf((5, 3), ft.int32))),
    (ValueError, "allowed must have shape", lambda: F.adjust_logits(leaf(*LOGITS), allowed=leaf((5, 2), ft.int32))),
    (ValueError, r"\[\.\.\., vocab\]", lambda: F.adjust_logits(leaf(()))),
])
def test_refusals(error, match, call):
    with pytest.raises(error, match=match):
        call()


def test_derivatives_that_do_not_exist_are_refused():
    from fugatensor_b200.autograd import DifferentiationError
    x = leaf(*LOGITS)
    with pytest.raises(DifferentiationError, match="adjust_logits"):
        ft.grad(ft.sum(F.adjust_logits(x, repetition=2.0)), x)
    d = ft.grad(F.cross_entropy(x, leaf(*TARGETS)), x)
    with pytest.raises(DifferentiationError, match="cross_entropy_grad"):
        ft.grad(ft.sum(d), x)


def test_operators_do_not_enter_a_partition():
    y = F.embedding(leaf(*TABLE), leaf(*IDS))
    with pytest.raises(TypeError, match="embedding is an operator"):
        y.engine.trace(ft.exp(y))


def test_a_loss_and_its_gradient_are_one_launch_unless_the_seed_needs_the_loss():
    x, t = leaf((5, 7)), leaf(*TARGETS)
    loss = F.cross_entropy(x, t)
    grad = ft.grad(loss, x)
    ((members, needs),) = operators.units([loss, grad])
    assert members == [loss, grad] and not needs
    squared = ft.grad(loss * loss, x)
    todo = operators.units([loss, squared])
    assert [len(m) for m, _ in todo] == [1, 1] and todo[1][1] == {0}
    other = F.cross_entropy(x, t, label_smoothing=0.5)
    assert len(operators.units([other, grad])) == 2  # another loss


def test_pairs_form_in_any_order_of_the_roots():
    x, t = leaf((5, 7)), leaf(*TARGETS)
    loss = F.cross_entropy(x, t)
    one, two = ft.grad(loss, x), ft.grad(loss, x)
    for roots in ([loss, one, two], [one, loss, two], [one, two, loss]):
        for todo in (operators.direct(roots), [m for m, _ in operators.units(roots)]):
            assert sorted(len(m) for m in todo) == [1, 2]
            assert any(m is loss for m in next(m for m in todo if len(m) == 2))
            assert sorted(id(m) for ms in todo for m in ms) == sorted(map(id, roots))
    assert operators.direct([ft.exp(x)]) is None
    assert operators.direct([F.cross_entropy(x * 2.0, t)]) is None


def test_gradients_of_one_operator_are_found_directly_or_through_the_graph():
    x, t = leaf((5, 7)), leaf(*TARGETS)
    direct = ft.grad(F.cross_entropy(x, t), x)
    (through,) = ft.grad((F.cross_entropy(x, t),), (x,))
    assert direct._expr[0] == through._expr[0] == "cross_entropy_grad"
    assert direct._expr[1][0] is through._expr[1][0] is x and direct._expr[2] == through._expr[2]
    unrelated = ft.grad(F.cross_entropy(x, t), leaf((3,)))
    assert unrelated.shape == (3,) and unrelated._expr[0] != "cross_entropy_grad"


def test_crossed_pairs_do_not_deadlock():
    """Each gradient's seed is the other loss: pairing both would be a cycle."""
    x, t, y, u = leaf((5, 7)), leaf(*TARGETS), leaf((5, 9)), leaf(*TARGETS)
    a, b = F.cross_entropy(x, t), F.cross_entropy(y, u)
    da, db = ft.grad(a * b, (x, y))
    todo = operators.units([a, b, da, db])
    done = set()
    for i, (members, needs) in enumerate(todo):
        assert needs <= done
        done.add(i)
    assert sorted(id(m) for ms, _ in todo for m in ms) == sorted(map(id, (a, b, da, db)))


def test_launches_wait_for_operators_behind_partitions():
    table, ids, t = leaf((10, 7)), leaf((5,), ft.int32), leaf(*TARGETS)
    y = F.embedding(table, ids)
    loss = F.cross_entropy(y * 2.0, t)
    d = ft.grad(loss, table)
    todo = operators.units([loss, d])
    kinds = [[m._expr[0] for m in ms] for ms, _ in todo]
    assert kinds == [["embedding"], ["cross_entropy", "cross_entropy_grad"], ["embedding_grad"]]
    assert [set(n) for _, n in todo] == [set(), {0}, {1}]


def test_constant_seeds_are_folded_and_others_are_operands():
    x = leaf((5, 7))
    loss = F.cross_entropy(x, leaf(*TARGETS))
    assert ft.grad(loss, x)._expr[2][4] == 1.0
    assert ft.grad(loss * 8.0 / 3.0, x)._expr[2][4] == float(torch.tensor(8.0) / torch.tensor(3.0))
    assert len(ft.grad(loss, x, seed=leaf(()))._expr[1]) == 3


def test_partitions_of_constants_have_a_plan():
    c = ft.exp(leaf((2,)).engine._splat(2.0, ft.fp32, (3,)))
    spec, _, leaves, _ = c.engine.compile(c)
    assert not leaves and [b["id"] for b in spec.execution_plan["buffers"]] == ["out0"]


def test_no_cpu_path():
    if torch.cuda.is_available():
        pytest.skip("a GPU is present")
    with pytest.raises(_fgt.CUDAError, match="no CPU execution path"):
        ft.evaluate(F.embedding(leaf(*TABLE), leaf(*IDS)))


@pytest.mark.parametrize("call,match,status", [
    (lambda: _native.embedding(3, 3, 8, 4, 2, 1.0, 256, 256, 256, 0), "indices must have dtype", 1),
    (lambda: _native.embedding(1, 1, 8, 4, 2, 1.0, 256, 256, 256, 0), "dtype must be", 1),
    (lambda: _native.embedding(3, 1, 8, 4, 2, 1.0, 260, 256, 256, 0), "table must be 16-byte aligned", 1),
    (lambda: _native.embedding(3, 1, 8, 4, 2, 1.0, 256, 0, 256, 0), "indices is NULL", 1),
    (lambda: _native.embedding(3, 1, -1, 4, 2, 1.0, 256, 256, 256, 0), "must not be negative", 1),
    (lambda: _native.embedding(3, 1, 2 ** 40, 2 ** 40, 2, 1.0, 256, 256, 256, 0), "too large", 1),
    (lambda: _native.embedding_grad(3, 1, 8, 4, 2, 1.0, -1, 256, 256, 0, 0, 0, 0), "dtable is NULL", 1),
    (lambda: _native.cross_entropy(3, 1, 3, 0.0, 0.0, 1.0, 2, 4, -100, 256, 256, 0, 256, 256, 256, 4096, 0), "unknown reduction", 1),
    (lambda: _native.cross_entropy(3, 1, 2, 2.0, 0.0, 1.0, 2, 4, -100, 256, 256, 0, 256, 256, 256, 4096, 0), "label_smoothing", 1),
    (lambda: _native.cross_entropy(3, 1, 2, 0.0, 0.0, 1.0, 2, 0, -100, 256, 256, 0, 256, 256, 256, 4096, 0), "vocab must be positive", 1),
    (lambda: _native.cross_entropy(3, 1, 2, 0.0, 0.0, 1.0, 2, 4, -100, 256, 256, 0, 0, 0, 256, 4096, 0), "neither loss nor dlogits", 1),
    (lambda: _native.cross_entropy(3, 1, 2, 0.0, 0.0, 1.0, 2, 4, -100, 256, 256, 0, 256, 256, 0, 0, 0), "workspace", 6),
    (lambda: _native.adjust_logits(3, 1, 1, 1, 2, 8, 4, 0, 0.0, 0.0, 0.0, 256, 256, 0, 0, 0, 0, 0, 0, 0, 0, 256, 0), "repetition must be positive", 1),
    (lambda: _native.adjust_logits(3, 1, 1, 1, 2, 8, 0, 0, 1.0, 0.0, 0.0, 256, 0, 256, 0, 0, 0, 0, 0, 0, 0, 256, 0), "lengths are given without tokens", 1),
    (lambda: _native.adjust_logits(3, 1, 1, 1, 2, 8, 0, 3, 1.0, 0.0, 0.0, 256, 0, 0, 0, 0, 0, 0, 256, 0, 0, 256, 0), "given together", 1),
    (lambda: _native.adjust_logits(3, 1, 1, 1, 2, 8, 0, 0, 1.0, 0.0, 0.0, 256, 0, 0, 0, 0, 0, 0, 0, 0, 258, 256, 0), "allowed must be 16-byte", 1),
])
def test_entry_points_validate_before_launching(call, match, status):
    with pytest.raises(_fgt.FgtError, match=match) as e:
        _fgt.check(call())
    assert e.value.status == status
