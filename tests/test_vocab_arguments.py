"""Arguments of the vocabulary operators at the ends of their ranges, on the host."""
import pytest
import torch

import fugatensor_b200 as ft
import fugatensor_b200.nn.functional as F
from fugatensor_b200 import _fgt, _native


def leaf(shape, dtype=ft.fp32):
    return ft.Tensor(ft.current_engine(), dtype, shape, data=torch.empty(0))


@pytest.mark.parametrize("reduction,loss", [(0, 0), (0, 256), (1, 0), (2, 0)])  # a reduced loss has a value: written on the GPU
def test_cross_entropy_of_no_rows_takes_outputs_without_addresses(reduction, loss):
    _fgt.check(_native.cross_entropy(3, 1, reduction, 0.0, 0.0, 1.0, 0, 4, -100, 0, 0, 0, loss, 0, 256, 4096, 0))


@pytest.mark.parametrize("dtype", [ft.int32, ft.int64])
@pytest.mark.parametrize("what", ["tokens", "bias_tokens"])
def test_lists_without_a_length_are_refused(dtype, what):
    """A single vector of logits has the shape () for a batch, which a rank-0 tensor has too."""
    lists = {what: leaf((), dtype)}
    if what == "bias_tokens":
        lists["bias"] = leaf(())
    with pytest.raises(ValueError, match=f"{what} must have shape"):
        F.adjust_logits(leaf((7,)), **lists)


TABLE, IDS, LOGITS, TARGETS = (10, 4), (3,), (5, 7), (5,)
F32_MAX = 2.0 ** 128 - 2.0 ** 104


@pytest.mark.parametrize("what,call", [
    ("scale", lambda x: F.embedding(leaf(TABLE), leaf(IDS, ft.int32), scale=x)),
    ("z_loss", lambda x: F.cross_entropy(leaf(LOGITS), leaf(TARGETS, ft.int32), z_loss=x)),
    ("repetition", lambda x: F.adjust_logits(leaf(LOGITS), repetition=x)),
    ("presence", lambda x: F.adjust_logits(leaf(LOGITS), presence=x)),
    ("frequency", lambda x: F.adjust_logits(leaf(LOGITS), frequency=x)),
])
def test_numbers_that_f32_does_not_hold_are_refused_when_the_node_is_made(what, call):
    for x in (1e300, -1e39, 2.0 ** 128 - 2.0 ** 103, 10 ** 400, float("inf"), float("nan")):
        with pytest.raises(ValueError, match=f"{what} must be finite"):
            call(x)
    call(F32_MAX)
    call(2.0 ** 128 - 2.0 ** 103 - 2.0 ** 76)  # rounds down to the largest f32


def test_a_repetition_that_is_zero_in_f32_is_refused():
    for x in (1e-60, 2.0 ** -150, 0, -1.0):
        with pytest.raises(ValueError, match="repetition must be positive"):
            F.adjust_logits(leaf(LOGITS), repetition=x)
    F.adjust_logits(leaf(LOGITS), repetition=2.0 ** -149)


def test_the_largest_z_loss_is_an_argument_of_the_entry_point():
    _fgt.check(_native.cross_entropy(3, 1, 0, 0.0, F32_MAX, 1.0, 0, 4, -100, 0, 0, 0, 0, 0, 0, 0, 0))
