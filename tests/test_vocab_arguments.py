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
