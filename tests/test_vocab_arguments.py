"""Arguments of the vocabulary operators at the ends of their ranges, on the host."""
import pytest

from fugatensor_b200 import _fgt, _native


@pytest.mark.parametrize("reduction,loss", [(0, 0), (0, 256), (1, 0), (2, 0)])  # a reduced loss has a value: written on the GPU
def test_cross_entropy_of_no_rows_takes_outputs_without_addresses(reduction, loss):
    _fgt.check(_native.cross_entropy(3, 1, reduction, 0.0, 0.0, 1.0, 0, 4, -100, 0, 0, 0, loss, 0, 256, 4096, 0))
