"""8-bit weights on the host: what is said of a matrix is looked at, and a model that is refused stays whole."""

import pytest
import torch
from test_eight_bit import e4m3

from llmserve_triton_kernels_b200 import ops


@pytest.mark.parametrize("bad", [0.3, 3.0, 0.0, -0.5, 2.0**-127, 1e-45, float("inf"), float("nan")])
@pytest.mark.parametrize("rows", [1, 128])
def test_powers_of_two_are_looked_at(bad, rows):
    """The tensor cores would take the exponent of a scale and drop the rest."""
    scales = torch.exp2(torch.tensor([[-126.0, 0.0], [5.0, 127.0]]))
    m = 2 if rows == 1 else 130
    assert ops.Quantized(e4m3(m, 256), scales, rows, powers_of_two=True).powers_of_two
    scales[1, 0] = bad
    with pytest.raises(ops.KernelError, match="powers of two"):
        ops.Quantized(e4m3(m, 256), scales, rows, powers_of_two=True)
    assert not ops.Quantized(e4m3(m, 256), scales, rows).powers_of_two  # any scales, where nothing is said of them


def test_powers_of_two_of_nothing():
    assert ops.Quantized(e4m3(0, 256), torch.ones(0, 2), 128, powers_of_two=True).powers_of_two
