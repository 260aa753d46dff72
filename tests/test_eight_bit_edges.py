"""8-bit weights on the host: what is said of a matrix is looked at, and a model that is refused stays whole."""

import plain_eight_bit as plain
import pytest
import torch
from test_eight_bit import BF16, E4M3, _small, e4m3

from llmserve_triton_kernels_b200 import ops
from llmserve_triton_kernels_b200.config.presets import PRESETS
from llmserve_triton_kernels_b200.config.registry import architecture_of
from llmserve_triton_kernels_b200.models.load import random_model


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


@pytest.mark.parametrize("cfg", [_small(intermediate_size=264), PRESETS["nurolorn-small"]], ids=["a matrix late in a layer", "a part that cannot"])
def test_a_refused_model_stays_as_it_was(cfg, monkeypatch):
    """Every matrix is looked at before the first is changed."""

    def quantize(w, rows=1):
        values, scales = plain.quantize(w, rows)
        return ops.Quantized(values.float().to(E4M3), scales.float(), rows)

    monkeypatch.setattr(ops, "quantize_blocks", quantize)
    model = random_model(architecture_of(cfg).config_class.from_dict(cfg), 0, BF16, "cpu")
    before = model.weight_bytes()
    with pytest.raises(ValueError, match="8-bit weights"):
        model.quantize_weights()
    assert model.weight_bytes() == before
    for _, part in model._named_parts:
        assert not any(isinstance(value, ops.Quantized) for value in vars(part).values())


def test_a_model_is_quantised_once(monkeypatch):
    """The second time there is no bfloat16 matrix left to start from."""
    monkeypatch.setattr(ops, "quantize_blocks", lambda w, rows=1: ops.Quantized(e4m3(*w.shape), torch.ones(-(-w.shape[0] // 128), -(-w.shape[1] // 128)), rows))
    model = random_model(architecture_of(_small()).config_class.from_dict(_small()), 0, BF16, "cpu")
    model.quantize_weights()
    before = model.weight_bytes()
    with pytest.raises(ValueError, match="8-bit weights"):
        model.quantize_weights()
    assert model.weight_bytes() == before
