"""From a model folder, or from a configuration and a seed, to a bound :class:`Model`."""

from __future__ import annotations

from pathlib import Path

import torch

from ..config.registry import get_architecture, read_config
from ..weights.loader import check_tensors, read_safetensors
from ..weights.random_init import random_tensors
from .model import Model

DTYPES = {"bfloat16": torch.bfloat16, "float32": torch.float32}


def resolve_dtype(dtype) -> torch.dtype:
    if isinstance(dtype, torch.dtype):
        if dtype not in DTYPES.values():
            raise ValueError(f"dtype must be one of {sorted(DTYPES)}, got {dtype}")
        return dtype
    if dtype not in DTYPES:
        raise ValueError(f"dtype must be one of {sorted(DTYPES)}, got {dtype!r}")
    return DTYPES[dtype]


def quantized_weights(weight_dtype) -> bool:
    """Whether ``weight_dtype`` asks for 8-bit weights: None (the compute type) or "float8" (e4m3)."""
    if weight_dtype not in (None, "float8", torch.float8_e4m3fn):
        raise ValueError(f"weight_dtype must be None or 'float8', got {weight_dtype!r}")
    return weight_dtype is not None


def resolve_cache_dtype(cache_dtype, dtype: torch.dtype, model=None) -> torch.dtype:
    """The pages' type: None (the compute type) or "float8" (e4m3, a power of two for every head's vector)."""
    if cache_dtype is None:
        return dtype
    if cache_dtype not in ("float8", torch.float8_e4m3fn):
        raise ValueError(f"cache_dtype must be None or 'float8', got {cache_dtype!r}")
    if model is not None and not model.takes_eight_bit_pages():
        raise ValueError("8-bit pages are built for bfloat16 grouped-query attention with heads of 64 or 128 lanes; this model has other layers that keep pages")
    return torch.float8_e4m3fn


def load_model(model_dir: str | Path, dtype="bfloat16", device="cuda:0", weight_dtype=None):
    """``(model, configuration)`` of the folder; the model class follows config.json's ``architectures``.  ``weight_dtype`` "float8":
    the layers' matrices are put into 8 bits once they are loaded."""
    quantize = quantized_weights(weight_dtype)
    arch, config = read_config(model_dir)
    model = (arch.model_class or Model)(arch.plan(config), resolve_dtype(dtype), device)
    tensors = read_safetensors(model_dir)
    check_tensors(tensors, model.tensor_specs(), model.ignored_tensor_names(), where=str(model_dir))
    model.bind(tensors)
    if quantize:
        model.quantize_weights()
    return model, config


def random_model(config, seed: int, dtype="bfloat16", device="cuda:0", std: float = 0.02, storage=torch.bfloat16, weight_dtype=None):
    """The model that :func:`write_random_model` would write and :func:`load_model` read back, without the disk."""
    quantize = quantized_weights(weight_dtype)
    arch = get_architecture(config.architecture)
    model = (arch.model_class or Model)(arch.plan(config), resolve_dtype(dtype), device)
    model.bind(random_tensors(model.tensor_specs(), seed, std, storage))
    if quantize:
        model.quantize_weights()
    return model
