"""The layer operators' checks and their compiled binding (layer norm, dropout, and both with a residual sum).

The binding (``_layers.so``, from ``csrc/layer_binding.cpp``) allocates outputs and workspaces with torch's caching
allocator, calls the C ABI on torch's current stream of the input's device and records the backward nodes, all
outside Python.  It registers the operators as ``torch.ops.serron.layer_norm``, ``dropout`` and
``dropout_add_layer_norm``, which tracers, fake tensors and function transforms see.  What it cannot be handed is refused here: checks of tensors raise ``RuntimeError`` worded as the
other operators' are, checks of numbers ``ValueError``.
"""

from __future__ import annotations

import importlib
import math
import operator
from types import ModuleType

import torch

from . import _lib

_binding: ModuleType | None = None


def binding() -> ModuleType:
    """The compiled binding (loaded once).  There is no fallback."""
    global _binding
    if _binding is None:
        _lib.load()
        try:
            _binding = importlib.import_module("._layers", __package__)
        except ImportError as exc:
            raise ImportError(
                f"serron_b200: the compiled binding of the layer operators cannot be loaded ({exc}); build it with "
                f"`make -C serron_b200/csrc` (or __graft_entry__.build()) for the installed torch"
            ) from exc
    return _binding


def check_input(name: str, input_: torch.Tensor) -> None:
    if not input_.is_cuda:
        raise RuntimeError(f"serron::{name}: input must be a CUDA tensor")
    if input_.dtype not in _lib.DTYPE_CODE:
        raise RuntimeError(f"serron::{name}: unsupported dtype {input_.dtype}")


def check_residual(name: str, input_: torch.Tensor, residual: torch.Tensor) -> None:
    if residual.shape != input_.shape:
        raise RuntimeError(f"serron::{name}: residual and input must share a shape, got {tuple(residual.shape)} and "
                           f"{tuple(input_.shape)}")
    if residual.dtype != input_.dtype:
        raise RuntimeError(f"serron::{name}: residual and input must share a dtype")
    if residual.device != input_.device:
        raise RuntimeError(f"serron::{name}: all tensors must be on one device")


def check_norm(name: str, input_: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, dim: int,
               eps: float) -> int:
    """The normalised dimension, counted from the front."""
    ndim = input_.dim()
    if not -ndim <= dim < ndim:
        raise ValueError(f"serron.{name}: dim {dim} is out of range for a {ndim}-D input")
    dim %= ndim
    length = input_.shape[dim]
    if length == 0:
        raise ValueError(f"serron.{name}: dimension {dim} of the input is empty")
    if not (eps >= 0 and math.isfinite(eps)):
        raise ValueError(f"serron.{name}: eps must be finite and not negative, got {eps}")
    for what, t in (("weight", weight), ("bias", bias)):
        if t is None:
            continue
        if t.dim() != 1 or t.shape[0] != length:
            raise RuntimeError(f"serron::{name}: {what} must have the shape ({length},) of the normalised dimension, "
                               f"got {tuple(t.shape)}")
        if t.device != input_.device:
            raise RuntimeError(f"serron::{name}: all tensors must be on one device")
        if t.dtype != input_.dtype and (t.dtype != torch.float32 or input_.dtype == torch.float64):
            raise RuntimeError(f"serron::{name}: {what} must be float32 or have the input's dtype, got {t.dtype}")
    if weight is not None and bias is not None and weight.dtype != bias.dtype:
        raise RuntimeError(f"serron::{name}: weight and bias must share a dtype")
    return dim


def check_drop(name: str, input_: torch.Tensor, p: float, seed: int | torch.Tensor, sequence: int
               ) -> tuple[float, int, torch.Tensor | None, int]:
    """``(p, seed, seed in a tensor, sequence)`` as the binding takes them."""
    tensor = None
    p, sequence = float(p), operator.index(sequence)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"serron.{name}: p must be between 0 and 1, got {p}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"serron.{name}: a seed in a tensor is one int64, got {seed.numel()} of {seed.dtype}")
        if seed.device != input_.device:
            raise RuntimeError(f"serron::{name}: all tensors must be on one device")
        seed, tensor = 0, seed
    else:
        seed = operator.index(seed)
        if not 0 <= seed < 1 << 64:
            raise ValueError(f"serron.{name}: seed must be in [0, 2^64), got {seed}")
    if not 0 <= sequence < 1 << 64:
        raise ValueError(f"serron.{name}: sequence must be in [0, 2^64), got {sequence}")
    return p, seed, tensor, sequence
