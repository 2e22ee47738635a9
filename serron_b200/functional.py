"""Stateless morphology on CUDA tensors.

Same functions, signatures, defaults and errors as packages/serron/torch-ext/serron/functional.py.
``erosion`` / ``dilation`` go through the autograd functions.  The derived operations run in one launch
(``serron_derived_forward``: both extremes from one staged tile for the gradient, the intermediate image
in shared memory for the others) when the input and the structuring element share a dtype, autocast is
off and the window is at most 7 a side; otherwise they are the reference's compositions.  Both give the
same bits.  The reconstructions run on the library's fixed-point solver instead of a Python loop.

``layer_norm``, ``dropout`` and ``dropout_add_layer_norm`` are what a network puts around the learnable
layers; the reference has no counterpart.  They compute in float32 (float64 for float64 inputs) and return the
input's dtype, so autocast leaves them as they are.  The gradients of the norms cannot be differentiated again, and there
are no forward-mode derivatives: both are errors.
"""

from __future__ import annotations

import math

import torch

from . import _flatness, _layer_ops, _ops
from ._autotune import ensure_loaded
from .autograd import _DerivedFunction, _DilateFunction, _ErodeFunction
from .enums import BORDER_TO_INT, BorderMode, DropoutUnit


def erosion(input_: torch.Tensor, kernel: torch.Tensor, *, border: BorderMode = BorderMode.REPLICATE) -> torch.Tensor:
    """Grayscale erosion (sliding minimum of ``input - kernel``)."""
    return _ErodeFunction.apply(input_, kernel, BORDER_TO_INT[border])


def dilation(input_: torch.Tensor, kernel: torch.Tensor, *, border: BorderMode = BorderMode.REPLICATE) -> torch.Tensor:
    """Grayscale dilation (sliding maximum of ``input + kernel``)."""
    return _DilateFunction.apply(input_, kernel, BORDER_TO_INT[border])


def _fused(mode: int, input_: torch.Tensor, kernel: torch.Tensor) -> bool:
    """Whether derived operation ``mode`` runs in one launch for these arguments (same bits either way)."""
    return (isinstance(input_, torch.Tensor) and isinstance(kernel, torch.Tensor) and input_.is_cuda
            and not torch.is_autocast_enabled("cuda") and _ops.derived_supported(mode, input_, kernel))


def opening(input_: torch.Tensor, kernel: torch.Tensor, *, border: BorderMode = BorderMode.REPLICATE) -> torch.Tensor:
    """Erosion followed by dilation."""
    if _fused(_ops.DERIVED_OPENING, input_, kernel):
        return _DerivedFunction.apply(input_, kernel, BORDER_TO_INT[border], _ops.DERIVED_OPENING)
    return dilation(erosion(input_, kernel, border=border), kernel, border=border)


def closing(input_: torch.Tensor, kernel: torch.Tensor, *, border: BorderMode = BorderMode.REPLICATE) -> torch.Tensor:
    """Dilation followed by erosion."""
    if _fused(_ops.DERIVED_CLOSING, input_, kernel):
        return _DerivedFunction.apply(input_, kernel, BORDER_TO_INT[border], _ops.DERIVED_CLOSING)
    return erosion(dilation(input_, kernel, border=border), kernel, border=border)


def gradient(input_: torch.Tensor, kernel: torch.Tensor, *, border: BorderMode = BorderMode.REPLICATE) -> torch.Tensor:
    """Morphological gradient ``dilation(input) - erosion(input)``."""
    if _fused(_ops.DERIVED_GRADIENT, input_, kernel):
        return _DerivedFunction.apply(input_, kernel, BORDER_TO_INT[border], _ops.DERIVED_GRADIENT)
    return dilation(input_, kernel, border=border) - erosion(input_, kernel, border=border)


def top_hat(input_: torch.Tensor, kernel: torch.Tensor, *, border: BorderMode = BorderMode.REPLICATE) -> torch.Tensor:
    """White top-hat ``input - opening(input)``."""
    if _fused(_ops.DERIVED_TOP_HAT, input_, kernel):
        return _DerivedFunction.apply(input_, kernel, BORDER_TO_INT[border], _ops.DERIVED_TOP_HAT)
    return input_ - opening(input_, kernel, border=border)


def black_hat(input_: torch.Tensor, kernel: torch.Tensor, *, border: BorderMode = BorderMode.REPLICATE) -> torch.Tensor:
    """Black top-hat ``closing(input) - input``."""
    if _fused(_ops.DERIVED_BLACK_HAT, input_, kernel):
        return _DerivedFunction.apply(input_, kernel, BORDER_TO_INT[border], _ops.DERIVED_BLACK_HAT)
    return closing(input_, kernel, border=border) - input_


_DEFAULT_CHECK_EVERY = 16


def _align_inputs(marker: torch.Tensor, mask: torch.Tensor, kernel: torch.Tensor, name: str
                  ) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor, bool]:
    """Validate a reconstruction's three tensors and bring them to their common dtype."""
    if marker.shape != mask.shape:
        raise ValueError(f"{name}: marker and mask must share a shape, got {tuple(marker.shape)} and {tuple(mask.shape)}")
    if marker.device != mask.device or marker.device != kernel.device:
        raise ValueError(
            f"{name}: marker, mask and kernel must be on one device, got {marker.device}, {mask.device} and {kernel.device}"
        )
    if torch.is_grad_enabled() and (marker.requires_grad or mask.requires_grad or kernel.requires_grad):
        raise RuntimeError(f"{name}: reconstruction has no backward pass yet; run it under torch.no_grad() or detach its inputs")
    dtype = torch.promote_types(torch.promote_types(marker.dtype, mask.dtype), kernel.dtype)
    flat = _flatness.is_flat(kernel)
    return marker.to(dtype), mask.to(dtype), _flatness.mark(kernel.to(dtype), flat), flat


def _require_nonnegative_anchor(kernel: torch.Tensor, name: str) -> None:
    """A negative (or NaN) anchor tap would make the geodesic step non-monotone."""
    ah, aw = kernel.shape[-2] // 2, kernel.shape[-1] // 2
    if not bool((kernel[..., ah, aw] >= 0).all().item()):
        raise ValueError(
            f"{name}: the structuring element's anchor tap kernel[..., {ah}, {aw}] must be >= 0, "
            f"otherwise the geodesic iteration is not monotone and need not converge"
        )


def _reconstruct(marker: torch.Tensor, mask: torch.Tensor, kernel: torch.Tensor, border: BorderMode, *,
                 dilate: bool, max_iter: int | None, check_every: int, name: str) -> torch.Tensor:
    if check_every < 1:
        raise ValueError(f"{name}: check_every must be >= 1, got {check_every}")
    if max_iter is not None and max_iter < 1:
        raise ValueError(f"{name}: max_iter must be >= 1 or None, got {max_iter}")
    marker, mask, kernel, flat = _align_inputs(marker, mask, kernel, name)
    if not flat:
        _require_nonnegative_anchor(kernel, name)
    ensure_loaded(marker.device)
    with torch.no_grad():
        return _ops.reconstruct(dilate, marker, mask, kernel, BORDER_TO_INT[border], max_iter, check_every)


def reconstruction_by_dilation(marker: torch.Tensor, mask: torch.Tensor, kernel: torch.Tensor, *,
                               border: BorderMode = BorderMode.CONSTANT, max_iter: int | None = None,
                               check_every: int = _DEFAULT_CHECK_EVERY) -> torch.Tensor:
    """Fixed point of ``min(dilation(y), mask)`` from ``y = min(marker, mask)``.

    ``max_iter`` bounds the reference's Jacobi iteration count: with it set the reference's schedule is
    replayed and the call raises exactly when the reference would; without it the fixed point is found
    by tile-local relaxation, which reaches the same (unique) fixed point far sooner.
    """
    return _reconstruct(marker, mask, kernel, border, dilate=True, max_iter=max_iter, check_every=check_every,
                        name="serron.reconstruction_by_dilation")


def reconstruction_by_erosion(marker: torch.Tensor, mask: torch.Tensor, kernel: torch.Tensor, *,
                              border: BorderMode = BorderMode.CONSTANT, max_iter: int | None = None,
                              check_every: int = _DEFAULT_CHECK_EVERY) -> torch.Tensor:
    """Fixed point of ``max(erosion(y), mask)`` from ``y = max(marker, mask)`` (the dual)."""
    return _reconstruct(marker, mask, kernel, border, dilate=False, max_iter=max_iter, check_every=check_every,
                        name="serron.reconstruction_by_erosion")


def layer_norm(input_: torch.Tensor, weight: torch.Tensor | None = None, bias: torch.Tensor | None = None, *,
               dim: int = 1, eps: float = 1e-5) -> torch.Tensor:
    """``(input - mean) / sqrt(var + eps) * weight + bias`` with mean and (biased) variance over dimension ``dim``.

    ``dim=1`` normalises the channels of an (N, C, H, W) map at every pixel, ``dim=-1`` the features of tokens.
    ``weight`` and ``bias`` have one entry per element of ``dim``, in float32 or in the input's dtype; either may be
    None.  Any dense memory order of ``input_`` (channels_last, a transposed view) is read and written as it lies.
    """
    _layer_ops.check_input("layer_norm", input_)
    dim = _layer_ops.check_norm("layer_norm", input_, weight, bias, dim, eps)
    return _layer_ops.binding().layer_norm(input_, weight, bias, dim, eps)


def dropout(input_: torch.Tensor, p: float = 0.5, *, seed: int | torch.Tensor, sequence: int = 0,
            unit: DropoutUnit = DropoutUnit.ELEMENT, residual: torch.Tensor | None = None) -> torch.Tensor:
    """``input / (1 - p)`` where kept and 0 where dropped, each ``unit`` with probability ``p``; plus ``residual``.

    The mask is never stored: decision j (in row-major order of the elements, channels or samples) keeps its unit when
    word j % 4 of the Philox4x32-10 block with counter (j // 4, sequence) and key ``seed`` is at least
    round(p * 2^32).  Calls with the same seed and sequence share their mask, so every call of a training step takes
    a ``sequence`` (or a seed) of its own.  ``seed`` is an integer below 2^64, or an int64 CUDA tensor of one element,
    which a captured CUDA graph reads anew at every replay.  A dropped unit is 0 whatever it held.
    """
    _layer_ops.check_input("dropout", input_)
    rule = _layer_ops.check_drop("dropout", input_, p, seed, sequence)
    if residual is not None:
        _layer_ops.check_residual("dropout", input_, residual)
    span, unit = 1, DropoutUnit(unit)
    if unit is not DropoutUnit.ELEMENT:
        lead = 2 if unit is DropoutUnit.CHANNEL else 1
        if input_.dim() < lead:
            raise ValueError(f"serron.dropout: unit {unit.value!r} needs an input of at least {lead} dimensions, got "
                             f"{input_.dim()}")
        span = max(1, math.prod(input_.shape[lead:]))
    return _layer_ops.binding().dropout(input_, residual, span, *rule)


def dropout_add_layer_norm(input_: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None = None,
                           bias: torch.Tensor | None = None, *, p: float = 0.5, seed: int | torch.Tensor,
                           sequence: int = 0, dim: int = 1, eps: float = 1e-5) -> tuple[torch.Tensor, torch.Tensor]:
    """``(y, h)`` with ``h = residual + dropout(input)`` and ``y = layer_norm(h, weight, bias)``, in one pass.

    The end of a residual branch and the beginning of the next: ``h`` goes on along the residual path, ``y`` into the
    next branch.  ``h`` is rounded to the input's dtype and normalised as it is returned.  Arguments as for
    :func:`dropout` (by element) and :func:`layer_norm`; ``p=0`` (evaluation) needs no particular seed.
    """
    _layer_ops.check_input("dropout_add_layer_norm", input_)
    rule = _layer_ops.check_drop("dropout_add_layer_norm", input_, p, seed, sequence)
    _layer_ops.check_residual("dropout_add_layer_norm", input_, residual)
    dim = _layer_ops.check_norm("dropout_add_layer_norm", input_, weight, bias, dim, eps)
    return _layer_ops.binding().dropout_add_layer_norm(input_, residual, weight, bias, *rule, dim, eps)
