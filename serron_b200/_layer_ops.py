"""Calls of the layer operators' C ABI: layer norm, dropout, and the two joined with a residual sum.

Tensors are checked here (the C ABI sees pointers, not devices or dtypes), outputs and workspaces come from
torch's caching allocator, and work is enqueued on torch's current stream of the input's device.  Checks of
tensors raise ``RuntimeError`` worded as the other operators' are; checks of numbers raise ``ValueError``.
"""

from __future__ import annotations

import math
import operator

import torch

from . import _lib

# how the saved statistics of a layer norm are held
_STATS = {torch.float32: torch.float32, torch.float64: torch.float64, torch.float16: torch.float32,
          torch.bfloat16: torch.float32}


# ------------------------------------------------------------------------------------------------
# validation
# ------------------------------------------------------------------------------------------------
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
               ) -> tuple[float, int | torch.Tensor, int]:
    """``(p, seed, sequence)`` as plain numbers (or a seed in a tensor)."""
    p, sequence = float(p), operator.index(sequence)
    if not 0.0 <= p <= 1.0:
        raise ValueError(f"serron.{name}: p must be between 0 and 1, got {p}")
    if isinstance(seed, torch.Tensor):
        if seed.dtype != torch.int64 or seed.numel() != 1:
            raise ValueError(f"serron.{name}: a seed in a tensor is one int64, got {seed.numel()} of {seed.dtype}")
        if seed.device != input_.device:
            raise RuntimeError(f"serron::{name}: all tensors must be on one device")
    else:
        seed = operator.index(seed)
        if not 0 <= seed < 1 << 64:
            raise ValueError(f"serron.{name}: seed must be in [0, 2^64), got {seed}")
    if not 0 <= sequence < 1 << 64:
        raise ValueError(f"serron.{name}: sequence must be in [0, 2^64), got {sequence}")
    return p, seed, sequence


def _seed_args(seed: int | torch.Tensor) -> tuple[int, int | None]:
    return (0, seed.data_ptr()) if isinstance(seed, torch.Tensor) else (seed, None)


# ------------------------------------------------------------------------------------------------
# layouts
# ------------------------------------------------------------------------------------------------
def norm_layout(x: torch.Tensor, dim: int) -> tuple[torch.Tensor, int, int, int]:
    """``(x, outer, length, inner)``: how the memory of ``x`` holds the rows of ``dim``.  Any dense order of the
    dimensions (channels_last, a transposed view) is taken as it lies; everything else is copied first."""
    shape, order = x.shape, range(x.dim())
    if not x.is_contiguous():
        order = sorted(order, key=lambda d: -x.stride(d))
        if not x.permute(order).is_contiguous():
            x = x.contiguous()
            order = range(x.dim())
    at = list(order).index(dim)
    sizes = [shape[d] for d in order]
    return x, math.prod(sizes[:at]), sizes[at], math.prod(sizes[at + 1:])


def _like(t: torch.Tensor, x: torch.Tensor) -> torch.Tensor:
    """``t`` in the dense memory order of ``x``."""
    return t if t.stride() == x.stride() else torch.empty_like(x).copy_(t)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _params(weight: torch.Tensor | None, bias: torch.Tensor | None, x: torch.Tensor
            ) -> tuple[torch.Tensor | None, torch.Tensor | None, int]:
    weight = None if weight is None else weight.contiguous()
    bias = None if bias is None else bias.contiguous()
    dtype = x.dtype if weight is None and bias is None else (bias if weight is None else weight).dtype
    return weight, bias, _lib.DTYPE_CODE[dtype]


def _workspace(x: torch.Tensor, outer: int, length: int, inner: int, backward: bool) -> tuple[torch.Tensor | None, int]:
    nbytes = _lib.load().serron_layer_norm_workspace_bytes(outer, length, inner, _lib.DTYPE_CODE[x.dtype], backward)
    if nbytes < 0:
        _lib.raise_for(_lib.ERR_INVALID)
    return (None if nbytes == 0 else torch.empty(nbytes, dtype=torch.uint8, device=x.device)), nbytes


def _stats(x: torch.Tensor, rows: int, wanted: bool) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    if not wanted:
        return None, None
    both = torch.empty((2, rows), dtype=_STATS[x.dtype], device=x.device)
    return both[0], both[1]


# ------------------------------------------------------------------------------------------------
# calls (arguments checked by the functions above)
# ------------------------------------------------------------------------------------------------
def layer_norm(input_: torch.Tensor, weight: torch.Tensor | None, bias: torch.Tensor | None, dim: int, eps: float,
               stats: bool) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor | None, torch.Tensor | None]:
    """``(y, x, mean, rstd)``: x is the input as the backward reads it; mean and rstd where ``stats`` asks for them."""
    x, outer, length, inner = norm_layout(input_, dim)
    weight, bias, param_code = _params(weight, bias, x)
    y = torch.empty_like(x)
    mean, rstd = _stats(x, outer * inner, stats)
    workspace, nbytes = _workspace(x, outer, length, inner, False)
    rc = _lib.load().serron_layer_norm(x.data_ptr(), outer, length, inner, _lib.DTYPE_CODE[x.dtype], _ptr(weight),
                                       _ptr(bias), param_code, eps, y.data_ptr(), _ptr(mean), _ptr(rstd),
                                       _ptr(workspace), nbytes, x.device.index, _lib.stream_of(x))
    _lib.raise_for(rc)
    return y, x, mean, rstd


def _empty_grads(needs: tuple[bool, bool], length: int, x: torch.Tensor, dtype: torch.dtype
                 ) -> tuple[torch.Tensor | None, torch.Tensor | None]:
    return tuple(torch.empty(length, dtype=dtype, device=x.device) if need else None for need in needs)


def layer_norm_backward(grad_output: torch.Tensor, x: torch.Tensor, mean: torch.Tensor, rstd: torch.Tensor,
                        weight: torch.Tensor | None, param_dtype: torch.dtype, dim: int,
                        needs: tuple[bool, bool, bool]) -> tuple[torch.Tensor | None, ...]:
    """Gradients of the input, the weight and the bias, those that ``needs`` asks for."""
    x, outer, length, inner = norm_layout(x, dim)
    grad_output = _like(grad_output, x)
    weight = None if weight is None else weight.contiguous()
    grad_input = torch.empty_like(x) if needs[0] else None
    grad_weight, grad_bias = _empty_grads(needs[1:], length, x, param_dtype)
    workspace, nbytes = _workspace(x, outer, length, inner, True)
    rc = _lib.load().serron_layer_norm_backward(
        grad_output.data_ptr(), x.data_ptr(), mean.data_ptr(), rstd.data_ptr(), outer, length, inner,
        _lib.DTYPE_CODE[x.dtype], _ptr(weight), _lib.DTYPE_CODE[param_dtype], _ptr(grad_input), _ptr(grad_weight),
        _ptr(grad_bias), _ptr(workspace), nbytes, x.device.index, _lib.stream_of(x))
    _lib.raise_for(rc)
    return grad_input, grad_weight, grad_bias


def dropout(input_: torch.Tensor, residual: torch.Tensor | None, span: int, p: float, seed: int | torch.Tensor,
            sequence: int) -> torch.Tensor:
    x = input_.contiguous()
    r = None if residual is None else residual.contiguous()
    y = torch.empty_like(x)
    rc = _lib.load().serron_dropout(x.data_ptr(), _ptr(r), x.numel(), span, _lib.DTYPE_CODE[x.dtype], p,
                                    *_seed_args(seed), sequence, y.data_ptr(), x.device.index, _lib.stream_of(x))
    _lib.raise_for(rc)
    return y


def dropout_add_layer_norm(input_: torch.Tensor, residual: torch.Tensor, weight: torch.Tensor | None,
                           bias: torch.Tensor | None, p: float, seed: int | torch.Tensor, sequence: int, dim: int,
                           eps: float, stats: bool) -> tuple[torch.Tensor, ...]:
    """``(y, h, mean, rstd)``."""
    x, r = input_.contiguous(), residual.contiguous()  # decisions are counted in the row-major order of the elements
    x, outer, length, inner = norm_layout(x, dim)
    weight, bias, param_code = _params(weight, bias, x)
    y, h = torch.empty_like(x), torch.empty_like(x)
    mean, rstd = _stats(x, outer * inner, stats)
    workspace, nbytes = _workspace(x, outer, length, inner, False)
    rc = _lib.load().serron_dropout_add_layer_norm(
        x.data_ptr(), r.data_ptr(), outer, length, inner, _lib.DTYPE_CODE[x.dtype], _ptr(weight), _ptr(bias),
        param_code, p, *_seed_args(seed), sequence, eps, h.data_ptr(), y.data_ptr(), _ptr(mean), _ptr(rstd),
        _ptr(workspace), nbytes, x.device.index, _lib.stream_of(x))
    _lib.raise_for(rc)
    return y, h, mean, rstd


def dropout_add_layer_norm_backward(grad_output: torch.Tensor, grad_sum: torch.Tensor | None, h: torch.Tensor,
                                    mean: torch.Tensor, rstd: torch.Tensor, weight: torch.Tensor | None,
                                    param_dtype: torch.dtype, p: float, seed: int | torch.Tensor, sequence: int,
                                    dim: int, needs: tuple[bool, bool, bool, bool]
                                    ) -> tuple[torch.Tensor | None, ...]:
    """Gradients of the input, the residual, the weight and the bias, those that ``needs`` asks for."""
    h, outer, length, inner = norm_layout(h, dim)
    grad_output = _like(grad_output, h)
    grad_sum = None if grad_sum is None else _like(grad_sum, h)
    weight = None if weight is None else weight.contiguous()
    grad_input = torch.empty_like(h) if needs[0] else None
    grad_residual = torch.empty_like(h) if needs[1] else None
    grad_weight, grad_bias = _empty_grads(needs[2:], length, h, param_dtype)
    workspace, nbytes = _workspace(h, outer, length, inner, True)
    rc = _lib.load().serron_dropout_add_layer_norm_backward(
        grad_output.data_ptr(), _ptr(grad_sum), h.data_ptr(), mean.data_ptr(), rstd.data_ptr(), outer, length, inner,
        _lib.DTYPE_CODE[h.dtype], _ptr(weight), _lib.DTYPE_CODE[param_dtype], p, *_seed_args(seed), sequence,
        _ptr(grad_input), _ptr(grad_residual), _ptr(grad_weight), _ptr(grad_bias), _ptr(workspace), nbytes,
        h.device.index, _lib.stream_of(h))
    _lib.raise_for(rc)
    return grad_input, grad_residual, grad_weight, grad_bias
