"""Learnable morphology layers (packages/serron/torch-ext/serron/modules.py:16-73).

``weight`` is a ``(channels, k, k)`` parameter, zero at construction (a flat structuring element).

``LayerNorm2d``, ``Dropout`` and ``DropoutAddLayerNorm2d`` are what a network puts around them (no reference
counterpart).
"""

from __future__ import annotations

import torch
from torch import nn

from . import functional as F
from .enums import BorderMode, DropoutUnit


class _MorphologyNd(nn.Module):
    def __init__(self, channels: int, kernel_size: int, *, border: BorderMode = BorderMode.REPLICATE,
                 dtype: torch.dtype = torch.float32, device: torch.device | str | None = None) -> None:
        super().__init__()
        self.channels = channels
        self.kernel_size = kernel_size
        self.border = border
        self.weight = nn.Parameter(torch.empty(channels, kernel_size, kernel_size, dtype=dtype, device=device))
        self.reset_parameters()

    def reset_parameters(self) -> None:
        with torch.no_grad():
            self.weight.zero_()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        raise NotImplementedError


class Erosion2d(_MorphologyNd):
    """Learnable 2-D erosion."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return F.erosion(x, self.weight, border=self.border)


class Dilation2d(_MorphologyNd):
    """Learnable 2-D dilation."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return F.dilation(x, self.weight, border=self.border)


class Opening2d(_MorphologyNd):
    """Learnable 2-D opening (erosion, then dilation, by the same weights)."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return F.opening(x, self.weight, border=self.border)


class Closing2d(_MorphologyNd):
    """Learnable 2-D closing (dilation, then erosion, by the same weights)."""

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return F.closing(x, self.weight, border=self.border)


class LayerNorm2d(nn.Module):
    """Layer norm of an ``(N, C, H, W)`` map over its channels, at every pixel by itself.

    ``weight`` (one at construction) and ``bias`` (zero) have an entry per channel; with ``affine=False`` there are none.
    """

    def __init__(self, channels: int, *, eps: float = 1e-5, affine: bool = True, dtype: torch.dtype = torch.float32,
                 device: torch.device | str | None = None) -> None:
        super().__init__()
        self.channels = channels
        self.eps = eps
        self.weight = nn.Parameter(torch.empty(channels, dtype=dtype, device=device)) if affine else None
        self.bias = nn.Parameter(torch.empty(channels, dtype=dtype, device=device)) if affine else None
        self.reset_parameters()

    def reset_parameters(self) -> None:
        if self.weight is not None:
            with torch.no_grad():
                self.weight.fill_(1.0)
                self.bias.zero_()

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return F.layer_norm(x, self.weight, self.bias, eps=self.eps)


def _draw_seed() -> int:
    """A seed from torch's CPU generator: ``torch.manual_seed`` repeats it, and recomputing a layer under restored
    generator states (activation checkpointing) draws the same mask."""
    return int(torch.randint(0, (1 << 63) - 1, (), dtype=torch.int64))


class Dropout(nn.Module):
    """Dropout of elements, channels or samples while training, and the sum with a residual where one is given."""

    def __init__(self, p: float = 0.5, *, unit: DropoutUnit = DropoutUnit.ELEMENT) -> None:
        super().__init__()
        self.p = p
        self.unit = unit

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x if residual is None else x + residual
        return F.dropout(x, self.p, seed=_draw_seed(), unit=self.unit, residual=residual)


class DropoutAddLayerNorm2d(LayerNorm2d):
    """``(layer_norm(h), h)`` with ``h = residual + dropout(x)``; nothing is dropped outside training."""

    def __init__(self, channels: int, p: float = 0.5, *, eps: float = 1e-5, affine: bool = True,
                 dtype: torch.dtype = torch.float32, device: torch.device | str | None = None) -> None:
        super().__init__(channels, eps=eps, affine=affine, dtype=dtype, device=device)
        self.p = p

    def forward(self, x: torch.Tensor, residual: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
        drops = self.training and self.p > 0.0
        return F.dropout_add_layer_norm(x, residual, self.weight, self.bias, p=self.p if drops else 0.0,
                                        seed=_draw_seed() if drops else 0, eps=self.eps)
