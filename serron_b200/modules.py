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


def _draw_seed(x: torch.Tensor) -> int:
    """A seed from torch's CPU generator: ``torch.manual_seed`` repeats it, and recomputing a layer under restored
    generator states (activation checkpointing) draws the same mask.  A CUDA graph would keep it for all of its replays."""
    if x.is_cuda and torch.cuda.is_current_stream_capturing():
        raise RuntimeError("serron: a dropout layer that draws its own seed would drop the same elements in every replay of "
                           "a captured CUDA graph; pass it seed= as an int64 tensor on the GPU and change that between replays")
    return int(torch.randint(0, (1 << 63) - 1, (), dtype=torch.int64))


class Dropout(nn.Module):
    """Dropout of elements, channels or samples while training, and the sum with a residual where one is given.

    Every call draws a seed of its own, unless it is given ``seed`` (and ``sequence``) as :func:`functional.dropout` takes
    them: a captured CUDA graph needs a seed in a tensor, and layers that share it a ``sequence`` each.
    """

    def __init__(self, p: float = 0.5, *, unit: DropoutUnit = DropoutUnit.ELEMENT) -> None:
        super().__init__()
        self.p = p
        self.unit = unit

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, *,
                seed: int | torch.Tensor | None = None, sequence: int = 0) -> torch.Tensor:
        if not self.training or self.p == 0.0:
            return x if residual is None else x + residual
        return F.dropout(x, self.p, seed=_draw_seed(x) if seed is None else seed, sequence=sequence, unit=self.unit,
                         residual=residual)


class DropoutAddLayerNorm2d(LayerNorm2d):
    """``(layer_norm(h), h)`` with ``h = residual + dropout(x)``; nothing is dropped outside training.

    Seeds are drawn or given as in :class:`Dropout`.
    """

    def __init__(self, channels: int, p: float = 0.5, *, eps: float = 1e-5, affine: bool = True,
                 dtype: torch.dtype = torch.float32, device: torch.device | str | None = None) -> None:
        super().__init__(channels, eps=eps, affine=affine, dtype=dtype, device=device)
        self.p = p

    def forward(self, x: torch.Tensor, residual: torch.Tensor, *, seed: int | torch.Tensor | None = None,
                sequence: int = 0) -> tuple[torch.Tensor, torch.Tensor]:
        p = self.p if self.training else 0.0
        if p == 0.0:
            seed, sequence = 0, 0
        elif seed is None:
            seed = _draw_seed(x)
        return F.dropout_add_layer_norm(x, residual, self.weight, self.bias, p=p, seed=seed, sequence=sequence,
                                        eps=self.eps)
