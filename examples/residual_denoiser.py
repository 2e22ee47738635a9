"""A residual network of learnable morphology that removes impulse noise, trained for a few steps.

Every block normalises its input over the channels, dilates or erodes it with learned structuring elements, mixes the
channels, drops a share of the result and adds it to the residual path; the sum and the next block's norm are one pass
(``DropoutAddLayerNorm2d``).  Whole channels are dropped before the head.  Run on a B200:

    python examples/residual_denoiser.py --steps 200
"""

from __future__ import annotations

import argparse
import os
import sys

import torch
from torch import nn

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))

import serron_b200 as serron  # noqa: E402


class Branch(nn.Module):
    """A learned dilation or erosion of every channel, then a mix of the channels."""

    def __init__(self, channels: int, layer: type[nn.Module]) -> None:
        super().__init__()
        self.morph = layer(channels, 3)
        self.mix = nn.Conv2d(channels, channels, 1)

    def forward(self, y: torch.Tensor) -> torch.Tensor:
        return self.mix(self.morph(y))


class Denoiser(nn.Module):
    def __init__(self, channels: int = 32, blocks: int = 4, p: float = 0.05) -> None:
        super().__init__()
        self.stem = nn.Conv2d(1, channels, 3, padding=1)
        self.norm = serron.LayerNorm2d(channels)
        layers = (serron.Erosion2d, serron.Dilation2d)
        self.branches = nn.ModuleList(Branch(channels, layers[k % 2]) for k in range(blocks))
        self.joins = nn.ModuleList(serron.DropoutAddLayerNorm2d(channels, p) for _ in range(blocks))
        self.drop = serron.Dropout(p, unit=serron.DropoutUnit.CHANNEL)
        self.head = nn.Conv2d(channels, 1, 1)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        h = self.stem(x)
        y = self.norm(h)
        for branch, join in zip(self.branches, self.joins):
            y, h = join(branch(y), h)  # y: normalised, into the next branch; h: along the residual path
        return self.head(self.drop(y))


def batch(n: int, size: int, gen: torch.Generator) -> tuple[torch.Tensor, torch.Tensor]:
    """Noisy and clean images of a few discs on a dark ground; a tenth of the pixels is set to 0 or 1."""
    device = gen.device
    at = torch.arange(size, device=device, dtype=torch.float32)
    centre = torch.rand(n, 5, 2, generator=gen, device=device) * size
    radius = size * (0.05 + 0.15 * torch.rand(n, 5, generator=gen, device=device))
    grey = 0.3 + 0.6 * torch.rand(n, 5, generator=gen, device=device)
    inside = ((at[:, None] - centre[..., 0, None, None]) ** 2 + (at - centre[..., 1, None, None]) ** 2
              <= radius[..., None, None] ** 2)
    clean = (inside * grey[..., None, None]).amax(1, keepdim=True)
    u = torch.rand(clean.shape, generator=gen, device=device)
    return torch.where(u < 0.05, 0.0, torch.where(u > 0.95, 1.0, clean)), clean


def train(steps: int, *, n: int = 16, size: int = 64, seed: int = 0, device: str = "cuda") -> tuple[nn.Module, list[float]]:
    """The trained network and the loss of every step."""
    torch.manual_seed(seed)
    gen = torch.Generator(device).manual_seed(seed)
    model = Denoiser().to(device)
    optimiser = torch.optim.Adam(model.parameters(), lr=3e-3)
    losses = []
    for _ in range(steps):
        noisy, clean = batch(n, size, gen)
        loss = (model(noisy) - clean).square().mean()
        optimiser.zero_grad()
        loss.backward()
        optimiser.step()
        losses.append(loss.detach())
    return model, torch.stack(losses).tolist()


def main() -> None:
    parser = argparse.ArgumentParser(description=__doc__)
    parser.add_argument("--steps", type=int, default=200)
    model, losses = train(parser.parse_args().steps)
    print(f"loss: first step {losses[0]:.4f}, last step {losses[-1]:.4f}")
    gen = torch.Generator("cuda").manual_seed(1)
    noisy, clean = batch(16, 64, gen)
    model.eval()
    with torch.no_grad():
        out = model(noisy)
    print(f"mean squared error: noisy {(noisy - clean).square().mean():.4f}, cleaned {(out - clean).square().mean():.4f}")


if __name__ == "__main__":
    main()
