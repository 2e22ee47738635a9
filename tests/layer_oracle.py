"""Layer norm, dropout and their join in 64 bits, and how far a 32-bit computation may be from them.

Error bounds.  u is the unit roundoff of the arithmetic (2^-24, or 2^-53 for float64), v that of the type a result is
stored in.  No input of a row's statistics takes part in more than K = 64 roundings (32 additions of a thread, 5 of a
warp, 32 warps or chunks at most, and the elementwise steps), so a mean is off by at most K u max|x| and everything
derived from it in proportion.  With X = max|x| rstd over the row (what a rounding of the mean costs xhat), A = max|xhat|
and G = max|g|:

* y:  v |y| + K u (|xhat| + X + 1) |w| + K u |b|
* dx: v |dx| + K u rstd G (1 + A + X)^2
* dw: v |dw| + 4 K u sum over rows of |gy| (|xhat| + X + 1), db: v |db| + 4 K u sum |gy|  (128 rows a first-level sum)

Types of 16 bits add half their smallest subnormal step.
"""

from __future__ import annotations

import numpy as np
import torch

K = 64
ROUNDOFF = {torch.float64: 2.0**-53, torch.float32: 2.0**-24, torch.float16: 2.0**-11, torch.bfloat16: 2.0**-8}
STEP = {torch.float64: 0.0, torch.float32: 2.0**-149, torch.float16: 2.0**-25, torch.bfloat16: 2.0**-134}

_M0, _M1, _W0, _W1 = 0xD2511F53, 0xCD9E8D57, 0x9E3779B9, 0xBB67AE85
_LOW = np.uint64(0xFFFFFFFF)


def philox(blocks: np.ndarray, sequence: int, seed: int) -> np.ndarray:
    """Words (len(blocks), 4) of the Philox4x32-10 blocks with counters (blocks, sequence) under ``seed``."""
    blocks = blocks.astype(np.uint64)
    c = [blocks & _LOW, blocks >> np.uint64(32), np.full_like(blocks, sequence & 0xFFFFFFFF),
         np.full_like(blocks, sequence >> 32)]
    k = [seed & 0xFFFFFFFF, seed >> 32]
    for _ in range(10):
        a, b = c[0] * np.uint64(_M0), c[2] * np.uint64(_M1)
        c = [(b >> np.uint64(32)) ^ c[1] ^ np.uint64(k[0]), b & _LOW,
             (a >> np.uint64(32)) ^ c[3] ^ np.uint64(k[1]), a & _LOW]
        k = [(k[0] + _W0) & 0xFFFFFFFF, (k[1] + _W1) & 0xFFFFFFFF]
    return np.stack(c, 1)


def kept(first: int, count: int, p: float, seed: int, sequence: int) -> torch.Tensor:
    """Decisions ``first`` .. ``first + count - 1``."""
    low = first // 4
    words = philox(np.arange(low, (first + count + 3) // 4), sequence, seed).reshape(-1)
    return torch.from_numpy(words[first - 4 * low:][:count] >= np.uint64(round(p * 2**32)))


def dropout(x: torch.Tensor, p: float, seed: int, sequence: int, span: int = 1,
            residual: torch.Tensor | None = None) -> torch.Tensor:
    """The exact bits: a 32-bit product, a 32-bit sum, one rounding (64 bits for float64)."""
    wide = torch.float64 if x.dtype == torch.float64 else torch.float32
    keep = kept(0, -(-x.numel() // span), p, seed, sequence).repeat_interleave(span)[:x.numel()].view(x.shape).to(x.device)
    scale = torch.tensor(1 / (1 - p) if p < 1 else 0.0, dtype=wide, device=x.device)
    y = torch.where(keep, x.to(wide) * scale, torch.zeros((), dtype=wide, device=x.device))
    return (y if residual is None else y + residual.to(wide)).to(x.dtype)


class Norm:
    """Layer norm over ``dim`` in 64 bits, with the bounds above.  ``work``: the type the kernels compute in."""

    def __init__(self, x, weight, bias, dim, eps):
        self.u = ROUNDOFF[torch.float64 if x.dtype == torch.float64 else torch.float32]
        self.dtype, self.dim = x.dtype, dim
        self.pdtype = next((t.dtype for t in (weight, bias) if t is not None), x.dtype)
        along = [-1 if d == dim % x.dim() else 1 for d in range(x.dim())]
        self.others = [d for d in range(x.dim()) if d != dim % x.dim()]
        self.w = None if weight is None else weight.double().view(along)
        self.b = None if bias is None else bias.double().view(along)
        xd = x.double()
        mean = xd.mean(dim, keepdim=True)
        self.rstd = 1 / ((xd - mean).square().mean(dim, keepdim=True) + eps).sqrt()
        self.xhat = (xd - mean) * self.rstd
        self.X = xd.abs().amax(dim, keepdim=True) * self.rstd
        self.y = self.xhat if self.w is None else self.xhat * self.w
        if self.b is not None:
            self.y = self.y + self.b

    def y_bound(self):
        w = 1.0 if self.w is None else self.w.abs()
        b = 0.0 if self.b is None else self.b.abs()
        own = ROUNDOFF[self.dtype] * self.y.abs() + STEP[self.dtype]
        return own + K * self.u * ((self.xhat.abs() + self.X + 1) * w + b)

    def backward(self, gy, add=None):
        """dx (plus ``add``), dw, db and their bounds."""
        gy = gy.double()
        g = gy if self.w is None else gy * self.w
        dx = self.rstd * (g - g.mean(self.dim, keepdim=True)
                          - self.xhat * (g * self.xhat).mean(self.dim, keepdim=True))
        G, A = g.abs().amax(self.dim, keepdim=True), self.xhat.abs().amax(self.dim, keepdim=True)
        dx_off = K * self.u * self.rstd * G * (1 + A + self.X).square()
        if add is not None:
            dx = dx + add.double()
            dx_off = dx_off + K * self.u * add.double().abs()
        self.dx_exact, self.dx_off = dx, dx_off
        dw, db = (gy * self.xhat).sum(self.others), gy.sum(self.others)
        v, s = ROUNDOFF[self.pdtype], STEP[self.pdtype]
        return [(dx, dx_off + ROUNDOFF[self.dtype] * dx.abs() + STEP[self.dtype]),
                (dw, v * dw.abs() + s + 4 * K * self.u * (gy.abs() * (self.xhat.abs() + self.X + 1)).sum(self.others)),
                (db, v * db.abs() + s + 4 * K * self.u * gy.abs().sum(self.others))]


def within(got: torch.Tensor, want: torch.Tensor, bound: torch.Tensor, what: str) -> None:
    assert got.shape == want.shape, (what, got.shape, want.shape)
    off = (got.double() - want).abs()
    bad = ~(off <= bound)
    if bool(bad.any()):
        at = int((off / bound.clamp_min(1e-300)).nan_to_num(float("inf")).argmax())
        raise AssertionError(f"{what}: {int(bad.sum())} of {bad.numel()} outside; worst at {at}: got "
                             f"{got.reshape(-1)[at].item()}, want {want.reshape(-1)[at].item()}, bound "
                             f"{bound.expand_as(want).reshape(-1)[at].item():.3g}")
