"""MXFP8 (blocks of 32 E4M3 values with an E8M0 scale) from its definition, in float64 on the CPU."""
from __future__ import annotations

import math

import torch

BLOCK = 32
# the 127 magnitudes of E4M3, ascending: code c < 127 stands for entry c
_MAGNITUDES = torch.tensor([(c & 7) / 8 * 2.0 ** -6 if c < 8 else (1 + (c & 7) / 8) * 2.0 ** ((c >> 3) - 7)
                            for c in range(127)], dtype=torch.float64)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values (..., K) of codes (..., K) and scales (..., K / 32)."""
    c = codes.view(torch.uint8).long()
    v = torch.cat([_MAGNITUDES, torch.tensor([math.nan], dtype=torch.float64)])[c & 127]
    v = v * torch.where(c > 127, -1.0, 1.0).double()
    size = torch.where(scales == 255, torch.tensor(math.nan, dtype=torch.float64),
                       torch.exp2(scales.double() - 127))
    return v * size.repeat_interleave(BLOCK, -1)


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales): a block's scale the smallest that keeps it within 448, each value to the nearest magnitude by
    search (the even code where two are equally near)."""
    y = x.double().unflatten(-1, (-1, BLOCK))
    top = y.abs().amax(-1)
    bad = ~torch.isfinite(top)
    safe = torch.where(bad, 1.0, top)
    steps = 448 * torch.exp2(torch.arange(-127, 128, dtype=torch.float64))  # the largest value of each scale
    s = torch.searchsorted(steps, safe.contiguous())
    a = (y / torch.exp2(s.double() - 127).unsqueeze(-1)).abs()
    a = torch.where(bad.unsqueeze(-1), 0.0, a)
    hi = torch.searchsorted(_MAGNITUDES, a.contiguous()).clamp(max=126)
    lo = (hi - 1).clamp(min=0)
    dl, dh = a - _MAGNITUDES[lo], _MAGNITUDES[hi] - a
    code = torch.where((dl < dh) | ((dl == dh) & (lo % 2 == 0)), lo, hi)
    code = torch.where(bad.unsqueeze(-1), 0, code + 128 * torch.signbit(y)).flatten(-2)
    return code.to(torch.uint8).view(torch.float8_e4m3fn), torch.where(bad, 255, s).to(torch.uint8)


def product(x: torch.Tensor, w: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(x w^T, bound): float64 values x (M, K), w (N, K); bound: how far the matrix instruction's cut products and its
    fp32 sums may be from it. The products of eight consecutive k are cut 13 bits below the largest; every sum of 128 k
    added to the accumulators rounds to fp32 (2^-24 of at most the sum of magnitudes; twice that is allowed, for the sums
    inside the instruction and of the parts of k)."""
    y, mag = x @ w.T, x.abs() @ w.abs().T
    pad = -x.shape[1] % 8
    xg, wg = (torch.nn.functional.pad(t.abs(), (0, pad)).unflatten(-1, (-1, 8)) for t in (x, w))
    top = torch.zeros_like(y)
    for g in range(xg.shape[1]):
        top += (xg[:, None, g] * wg[None, :, g]).amax(-1)
    return y, 7 * 2.0 ** -13 * top + (x.shape[1] / 128 + 6) * 2.0 ** -23 * mag
