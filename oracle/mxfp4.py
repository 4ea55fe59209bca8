"""MXFP4 (blocks of 32 E2M1 values with an E8M0 scale) from its definition, in float64 on the CPU."""
from __future__ import annotations

import math

import torch

BLOCK = 32
_MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def values(codes: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """float64 values (..., K) of codes (..., K / 2) and scales (..., K / 32)."""
    two = torch.stack([codes & 15, codes >> 4], -1).flatten(-2).long()
    v = _MAGNITUDES[two & 7] * torch.where(two > 7, -1.0, 1.0).double()
    size = torch.where(scales == 255, torch.tensor(math.nan, dtype=torch.float64),
                       torch.exp2(scales.double() - 127))
    return v * size.repeat_interleave(BLOCK, -1)


def quantize(x: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """(codes, scales): a block's scale from its largest magnitude, each value to the nearest magnitude by search
    (the even code where two are equally near), saturating."""
    y = x.double().unflatten(-1, (-1, BLOCK))
    top = y.abs().amax(-1)
    bad = ~torch.isfinite(top)
    safe = torch.where(bad, 1.0, top)
    exp = torch.where(safe == 0, -127.0, torch.floor(torch.log2(safe.clamp(min=2.0 ** -200))) - 2).clamp(min=-127)
    # log2 may round up next to a power of two: the definition is exact, so step back where it did
    exp = torch.where((safe > 0) & (torch.exp2(exp + 2) > safe) & (exp > -127), exp - 1, exp)
    a = (y / torch.exp2(exp).unsqueeze(-1)).abs().nan_to_num(0.0, 0.0, 0.0)
    d = (a.unsqueeze(-1) - _MAGNITUDES).abs()
    near = d == d.amin(-1, keepdim=True)
    odd = torch.arange(8) % 2
    code = torch.argmax(near.double() * 2 - odd.double() * 0.5, -1)  # one of the nearest, an even one first
    code = (code + 8 * torch.signbit(y)).to(torch.uint8)
    code = torch.where(bad.unsqueeze(-1), torch.zeros_like(code), code).flatten(-2)
    scale = torch.where(bad, 255.0, exp + 127).to(torch.uint8)
    return code[..., 0::2] | (code[..., 1::2] << 4), scale


def attention(q, k, v, seen, scale: float):
    """(o, spread): o (B, Hq, Sq, D) = softmax over the first seen[b, i] rows of k / v (B, Hkv, rows, D), zeros where
    that is none; spread: the same weights over |v|, for error bounds. float64."""
    B, Hq, Sq, D = q.shape
    G = Hq // k.shape[1]
    o, spread = torch.zeros(B, Hq, Sq, D, dtype=torch.float64), torch.zeros(B, Hq, Sq, D, dtype=torch.float64)
    for b in range(B):
        for i in range(Sq):
            n = int(seen[b, i])
            if n <= 0:
                continue
            for h in range(Hq):
                w = torch.softmax(k[b, h // G, :n].double() @ q[b, h, i].double() * scale, 0)
                o[b, h, i] = w @ v[b, h // G, :n].double()
                spread[b, h, i] = w @ v[b, h // G, :n].double().abs()
    return o, spread
