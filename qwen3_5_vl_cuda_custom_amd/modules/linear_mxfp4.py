"""A linear layer with its weight in MXFP4 (no reference counterpart; the reference's weights are bf16 or fp32)."""
from __future__ import annotations

import torch
from torch import nn

from ..kernels import matmul_mxfp4, mxfp4_dequantize, mxfp4_quantize
from ..kernels.mxfp4 import MX_BLOCK
from .linear import CudaLinear


class CudaLinearMXFP4(nn.Module):
    """CudaLinear for inference with a four-bit weight: buffers `weight_codes` (out, in / 2) and `weight_scales`
    (out, in / 32), `bias` (out) or None. bf16 input; x·Wᵀ + b (+ residual) with the weight as quantised."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True) -> None:
        super().__init__()
        if in_features % MX_BLOCK:
            raise ValueError(f"CudaLinearMXFP4: in_features {in_features} must be a multiple of {MX_BLOCK}")
        self.in_features = in_features
        self.out_features = out_features
        self.register_buffer("weight_codes", torch.zeros(out_features, in_features // 2, dtype=torch.uint8))
        self.register_buffer("weight_scales", torch.zeros(out_features, in_features // MX_BLOCK, dtype=torch.uint8))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features), requires_grad=False)
        else:
            self.register_parameter("bias", None)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: CudaLinear) -> "CudaLinearMXFP4":
        """The layer quantised from a CudaLinear on the GPU (bf16 or fp32 weight; the bias becomes bf16)."""
        q = cls(linear.in_features, linear.out_features, bias=False)
        q.weight_codes, q.weight_scales = mxfp4_quantize(linear.weight.detach())
        if linear.bias is not None:
            q.bias = nn.Parameter(linear.bias.detach().to(torch.bfloat16, copy=True), requires_grad=False)
        return q

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The weight (out, in) that the codes stand for."""
        return mxfp4_dequantize(self.weight_codes, self.weight_scales, dtype)

    @property
    def pair(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(weight_codes, weight_scales), as the products over several weights take them."""
        return self.weight_codes, self.weight_scales

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, *,
                out: torch.Tensor | None = None) -> torch.Tensor:
        return matmul_mxfp4(x, self.weight_codes, self.weight_scales, self.bias, residual, out=out)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"
