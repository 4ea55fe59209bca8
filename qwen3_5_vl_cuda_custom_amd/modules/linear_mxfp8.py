"""A linear layer with its weight in MXFP8 (no reference counterpart; the reference's weights are bf16 or fp32)."""
from __future__ import annotations

import torch
from torch import nn

from ..kernels import add_rmsnorm_mxfp8, matmul_mxfp8, mxfp8_dequantize, mxfp8_quantize
from ..kernels.mxfp8 import MX8_BLOCK
from .linear import CudaLinear
from .linear_mxfp4 import CudaLinearMXFP4
from .norms import CudaRMSNorm


class CudaLinearMXFP8(nn.Module):
    """CudaLinear for inference with an eight-bit weight: buffers `weight_codes` (out, in) float8_e4m3fn and
    `weight_scales` (out, in / 32), `bias` (out) or None. x·Wᵀ + b (+ residual) in bf16 with x (bf16 rows, which are
    quantised first, or a pair of codes and scales) and the weight as quantised."""

    def __init__(self, in_features: int, out_features: int, bias: bool = True) -> None:
        super().__init__()
        if in_features % MX8_BLOCK:
            raise ValueError(f"CudaLinearMXFP8: in_features {in_features} must be a multiple of {MX8_BLOCK}")
        self.in_features = in_features
        self.out_features = out_features
        self.register_buffer("weight_codes", torch.zeros(out_features, in_features, dtype=torch.float8_e4m3fn))
        self.register_buffer("weight_scales", torch.zeros(out_features, in_features // MX8_BLOCK, dtype=torch.uint8))
        if bias:
            self.bias = nn.Parameter(torch.zeros(out_features), requires_grad=False)
        else:
            self.register_parameter("bias", None)

    def _apply(self, fn, recurse: bool = True):
        # .to(dtype), .bfloat16() and the like convert every buffer of a floating-point type: the codes go as bytes.
        self.weight_codes = self.weight_codes.view(torch.uint8)
        try:
            return super()._apply(fn, recurse)
        finally:
            self.weight_codes = self.weight_codes.view(torch.float8_e4m3fn)

    @classmethod
    @torch.no_grad()
    def from_linear(cls, linear: CudaLinear) -> "CudaLinearMXFP8":
        """The layer quantised from a CudaLinear on the GPU (bf16 or fp32 weight; the bias becomes bf16)."""
        q = cls(linear.in_features, linear.out_features, bias=False)
        q.weight_codes, q.weight_scales = mxfp8_quantize(linear.weight.detach())
        if linear.bias is not None:
            q.bias = nn.Parameter(linear.bias.detach().to(torch.bfloat16, copy=True), requires_grad=False)
        return q

    def dequantize(self, dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
        """The weight (out, in) that the codes stand for."""
        return mxfp8_dequantize(self.weight_codes, self.weight_scales, dtype)

    @property
    def pair(self) -> tuple[torch.Tensor, torch.Tensor]:
        """(weight_codes, weight_scales), as the products over several weights take them."""
        return self.weight_codes, self.weight_scales

    def forward(self, x: torch.Tensor | tuple[torch.Tensor, torch.Tensor], residual: torch.Tensor | None = None, *,
                out: torch.Tensor | None = None) -> torch.Tensor:
        return matmul_mxfp8(x, self.pair, self.bias, residual, out=out)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


QUANTIZED_LINEARS = (CudaLinearMXFP4, CudaLinearMXFP8)


def norm_to_eight_bits(x: torch.Tensor, norm: CudaRMSNorm | None) -> torch.Tensor | tuple[torch.Tensor, torch.Tensor]:
    """What a projection of eight-bit weights takes: the rows normalised and in eight bits by one launch, or x where
    there is no norm."""
    if norm is None:
        return x
    if x.dtype != torch.bfloat16:
        raise TypeError(f"eight-bit linear layers take bfloat16 rows, got {x.dtype}")
    return add_rmsnorm_mxfp8(x, None, norm.weight, norm.eps)[1:]
