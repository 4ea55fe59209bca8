"""Linear layers with their weight in MXFP4 (no reference counterpart; the reference's weights are bf16 or fp32)."""
from __future__ import annotations

import torch
from torch import nn

from ..kernels import matmul_mxfp4, mxfp4_dequantize, mxfp4_quantize
from ..kernels.mxfp4 import MX_BLOCK
from .linear import CudaLinear
from .mlp import CudaSwiGLUMLP
from .text_decoder import CudaTextDecoderLayer


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

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None, *,
                out: torch.Tensor | None = None) -> torch.Tensor:
        return matmul_mxfp4(x, self.weight_codes, self.weight_scales, self.bias, residual, out=out)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def quantize_text_linears(model: nn.Module, *, lm_head: bool = False) -> list[str]:
    """Replace the linear layers of every CudaTextDecoderLayer in `model` (q/k/v/o and the dense MLP's gate/up/down;
    with lm_head=True also `model.lm_head`) by CudaLinearMXFP4, in place. Returns the names replaced. Experts, norms,
    embeddings and the vision tower keep their type, as do layers whose input size is no multiple of 32. For bf16
    inference: run under torch.no_grad(); the new layers have no backward."""
    done = []

    def swap(parent: nn.Module, name: str, path: str) -> None:
        old = getattr(parent, name, None)
        if type(old) is CudaLinear and old.in_features % MX_BLOCK == 0:
            setattr(parent, name, CudaLinearMXFP4.from_linear(old))
            done.append(f"{path}.{name}" if path else name)

    for path, layer in list(model.named_modules()):
        if not isinstance(layer, CudaTextDecoderLayer):
            continue
        at = f"{path}." if path else ""
        for name in ("q_proj", "k_proj", "v_proj", "o_proj"):
            swap(layer.self_attn, name, f"{at}self_attn")
        if isinstance(layer.mlp, CudaSwiGLUMLP):
            for name in ("gate_proj", "up_proj", "down_proj"):
                swap(layer.mlp, name, f"{at}mlp")
    if lm_head:
        swap(model, "lm_head", "")
    return done
