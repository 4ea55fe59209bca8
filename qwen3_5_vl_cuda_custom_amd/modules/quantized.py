"""Replacing a model's linear layers by their four-bit or eight-bit form (no reference counterpart)."""
from __future__ import annotations

from torch import nn

from .linear import CudaLinear
from .linear_mxfp4 import CudaLinearMXFP4
from .linear_mxfp8 import CudaLinearMXFP8
from .mlp import CudaSwiGLUMLP
from .text_decoder import CudaTextDecoderLayer

_FORMATS = {"mxfp4": CudaLinearMXFP4, "mxfp8": CudaLinearMXFP8}


def quantize_text_linears(model: nn.Module, *, lm_head: bool = False, weight_format: str = "mxfp4") -> list[str]:
    """Replace the linear layers of every CudaTextDecoderLayer in `model` (q/k/v/o and the dense MLP's gate/up/down;
    with lm_head=True also `model.lm_head`) by CudaLinearMXFP4, or with weight_format="mxfp8" by CudaLinearMXFP8 (whose
    products take their inputs in eight bits too), in place. Returns the names replaced. Experts, norms, embeddings and
    the vision tower keep their type, as do layers whose input size is no multiple of 32. For bf16 inference: run under
    torch.no_grad(); the new layers have no backward."""
    if weight_format not in _FORMATS:
        raise ValueError(f"quantize_text_linears: weight_format must be 'mxfp4' or 'mxfp8', got {weight_format!r}")
    kind = _FORMATS[weight_format]
    done = []

    def swap(parent: nn.Module, name: str, path: str) -> None:
        old = getattr(parent, name, None)
        if type(old) is CudaLinear and old.in_features % 32 == 0:  # either format's blocks
            setattr(parent, name, kind.from_linear(old))
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
