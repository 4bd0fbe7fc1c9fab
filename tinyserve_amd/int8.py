"""Linears over int8 checkpoints: int8 weights with a float32 scale per row (output channel).

``Int8Linear`` stands where a model has an ``nn.Linear`` whose checkpoint holds ``weight`` (int8 [out, in]) and
``weight_scale`` ([out, 1] or [out]): the activations are quantised per token inside the call (ops.int8_quantize's
rule), the product runs on the int8 matrix cores. ``replace_linear_with_int8`` swaps a model's linears as
``fp8.replace_linear_with_fp8`` does for FP8 weights.
"""
from __future__ import annotations

import logging

import torch
import torch.nn as nn

from . import ops
from .fp8 import FormatModule, replace_linears

logger = logging.getLogger(__name__)


class Int8Module(FormatModule):
    """FormatModule for int8 parameters and their scales (``*_scale``)."""

    def _is_format(self, name: str, p: torch.Tensor) -> bool:
        return p.dtype == torch.int8 or name.endswith("_scale")


class Int8Linear(Int8Module):
    """y = deq(int8_quantize(x)) @ deq(weight)^T + bias, in x's dtype; in_features a multiple of 16, at most 131056.
    Casting the model leaves codes and scales as they are."""

    def __init__(self, weight: torch.Tensor, weight_scale: torch.Tensor, bias: torch.Tensor | None = None,
                 device: torch.device | str = "cuda"):
        super().__init__()
        if weight.dtype != torch.int8 or weight.dim() != 2:
            raise ValueError(f"weight must be int8 [out, in], got {weight.dtype} {tuple(weight.shape)}")
        self.out_features, self.in_features = weight.shape
        if self.in_features % 16 or self.in_features > ops.INT8_MAX_K:
            raise ValueError(f"in_features ({self.in_features}) must be a multiple of 16 of at most {ops.INT8_MAX_K}")
        if tuple(weight_scale.shape) not in ((self.out_features,), (self.out_features, 1)):
            raise ValueError(f"weight_scale must be [{self.out_features}, 1], got {list(weight_scale.shape)}")
        self.weight = nn.Parameter(weight.to(device), requires_grad=False)
        self.weight_scale = nn.Parameter(weight_scale.to(device=device, dtype=torch.float32).reshape(-1, 1), requires_grad=False)
        self.bias = None if bias is None else nn.Parameter(bias.detach().to(device), requires_grad=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = ops.int8_linear(x, self.weight, self.weight_scale, self.bias)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def replace_linear_with_int8(model: nn.Module, weights: dict[str, tuple[torch.Tensor, torch.Tensor]],
                             device: torch.device | str = "cuda") -> int:
    """Replace ``nn.Linear`` modules named in ``weights`` (path -> (weight, weight_scale)) by ``Int8Linear``
    (fp8.replace_linears)."""
    replaced = replace_linears(model, weights, lambda w, s, b: Int8Linear(w, s, b, device))
    logger.info("Int8Linear now backs %d linear layer(s)", replaced)
    return replaced
