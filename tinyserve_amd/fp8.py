"""Linears over FP8 checkpoints: e4m3 weights with a float32 scale per block of 128 x 128.

``FP8Linear`` stands where a model has an ``nn.Linear`` whose checkpoint holds ``weight``
(float8_e4m3fn [out, in]) and ``weight_scale_inv`` (float32 [ceil(out / 128), ceil(in / 128)]): the
activations are quantised per token and 128 columns inside the call (ops.fp8_quantize's rule), the
product runs on the FP8 matrix cores. ``replace_linear_with_fp8`` swaps a model's linears as
``ggml_linear.replace_linear_with_ggml`` does for GGUF weights.
"""
from __future__ import annotations

import logging

import torch
import torch.nn as nn

from . import ops

logger = logging.getLogger(__name__)


class FormatModule(nn.Module):
    """A module some of whose parameters (``_is_format``: codes and their scales) keep their types when the model
    around it is cast (``.to(dtype)``, ``.half()``, ``.type(dtype)``): they are a format, not values of some precision."""

    def _is_format(self, name: str, p: torch.Tensor) -> bool:
        raise NotImplementedError

    def _apply(self, fn, recurse=True):
        fixed = {id(p) for n, p in self._parameters.items() if p is not None and self._is_format(n, p)}

        def keep(t):
            if id(t) not in fixed:
                return fn(t)
            raw = t.detach().view(torch.uint8 if t.element_size() == 1 else torch.int32)  # casts leave integers alone
            out = fn(raw)
            return (out if out.dtype == raw.dtype else raw.to(out.device)).view(t.dtype)

        return super()._apply(keep, recurse)


class FP8Module(FormatModule):
    """FormatModule for e4m3 parameters and block scales (``*_scale_inv``)."""

    def _is_format(self, name: str, p: torch.Tensor) -> bool:
        return p.dtype == torch.float8_e4m3fn or name.endswith("_scale_inv")


class FP8Linear(FP8Module):
    """y = deq(fp8_quantize(x)) @ deq(weight)^T + bias, in x's dtype; in_features a multiple of 16. Casting
    the model leaves codes and scales as they are."""

    def __init__(self, weight: torch.Tensor, weight_scale_inv: torch.Tensor, bias: torch.Tensor | None = None,
                 device: torch.device | str = "cuda"):
        super().__init__()
        if weight.dtype != torch.float8_e4m3fn or weight.dim() != 2:
            raise ValueError(f"weight must be float8_e4m3fn [out, in], got {weight.dtype} {tuple(weight.shape)}")
        self.out_features, self.in_features = weight.shape
        if self.in_features % 16:
            raise ValueError(f"in_features ({self.in_features}) must be a multiple of 16")
        want = tuple(-(-n // ops.FP8_BLOCK) for n in weight.shape)
        if tuple(weight_scale_inv.shape) != want:
            raise ValueError(f"weight_scale_inv must be {list(want)}, got {list(weight_scale_inv.shape)}")
        self.weight = nn.Parameter(weight.to(device), requires_grad=False)
        self.weight_scale_inv = nn.Parameter(weight_scale_inv.to(device=device, dtype=torch.float32), requires_grad=False)
        self.bias = None if bias is None else nn.Parameter(bias.detach().to(device), requires_grad=False)

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        y = ops.fp8_linear(x, self.weight, self.weight_scale_inv, self.bias)
        return y if x.dim() == 2 else y.view(*x.shape[:-1], self.out_features)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def replace_linears(model: nn.Module, weights: dict[str, tuple[torch.Tensor, torch.Tensor]], make) -> int:
    """Replace ``nn.Linear`` modules named in ``weights`` (path -> (weight, scales)) by ``make(weight, scales, bias)``,
    keeping their biases; returns the number replaced. Paths that do not resolve to an ``nn.Linear`` are skipped;
    meta-device biases are dropped."""
    replaced = 0
    for name, (weight, scales) in weights.items():
        path, _, attr = name.rpartition(".")
        try:
            parent = model.get_submodule(path)
        except AttributeError:
            continue
        old = getattr(parent, attr, None)
        if not isinstance(old, nn.Linear):
            continue
        bias = old.bias if old.bias is not None and old.bias.device.type != "meta" else None
        setattr(parent, attr, make(weight, scales, bias))
        replaced += 1
    return replaced


def replace_linear_with_fp8(model: nn.Module, weights: dict[str, tuple[torch.Tensor, torch.Tensor]],
                            device: torch.device | str = "cuda") -> int:
    """Replace ``nn.Linear`` modules named in ``weights`` (path -> (weight, weight_scale_inv)) by
    ``FP8Linear`` (replace_linears)."""
    replaced = replace_linears(model, weights, lambda w, s, b: FP8Linear(w, s, b, device))
    logger.info("FP8Linear now backs %d linear layer(s)", replaced)
    return replaced
