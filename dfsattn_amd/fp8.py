"""Linear layers on 8-bit operands.

``Fp8Linear`` holds a layer's weight as ``ops.quantize_fp8`` leaves it (e4m3
codes with a power of two for each 128 channels of a row) and runs
``ops.linear_fp8``; its input is quantised within the call, or comes quantised
from the operator before (``DiTBlock`` runs its feed-forward products that way:
the norm before them and the first product leave their results as operands).
``install_fp8`` puts such layers into a ``WanLikeDiT``.

A weight takes half the memory; a code is off by 2^-4 of its value at most, or, for
values below 2^-6 of their block's scale (whose largest value is at most 448 of it),
by 2^-10 of the scale, so layers differ from their 16-bit originals by a few percent
of an output's size.
"""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from . import ops


class Fp8Linear(nn.Module):
    """x @ weight.T + bias on 8-bit operands, in x's type (bf16 or f16). Codes and
    scales are kept as bytes, so that casts of the module leave them alone;
    ``dtype``, that of the layer it stands for, follows them."""

    def __init__(self, codes: torch.Tensor, scales: torch.Tensor, bias: Optional[torch.Tensor] = None,
                 dtype: torch.dtype = torch.bfloat16):
        super().__init__()
        self.out_features, self.in_features = codes.shape
        self.register_buffer("codes", codes.view(torch.uint8))
        self.register_buffer("scales", scales.view(torch.uint8))
        self.register_buffer("bias", bias)
        self.register_buffer("_like", torch.empty(0, dtype=dtype, device=codes.device), persistent=False)

    @property
    def dtype(self) -> torch.dtype:
        return self._like.dtype

    @classmethod
    @torch.no_grad()
    def from_linear(cls, layer: nn.Linear) -> "Fp8Linear":
        """Of an nn.Linear with bf16 or f16 weights on the GPU."""
        bias = None if layer.bias is None else layer.bias.detach().clone()
        return cls(*ops.quantize_fp8(layer.weight.detach()), bias, layer.weight.dtype)

    def forward(self, x: torch.Tensor, x_scales: Optional[torch.Tensor] = None, **options):
        """``options``: those of ``ops.linear_fp8``."""
        return ops.linear_fp8(x, self.codes.view(ops.E4M3), self.scales.view(ops.E8M0), x_scales, self.bias, **options)

    def extra_repr(self) -> str:
        return f"in_features={self.in_features}, out_features={self.out_features}, bias={self.bias is not None}"


def install_fp8(model, attention: bool = True, ffn: bool = True) -> int:
    """Puts ``Fp8Linear`` layers in the place of the projections of every
    attention and of the feed-forward products of a WanLikeDiT on the GPU; returns
    how many."""
    count = 0

    def replace(holder, name) -> None:
        nonlocal count
        layer = holder[name] if isinstance(name, int) else getattr(holder, name)
        if isinstance(layer, nn.Linear):
            new = Fp8Linear.from_linear(layer)
            if isinstance(name, int):
                holder[name] = new
            else:
                setattr(holder, name, new)
            count += 1

    for block in model.blocks:
        if attention:
            for attn in (block.attn1, block.attn2):
                for name in ("to_q", "to_k", "to_v"):
                    replace(attn, name)
                replace(attn.to_out, 0)
        if ffn:
            replace(block.ffn, 0)
            replace(block.ffn, 2)
    return count
