"""Projections in 8-bit integers: one fp32 scale per token of x and per output channel of W.

    w8 = int8_weight(linear.weight)     # once, and after every change of the weight
    y = int8_linear(x, w8)              # F.linear(x, weight), both operands rounded to 8 bits

A row's scale is max|row| / 127 and its codes are rint(x (127 / max|row|)); the products are summed exactly in
32-bit integers, so y = (acc sx) sw depends on nothing but the codes and scales (no order of summation, no
split). A token with a NaN or an infinity gives a row of NaN. Serving only: there is no derivative, and calls
with tensors that require a gradient are refused under grad mode, those with dual tensors always (`int8_weight`
takes a parameter as the constant that it is at the time).
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple

import torch

from . import _lib as L

FEW_ROWS, FEW_WIDTH = 64, 4096  # most tokens and inputs of a call with the decode step's predicate or exchange mass


class Int8Weight(NamedTuple):
    """A weight [N, K] in 8 bits: codes int8 [N, K rounded up to 128], scales fp32 [N], and K."""

    q: torch.Tensor
    scale: torch.Tensor
    in_features: int


def quantize_rows(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """The rows of x [M, K] (bf16 or fp32) in 8 bits: (codes int8 [M, K rounded up to 128], zeros past K;
    scales fp32 [M])."""
    return L.native().quantize_rows(x)


def int8_weight(w: torch.Tensor) -> Int8Weight:
    """A projection's weight [N, K] (bf16 or fp32) with a scale per output channel."""
    q, scale = quantize_rows(w.detach())
    return Int8Weight(q, scale, w.shape[1])


def int8_linear(x: torch.Tensor, w: Int8Weight, out: Optional[torch.Tensor] = None, run: Optional[torch.Tensor] = None,
                g: Optional[torch.Tensor] = None, xm: Optional[torch.Tensor] = None) -> torch.Tensor:
    """y [..., N] = x [..., K] W^T in x's dtype (bf16 or fp32), x quantised per token in the call.

    Up to 64 tokens of K <= 4096 may take what `skinny_linear` takes: `run` (a device flag; 0 leaves `out`
    untouched), g (fp32 [M, H], contiguous) and xm (fp32 [M], the mean of g over the heads). Such calls are one
    launch, as are those of up to 16 tokens and those of up to 64 that few workgroups hold; others are two."""
    return L.native().int8_linear(x, w.q, w.scale, w.in_features, out, run, g, xm)
