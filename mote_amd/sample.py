"""The next token of every sequence from its logits and one random number: temperature, top-k, top-p and min-p.

The draw at the end of a decode step (GraphDecoder._sample, mote/infer/graph.py:243), for any number of sequences with
settings of their own: one launch up to 8192 logits a row, three beyond. It can be captured: random numbers and settings
may be device tensors that change between replays.

Tokens stand in the order of their logits, the lowest index first among equal ones, with the weights
w = exp((x - max) / temperature). Kept are the first `top_k`; of these the shortest run from the first on that holds at
least `top_p` of their weight; of those the ones with w >= min_p. The first is always kept. The token is the first in
that order whose running weight exceeds u times the weight kept: equal u give equal tokens, whatever the batch.
"""

from __future__ import annotations

from typing import Optional, Union

import torch

from . import _lib as L


def sample_tokens(logits: torch.Tensor, u: torch.Tensor, temperature: Union[float, torch.Tensor] = 1.0,
                  top_k: Union[int, torch.Tensor] = 0, top_p: Union[float, torch.Tensor] = 1.0,
                  min_p: Union[float, torch.Tensor] = 0.0, out: Optional[torch.Tensor] = None,
                  run: Optional[torch.Tensor] = None) -> torch.Tensor:
    """Token ids int64 [B] for logits [B, V] (bf16 or fp32, V <= 2^20) and u fp32 [B] in [0, 1).

    temperature, top_p, min_p: a number, or fp32 [B] on the device; top_k: a number, or int64 [B]. A temperature of 0
        and a min_p above 1 take the first token; top_k 0, top_p 1 and min_p 0 leave all.
    out: int64 [B] to write instead of a new tensor, apart from every operand.
    run: optional one-element bool / uint8 device tensor: when it holds 0 nothing is written.
    A row without a logit above -inf, with a NaN, or whose u or a setting is NaN gives -1. There is no derivative:
    logits that require a gradient are refused under grad mode, dual tensors always."""
    return L.native().sample_tokens(logits, u, temperature, top_k, top_p, min_p, out, run)
