"""Plain forms of the quantised formats, on the CPU in 64 bits with the formats' own rounding points.

4 bits: groups of 32 values share a bf16 scale, codes are e2m1. 8 bits: a row shares an fp32 scale, and in the
paged cache a block of 64 rows of a head does, whose codes are e4m3. Every 32-bit quotient and product of the
definition is taken in fp64 and rounded (a quotient or product of two fp32 values is rounded correctly that way), so
codes and scales are the definition's bit for bit.
"""

from __future__ import annotations

from typing import Tuple

import torch

GROUP = 32
MAGNITUDES = torch.tensor([0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0], dtype=torch.float64)


def _f32(x: torch.Tensor) -> torch.Tensor:
    return x.to(torch.float32).to(torch.float64)


def nearest_code(t: torch.Tensor) -> torch.Tensor:
    """The e2m1 code (0..7) of each fp64 magnitude: the nearest value, ties to the even code, 6 at most."""
    d = (t.clamp(max=6.0)[..., None] - MAGNITUDES).abs()
    best = d.amin(-1, keepdim=True)
    cand = d == best                                  # one code, or two neighbours at a tie
    code = torch.arange(8).expand_as(cand)
    even = torch.where(cand & (code % 2 == 0), code, torch.full_like(code, 99)).amin(-1)
    lone = torch.where(cand, code, torch.full_like(code, 99)).amin(-1)
    return torch.where(cand.sum(-1) == 2, even, lone)


def encode4(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows [..., D] -> (signed codes as values of MAGNITUDES [..., D] fp64, scales bf16 [..., G])."""
    x = x.double()
    D = x.shape[-1]
    G = -(-D // GROUP)
    vals, scales = torch.zeros_like(x), torch.zeros(*x.shape[:-1], G, dtype=torch.bfloat16)
    for g in range(G):
        part = x[..., g * GROUP: (g + 1) * GROUP]
        finite = torch.isfinite(part).all(-1)
        top = torch.where(finite[..., None], part, 0.0).abs().amax(-1)
        s = _f32(top / 6.0).float().bfloat16()
        s = torch.where(s.float() < 2.0 ** -126, torch.zeros_like(s), s)
        live = finite & (s > 0)
        inv = _f32(1.0 / torch.where(live, s.double(), 1.0))
        t = _f32(torch.where(live[..., None], part, 0.0) * inv[..., None])
        vals[..., g * GROUP: (g + 1) * GROUP] = torch.sign(t) * MAGNITUDES[nearest_code(t.abs())]
        scales[..., g] = torch.where(finite, s, torch.full_like(s, float("nan")))
    return vals, scales


def values4(vals: torch.Tensor, scales: torch.Tensor) -> torch.Tensor:
    """fp64 values of encoded rows."""
    D = vals.shape[-1]
    return vals * scales.double().repeat_interleave(GROUP, -1)[..., :D]


def unpack_codes(codes: torch.Tensor, D: int) -> torch.Tensor:
    """Stored bytes [..., 16 G] -> signed code values [..., D] fp64."""
    nib = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)[..., :D].long()
    return torch.where(nib >= 8, -1.0, 1.0).double() * MAGNITUDES[nib % 8]


def nearest_e4m3(t: torch.Tensor) -> torch.Tensor:
    """The e4m3 value nearest to each fp64 value (ties to the even mantissa, 448 at most)."""
    n = torch.arange(127)
    mag = torch.where(n < 8, (n % 8).double() * 2.0 ** -9, (1.0 + (n % 8).double() / 8.0) * torch.pow(2.0, (n // 8 - 7).double()))
    a = t.abs().clamp(max=448.0)
    hi = torch.searchsorted(mag, a.contiguous()).clamp(max=126)   # the first value >= a
    lo = (hi - 1).clamp(min=0)
    up, down = mag[hi] - a, a - mag[lo]
    pick = torch.where(up < down, hi, torch.where(down < up, lo, torch.where(hi % 2 == 0, hi, lo)))
    return torch.where(t < 0, -1.0, 1.0).double() * mag[pick]


def block8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Blocks [..., 64, D] -> (codes as values fp64, scales fp64 [...], NaN for blocks with a NaN or an infinity)."""
    x = x.double()
    finite = torch.isfinite(x).flatten(-2).all(-1)
    top = torch.where(finite[..., None, None], x, 0.0).abs().amax((-1, -2))
    live = finite & (top >= 2.0 ** -112)
    safe = torch.where(live, top, 1.0)
    t = _f32(torch.where(live[..., None, None], x, 0.0) * _f32(448.0 / safe)[..., None, None])
    scale = torch.where(live, _f32(safe / 448.0), 0.0)
    return nearest_e4m3(t), torch.where(finite, scale, float("nan"))


def values8(x: torch.Tensor) -> torch.Tensor:
    """fp64 values that blocks [..., 64, D] have in 8 bits (32-bit numbers)."""
    codes, scale = block8(x)
    return _f32(codes * scale[..., None, None])


def held8(rows: torch.Tensor) -> torch.Tensor:
    """fp64 values of the rows [H, n, D] of one sequence as the paged cache holds them: whole blocks in 8 bits, the
    rest as it is."""
    n = rows.shape[1] // 64 * 64
    whole = values8(rows[:, :n].unflatten(1, (-1, 64))).flatten(1, 2) if n else rows[:, :0].double()
    return torch.cat([whole, rows[:, n:].double()], 1)


def quantize8(x: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
    """Rows [M, K] -> (codes fp64 [M, K], scales fp64 [M], NaN for rows with a NaN or an infinity)."""
    x = x.double()
    finite = torch.isfinite(x).all(-1)
    top = torch.where(finite[:, None], x, 0.0).abs().amax(-1)
    live = finite & (top >= 2.0 ** -120)
    safe = torch.where(live, top, 1.0)
    q = torch.round(_f32(torch.where(live[:, None], x, 0.0) * _f32(127.0 / safe)[:, None]))
    scale = torch.where(live, _f32(safe / 127.0), 0.0)
    return q, torch.where(finite, scale, float("nan"))


def int8_linear_ref(x: torch.Tensor, w: torch.Tensor) -> torch.Tensor:
    """y [M, N] in fp64 of the rows and channels rounded to 8 bits."""
    q, sx = quantize8(x)
    wq, sw = quantize8(w)
    return (q @ wq.t()) * sx[:, None] * sw
