"""The {P2, I~} cache held in 4 bits: rows written and read back, and the decode step over them.

A row of D values (a multiple of 8, at most 128) is G = ceil(D / 32) groups of 32; a group has one bf16
scale, max|x| / 6, and an e2m1 code per value (0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign; include/mote_relation.h
has every rounding point): 18 bytes a group, 3.6 times fewer than bf16. Scales follow the magnitude of their
own 32 values, so channels of unlike size and single outliers cost their own group only. A group that holds a
NaN or an infinity reads back as NaN.

Nothing here has a derivative: calls with rows, parameters or outputs that require a gradient are refused under
grad mode, those with dual tensors always.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib as L

GROUP = 32  # values that share a scale


class Cache4(NamedTuple):
    """One layer's rows: codes uint8 [B, H, capacity, 16 G] (two a byte) and scales bf16 [B, H, capacity, G].
    Views of larger stores are taken as long as the rows of a head lie back to back."""

    p2: torch.Tensor
    p2_scale: torch.Tensor
    info: torch.Tensor
    info_scale: torch.Tensor


def groups(d_head: int) -> int:
    if not 0 < d_head <= 128 or d_head % 8:
        raise ValueError(f"head dim {d_head} unsupported (need 8 <= D <= 128, D % 8 == 0)")
    return -(-d_head // GROUP)


def cache4_zeros(B: int, H: int, capacity: int, d_head: int, device) -> Cache4:
    """A cache whose rows are all zero."""
    G = groups(d_head)
    mk = lambda n, dt: torch.zeros(B, H, capacity, n, device=device, dtype=dt)
    return Cache4(mk(16 * G, torch.uint8), mk(G, torch.bfloat16), mk(16 * G, torch.uint8), mk(G, torch.bfloat16))


def _start(start) -> Tuple[int, Optional[torch.Tensor]]:
    return (0, start) if torch.is_tensor(start) else (int(start), None)


def cache4_write(cache: Cache4, p2: torch.Tensor, info: torch.Tensor, start: Union[int, torch.Tensor] = 0,
                 lens: Optional[torch.Tensor] = None) -> None:
    """Rows start + t of every sequence and head from p2 / info [B, H, T, D] (bf16 or fp32, any strides).

    start: an int (start + T rows have to fit), or int64 [B] on the device, a row per sequence; rows that a
        device position takes out of [0, capacity) are skipped.
    lens: int64 [B] on the device: sequence b writes its first lens[b] rows; the rest of a padded batch
        leaves the cache as it was."""
    n, dev = _start(start)
    L.native().cache4_write(*cache, p2, info, n, dev, lens)


def cache4_read(cache: Cache4, d_head: int, start: Union[int, torch.Tensor] = 0, rows: Optional[int] = None,
                dtype: torch.dtype = torch.bfloat16, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(P2, I~) rows start .. start + rows as [B, H, rows, d_head] in `dtype`, each value rounded once.

    start: an int, or int64 [B] on the device (rows that it takes out of [0, capacity) read as NaN).
    rows: all from an int start on by default.
    out: two views to write instead of new tensors (their dtype counts; any strides of whole 16-byte chunks),
        every row at a place of its own and none in the cache."""
    n, dev = _start(start)
    if rows is None:
        if dev is not None:
            raise ValueError("cache4_read: device positions need a number of rows")
        rows = cache.p2.shape[2] - n
    o2, oi = out if out is not None else (None, None)
    return L.native().cache4_read(*cache, d_head, n, dev, rows, dtype, o2, oi)


def decode4_workspace(B: int, H: int, d_head: int, capacity: int, device) -> torch.Tensor:
    """A workspace for `relation_decode4` at these sizes: completion counters and per-split partials, zeroed
    here once; every call leaves the counters at zero again. Calls whose workspace has as many bytes may share
    it one after the other (the layers of a step, captured graphs that are replayed in turn); they must not
    overlap. It is passed whole: a part of one is no workspace for smaller sizes."""
    a = L.Decode4Args()
    a.B, a.H, a.D, a.capacity = B, H, d_head, capacity
    with L.device_of(device):
        n = int(L.lib().mote_relation_decode4_workspace(a))
    return torch.zeros(max(n, 16), device=device, dtype=torch.uint8)


def relation_decode4(p1: torch.Tensor, p2: torch.Tensor, info: torch.Tensor, S: torch.Tensor, cache: Cache4,
                     lam: torch.Tensor, tau_s: float = 2.0, inv_freq: Optional[torch.Tensor] = None,
                     theta: Optional[torch.Tensor] = None, layer_idx: int = 0, advance: bool = False,
                     workspace: Optional[torch.Tensor] = None, y: Optional[torch.Tensor] = None,
                     g: Optional[torch.Tensor] = None, xm: Optional[torch.Tensor] = None,
                     run: Optional[torch.Tensor] = None, rope_f32: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One decode step for B sequences over a cache in 4 bits: `relation_decode` (its arguments, its
    workspace rule, its predicate) with the rows before S at their 4-bit values. The new chunk itself takes
    part as it is (the Self score and its share of y) and is then stored in 4 bits at row S.

    p1, p2, info: raw projections of the new chunk, [B, H, dh] (head stride dh, any batch stride), bf16 or
        fp32; the step's arithmetic rounds to that dtype where relation_decode rounds to the cache's.
    S: int64 [B] device positions. S[b] outside [0, capacity): NaN in y[b] and g[b], nothing stored.
    lam, inv_freq, theta: a layer's own parameters are taken under torch.no_grad() (they have no backward here).
    Returns (y [B, H, dh], g [B, H] fp32)."""
    return L.native().relation_decode4(p1, p2, info, S, *cache, lam, tau_s, inv_freq, theta, layer_idx, advance, workspace,
                                       y, g, xm, run, rope_f32)
