"""The {P2, I~} cache in pages of 8-bit values: rows appended and read back, and the decode step over them.

A sequence's rows form blocks of 64. A whole block of a head is held in 8 bits, P2 and I~ apart: one fp32 scale,
max|x| / 448, and an e4m3 code per value (include/mote_relation.h has every rounding point), half of bf16's bytes.
It lies in a page of a pool that the sequence's row of the table names, and is never written again, so sequences
may share it (`pages_fork`). The newest rows, fewer than 64, stay in the model's dtype in the sequence's tail: every
row is rounded once, and with its whole block known. A block that holds a NaN or an infinity reads back as NaN.

The table's pages are the caller's: `pages_reserve` gives them out, or RelationArena8 does. A block that has no page
(a number outside the pool) when it becomes whole is lost, and reads back as NaN.

Nothing here has a derivative: calls with rows, parameters or outputs that require a gradient are refused under
grad mode, those with dual tensors always.
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Tuple, Union

import torch

from . import _lib as L

PAGE = 64  # rows of a block


class Cache8(NamedTuple):
    """One layer's rows. Pages of P2 codes uint8 [P, H, C, 64, 16] (C = ceil(D / 16) chunks of dims) and of I~ codes
    uint8 [P, H, 16 C, 64], with their scales fp32 [P, H]; tails [B, H, 64, D]; the table int32 [B, blocks]. Views
    of larger stores are taken as long as a page, a sequence's tail and a row of the table lie back to back."""

    p2: torch.Tensor
    p2_scale: torch.Tensor
    info: torch.Tensor
    info_scale: torch.Tensor
    p2_tail: torch.Tensor
    info_tail: torch.Tensor
    table: torch.Tensor


def chunks(d_head: int) -> int:
    if not 0 < d_head <= 128 or d_head % 8:
        raise ValueError(f"head dim {d_head} unsupported (need 8 <= D <= 128, D % 8 == 0)")
    return -(-d_head // 16)


def cache8_zeros(B: int, H: int, pages: int, max_rows: int, d_head: int, device, dtype: torch.dtype = torch.bfloat16) -> Cache8:
    """A pool whose pages are all zero, empty tails and a table without pages, for up to `max_rows` rows a sequence."""
    if pages < 1 or max_rows < 1:
        raise ValueError(f"a cache of {pages} pages for {max_rows} rows")
    C = chunks(d_head)
    mk = lambda *s: torch.zeros(*s, device=device, dtype=torch.uint8)
    scale = lambda: torch.zeros(pages, H, device=device, dtype=torch.float32)
    tail = lambda: torch.zeros(B, H, PAGE, d_head, device=device, dtype=dtype)
    table = torch.full((B, -(-max_rows // PAGE)), -1, device=device, dtype=torch.int32)
    return Cache8(mk(pages, H, C, PAGE, 16), scale(), mk(pages, H, 16 * C, PAGE), scale(), tail(), tail(), table)


def _number(x) -> Tuple[int, Optional[torch.Tensor]]:
    return (0, x) if torch.is_tensor(x) else (int(x), None)


def cache8_write(cache: Cache8, p2: torch.Tensor, info: torch.Tensor, start: Union[int, torch.Tensor] = 0,
                 lens: Optional[torch.Tensor] = None) -> None:
    """New rows p2 / info [B, H, T, D] (the tails' dtype, any strides) behind the `start` rows that a sequence holds.

    start: an int (start + T rows have to fit the table), or int64 [B] on the device, a number per sequence; a
        sequence whose number the table does not reach stores nothing, rows past the table's end are dropped.
    lens: int64 [B] on the device: sequence b takes its first lens[b] rows; the rest of a padded batch is not read."""
    n, dev = _number(start)
    L.native().cache8_write(list(cache), p2, info, n, dev, lens)


def cache8_read(cache: Cache8, held: Union[int, torch.Tensor], start: Union[int, torch.Tensor] = 0, rows: Optional[int] = None,
                dtype: Optional[torch.dtype] = None, out: Optional[Tuple[torch.Tensor, torch.Tensor]] = None
                ) -> Tuple[torch.Tensor, torch.Tensor]:
    """(P2, I~) rows start .. start + rows as [B, H, rows, D] in `dtype` (the tails' by default), each value rounded once.

    held: how many rows the sequences hold, an int or int64 [B] on the device: it says which block is the tail's.
        Positions that a sequence does not hold read as zeros.
    start: an int, or int64 [B] on the device.
    rows: all that are held from an int start on by default (with `held` an int).
    out: two views to write instead of new tensors (their dtype counts; any strides of whole 16-byte chunks), every
        row at a place of its own and none in the cache."""
    h, hdev = _number(held)
    n, dev = _number(start)
    if rows is None:
        if dev is not None or hdev is not None:
            raise ValueError("cache8_read: device positions need a number of rows")
        rows = max(h - n, 0)
    o2, oi = out if out is not None else (None, None)
    dtype = cache.p2_tail.dtype if dtype is None else dtype
    return L.native().cache8_read(list(cache), h, hdev, n, dev, rows, dtype, o2, oi)


def decode8_workspace(B: int, H: int, d_head: int, max_rows: int, device) -> torch.Tensor:
    """A workspace for `relation_decode8` at these sizes (`max_rows`: 64 times the table's width): completion counters
    and per-split partials, zeroed here once; every call leaves the counters at zero again. Calls whose workspace has
    as many bytes may share it one after the other (the layers of a step, captured graphs that are replayed in turn);
    they must not overlap. It is passed whole: a part of one is no workspace for smaller sizes."""
    a = L.Decode8Args()
    a.B, a.H, a.D, a.cache.blocks = B, H, d_head, -(-max_rows // PAGE)
    with L.device_of(device):
        n = int(L.lib().mote_relation_decode8_workspace(a))
    return torch.zeros(max(n, 16), device=device, dtype=torch.uint8)


def relation_decode8(p1: torch.Tensor, p2: torch.Tensor, info: torch.Tensor, S: torch.Tensor, cache: Cache8,
                     lam: torch.Tensor, tau_s: float = 2.0, inv_freq: Optional[torch.Tensor] = None,
                     theta: Optional[torch.Tensor] = None, layer_idx: int = 0, advance: bool = False,
                     workspace: Optional[torch.Tensor] = None, y: Optional[torch.Tensor] = None,
                     g: Optional[torch.Tensor] = None, xm: Optional[torch.Tensor] = None,
                     run: Optional[torch.Tensor] = None, rope_f32: bool = False) -> Tuple[torch.Tensor, torch.Tensor]:
    """One decode step for B sequences over a paged cache in 8 bits: `relation_decode` (its arguments, its workspace
    rule, its predicate) with the rows of whole blocks at their 8-bit values and the tail's as they are. The new
    chunk takes part as it is and becomes row S: of the tail, or with it, when it makes the block whole, of a page.

    p1, p2, info: raw projections of the new chunk, [B, H, dh] (head stride dh, any batch stride), in the tails'
        dtype (bf16 or fp32).
    S: int64 [B] device positions. S[b] outside [0, 64 blocks): NaN in y[b] and g[b], nothing stored. A whole block
        without a page: NaN in y[b] and g[b].
    lam, inv_freq, theta: a layer's own parameters are taken under torch.no_grad() (they have no backward here).
    Returns (y [B, H, dh], g [B, H] fp32)."""
    return L.native().relation_decode8(p1, p2, info, S, list(cache), lam, tau_s, inv_freq, theta, layer_idx, advance, workspace,
                                       y, g, xm, run, rope_f32)
