"""The pages of the cache in 8 bits (`cache8`): given out, shared, given back and moved, on the device in stream order.

    table  int32 [B, blocks]   the page of block j (64 rows) of sequence b, -1 where there is none
    refs   int32 [pages]       the entries that name a page (0: free)

A page is written once, when its block becomes whole, and only read afterwards, so several sequences may name it:
a fork shares the whole blocks of a prompt and copies its newest rows alone. Pages go out from the lowest free number
on, in the order of (sequence, block), so every call's result is a function of its operands; counts go by integer
atomics. Sequences are named on the host; nothing here waits for the device, and every call can be captured (its
lists are then part of the graph).
"""

from __future__ import annotations

from typing import NamedTuple, Optional, Sequence, Tuple, Union

import torch

from . import _lib as L


class PagePool(NamedTuple):
    """The pages of a whole arena: codes uint8 [planes, pages, bytes of a page], scales fp32 [planes, pages, H], and refs
    int32 [pages]. A plane is P2 or I~ of one layer."""

    codes: torch.Tensor
    scales: torch.Tensor
    refs: torch.Tensor


def pages_free(refs: torch.Tensor, table: torch.Tensor, seqs: Sequence[int]) -> None:
    """The sequences give their pages back and have none; each is named once."""
    L.native().pages_free(refs, table, list(seqs))


def pages_fork(refs: torch.Tensor, table: torch.Tensor, S: torch.Tensor, src: int, dst: Sequence[int],
               tails: Optional[torch.Tensor] = None) -> None:
    """Each of the sequences `dst` gives its pages back and continues `src`: it shares the pages of src's S[src] // 64
    whole blocks, and S[dst] = S[src].

    S: int64 [B], the rows that each sequence holds. (Pages that src has reserved behind them stay its own: the
        next blocks of dst need pages of their own, which `pages_reserve` gives.)
    tails: [planes, B, H, 64, D] (bf16 or fp32): the S[src] % 64 newest rows of src are copied in every plane."""
    L.native().pages_fork(refs, table, S, int(src), list(dst), tails)


def pages_reserve(refs: torch.Tensor, table: torch.Tensor, rows: Union[int, torch.Tensor]) -> torch.Tensor:
    """Every sequence gets pages for the rows // 64 whole blocks of its first `rows` rows where it has none yet. rows:
    one number, or int64 [B] on the device. Returns how many entries the pool had no page for (int32 [1], on the
    device): those stay -1. The whole table is walked, 1 to 2 us for every 1024 entries: a call for a token that
    completes no block is better not made."""
    n, dev = (0, rows) if torch.is_tensor(rows) else (int(rows), None)
    return L.native().pages_reserve(refs, table, n, dev)


def pages_compact(pool: PagePool, table: torch.Tensor, into: PagePool) -> Tuple[torch.Tensor, torch.Tensor]:
    """The pages in use copied into another pool (smaller, larger or as large), in the order of their numbers from 0
    on; its counts are set, its other pages left as they were. Returns (the table in the new numbers, how many
    entries the new pool had no room for, int32 [1]): those are -1."""
    return L.native().pages_compact(list(pool), table, list(into))
