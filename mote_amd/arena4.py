"""The decode arena with its rows in 4 bits: RelationArena's interface over the format of `cache4`.

    arena = RelationArena4(n_layers, n_heads, capacity, d_head, device, torch.bfloat16, batch)
    state = ArenaState(arena)
    mixer(x, cache=state[layer])                       # a prompt window: rows stored in 4 bits
    RelationDecodeStep(mixer, arena, layer)(x, S)      # the decode step over them

`dtype` is the dtype that rows come in and are read back in (the model's); a row and head take 18 bytes per
32 dims instead of 64 in bf16. What a window or a step adds takes part in it as it is: a prompt window's own
rows are read unrounded by its own queries (ArenaLayer4.extend), as relation_decode4's new chunk is; the rows
before it are read at their 4-bit values. A prompt in two windows therefore differs from one window by the
rounding of the first window's rows, as it differs from the same arena in bf16.

Growth, residency (`owner`, `n_valid`, `claim`) and the rules of a batched arena are RelationArena's.
"""

from __future__ import annotations

from typing import Optional, Tuple

import torch

from .arena import ArenaLayer, ArenaState, RelationArena
from .cache4 import Cache4, cache4_read, cache4_write, groups


class RelationArena4(RelationArena):
    """`store` holds the codes, uint8 [n_layers, 2, batch, H, capacity, 16 G], `scales` bf16 [..., G]."""

    in_place = False
    kind = "cache4"

    def __init__(self, n_layers: int, n_heads: int, capacity: int, d_head: int, device, dtype=torch.bfloat16, batch: int = 1):
        if dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"an arena in 4 bits reads rows in bfloat16 or float32, not {dtype}")
        self.groups = groups(d_head)
        self.scales: Optional[torch.Tensor] = None
        super().__init__(n_layers, n_heads, capacity, d_head, device, dtype, batch)

    def _zeros(self, capacity: int) -> torch.Tensor:
        shape = (self.n_layers, 2, self.batch, self.n_heads, capacity)
        scales = torch.zeros((*shape, self.groups), device=self.device, dtype=torch.bfloat16)
        codes = torch.zeros((*shape, 16 * self.groups), device=self.device, dtype=torch.uint8)
        self.scales = scales  # once both are there: a growth that fails leaves the arena as it was
        return codes

    @property
    def bytes_per_chunk(self) -> int:
        return self.n_layers * 2 * self.batch * self.n_heads * self.groups * 18

    def nbytes(self) -> int:
        return self.store.numel() + 2 * self.scales.numel()

    def cache(self, layer: int) -> Cache4:
        """A layer's rows, as `cache4` and `relation_decode4` take them (views of the store)."""
        return Cache4(self.store[layer, 0], self.scales[layer, 0], self.store[layer, 1], self.scales[layer, 1])

    def layer(self, layer: int, state: ArenaState) -> "ArenaLayer4":
        return ArenaLayer4(self, layer, state)

    def _no_views(self):
        raise TypeError("an arena in 4 bits has no rows to view: use cache(layer), or a layer's views()")

    @property
    def buf(self):
        self._no_views()

    def p2(self, layer: int):
        self._no_views()

    def info(self, layer: int):
        self._no_views()

    def rows(self, c0: int, c1: int):
        self._no_views()

    def _reallocate(self, capacity: int) -> None:
        owner, live = self._resident
        if self.batch > 1:
            live = self.capacity  # no per-slot record: every slot's rows travel
        elif owner is None:
            live = 0
        codes, scales = self.store, self.scales
        if live == 0:
            self.store = self.scales = codes = scales = None  # the peak is the new size
            self._resident = (None, 0)
        with self._allocation_scope():
            self.store = self._zeros(capacity)
        if live:
            self.store[..., :live, :].copy_(codes[..., :live, :])
            self.scales[..., :live, :].copy_(scales[..., :live, :])
        self.generation += 1


class ArenaLayer4(ArenaLayer):
    """A layer of the state: `write` stores rows in 4 bits, `views` reads rows back."""

    __slots__ = ()

    def _cast(self, p2: torch.Tensor, info: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        return p2.to(self.arena.dtype), info.to(self.arena.dtype)

    def write(self, p2: torch.Tensor, info: torch.Tensor) -> None:
        """Store T new rows [n, n + T) of every sequence; p2 / info are [batch, H, T, dh]."""
        n, T = self.state.n, p2.shape[2]
        if n + T > self.arena.capacity:
            raise RuntimeError(f"arena overflow: rows up to {n + T} in a capacity of {self.arena.capacity}")
        cache4_write(self.arena.cache(self.layer), *self._cast(p2, info), n)

    def views(self, upto: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """(P2, I~) rows [0, upto) at their 4-bit values, as new [batch, H, upto, dh] tensors in the arena's dtype."""
        return cache4_read(self.arena.cache(self.layer), self.arena.d_head, 0, upto, dtype=self.arena.dtype)

    def extend(self, p2: torch.Tensor, info: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Store T new rows as `write` does; rows [0, n + T) for their own queries: the stored ones at their 4-bit
        values, the new ones as they are. Nothing of them is kept beside the arena's rows."""
        a, n, T = self.arena, self.state.n, p2.shape[2]
        new = self._cast(p2, info)
        self.write(*new)
        if n == 0:
            return new
        out = tuple(torch.empty(a.batch, a.n_heads, n + T, a.d_head, device=a.device, dtype=a.dtype) for _ in range(2))
        cache4_read(a.cache(self.layer), a.d_head, 0, n, out=tuple(t[:, :, :n] for t in out))
        for t, rows in zip(out, new):
            t[:, :, n:].copy_(rows)
        return out
