"""The decode arena in pages of 8-bit values: RelationArena's interface over the cache of `cache8` and its pages.

    arena = RelationArena8(n_layers, n_heads, capacity, d_head, device, torch.bfloat16, batch)
    state = ArenaState(arena)
    mixer(x, cache=state[layer])                       # a prompt window: whole blocks stored in 8 bits
    RelationDecodeStep(mixer, arena, layer)(x, S)      # the decode step over them
    arena.fork(0, [1, 2, 3], S)                        # three continuations of sequence 0 share its whole blocks
    arena.release([3])                                 # a sequence has ended: its pages are free again

One table row per sequence serves every layer. Without `pages` every sequence owns pages for its whole capacity, as in
RelationArena; with it the pool has that many pages for all, and `ensure` gives them out as the sequences grow (whole
blocks that are shared by a fork are held once). What a window or a step adds takes part in it as it is, and so do the
rows of a block that is not whole yet; the rows before are read at their 8-bit values.

Rows are appended. A state may go back to a whole block (n % 64 == 0) that no other sequence shares, and replace what
was behind it, but not into the middle of a block: a block is in 8 bits once it is whole. The arena sees windows and forks,
not the positions of steps, which are the caller's on the device: a window that begins inside a block that steps have gone
past is not refused and finds rows of a later block in the tail, and a step moved back to a block that forks share
writes into their page.
"""

from __future__ import annotations

from typing import List, Optional, Sequence, Tuple

import torch

from .arena import ArenaLayer, ArenaState, RelationArena
from .cache8 import PAGE, Cache8, cache8_read, cache8_write, chunks
from .pages import PagePool, pages_compact, pages_fork, pages_free, pages_reserve


class RelationArena8(RelationArena):
    """`store` holds the codes, uint8 [n_layers, 2, pages, H, 64 * 16 C], `scales` fp32 [n_layers, 2, pages, H], `tails`
    [n_layers, 2, batch, H, 64, dh] in `dtype`, `table` int32 [batch, capacity / 64], `refs` int32 [pages]."""

    in_place = False
    kind = "cache8"

    def __init__(self, n_layers: int, n_heads: int, capacity: int, d_head: int, device, dtype=torch.bfloat16, batch: int = 1,
                 pages: Optional[int] = None):
        if dtype not in (torch.bfloat16, torch.float32):
            raise TypeError(f"an arena in 8 bits reads rows in bfloat16 or float32, not {dtype}")
        if pages is not None and pages < 1:
            raise ValueError(f"an arena of {pages} pages")
        self.chunks = chunks(d_head)
        self.own = pages is None  # every sequence has pages for its whole capacity
        self._pages = pages
        self.scales = self.tails = self.table = self.refs = None
        self._views = (-1, {})
        super().__init__(n_layers, n_heads, capacity, d_head, device, dtype, batch)

    # ---- sizing ---------------------------------------------------------------------------------
    def _pool(self, pages: int) -> Tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
        mk = lambda *s, dt: torch.zeros(*s, device=self.device, dtype=dt)
        return (mk(self.n_layers, 2, pages, self.n_heads, 16 * self.chunks * PAGE, dt=torch.uint8),
                mk(self.n_layers, 2, pages, self.n_heads, dt=torch.float32), mk(pages, dt=torch.int32))

    def _zeros(self, capacity: int) -> torch.Tensor:
        """The first store: the pool, the tails and the table of `capacity` rows a sequence."""
        blocks = -(-int(capacity) // PAGE)
        pages = self.batch * blocks if self.own else self._pages
        store, self.scales, self.refs = self._pool(pages)
        self.tails = torch.zeros(self.n_layers, 2, self.batch, self.n_heads, PAGE, self.d_head, device=self.device, dtype=self.dtype)
        self.table = torch.full((self.batch, blocks), -1, device=self.device, dtype=torch.int32)
        self._rows: List[int] = [0] * self.batch    # rows that a sequence has pages for (host record)
        self._held: List[int] = [0] * self.n_layers  # rows that windows have stored, at least
        self._shared = 0  # rows in blocks that forks may share
        if self.own:
            self.table.copy_(torch.arange(pages, dtype=torch.int32).view(self.batch, blocks))
            self.refs.fill_(1)
            self._rows = [PAGE * blocks] * self.batch
        return store

    @property
    def capacity(self) -> int:
        return PAGE * self.table.shape[1]

    @property
    def pages(self) -> int:
        return self.store.shape[2]

    @property
    def bytes_per_chunk(self) -> int:
        """Bytes of one more row across every layer, kind, sequence and head (a whole block's, by its rows)."""
        return -(-self.n_layers * 2 * self.batch * self.n_heads * (16 * self.chunks * PAGE + 4) // PAGE)

    def nbytes(self) -> int:
        return sum(t.numel() * t.element_size() for t in (self.store, self.scales, self.tails, self.table, self.refs))

    # ---- views ----------------------------------------------------------------------------------
    def cache(self, layer: int) -> Cache8:
        """A layer's pool and tails with the table, as `cache8` and `relation_decode8` take them (views, the same ones until
        a tensor of the arena is reallocated)."""
        if self._views[0] != self.generation:
            self._views = (self.generation, {})
        c = self._views[1].get(layer)
        if c is None:
            c = self._views[1][layer] = self._cache(layer)
        return c

    def _cache(self, layer: int) -> Cache8:
        C, P, H = self.chunks, self.pages, self.n_heads
        return Cache8(self.store[layer, 0].view(P, H, C, PAGE, 16), self.scales[layer, 0],
                      self.store[layer, 1].view(P, H, 16 * C, PAGE), self.scales[layer, 1],
                      self.tails[layer, 0], self.tails[layer, 1], self.table)

    def layer(self, layer: int, state: ArenaState) -> "ArenaLayer8":
        return ArenaLayer8(self, layer, state)

    def _no_views(self):
        raise TypeError("an arena in 8 bits has no rows to view: use cache(layer), or a layer's views()")

    @property
    def buf(self):
        self._no_views()

    def p2(self, layer: int):
        self._no_views()

    def info(self, layer: int):
        self._no_views()

    def rows(self, c0: int, c1: int):
        self._no_views()

    # ---- growth and pages ------------------------------------------------------------------------
    def ensure(self, n_chunks: int, seqs: Optional[Sequence[int]] = None) -> bool:
        """Make room for `n_chunks` rows of every sequence, or of `seqs`: a table that reaches them, and pages for them. The
        others keep what they have: name those that run, and the ended ones hold no pages, shorter ones no more than they
        need. Returns True when a tensor of the arena was reallocated. Pages that are given out within the pool change the
        table in place, which captured graphs see; a call that gives none out costs no launch."""
        named = range(self.batch) if seqs is None else list(seqs)
        for b in named:
            if not 0 <= b < self.batch:
                raise ValueError(f"no sequence {b} of {self.batch}")
        grown = False
        if n_chunks > self.capacity:
            factor = 1 << max(0, (int(n_chunks) - 1) // self.capacity).bit_length()
            self._widen(self.capacity * factor)
            grown = True
        want = self.capacity if self.own else int(n_chunks)
        rows = list(self._rows)
        for b in named:
            rows[b] = max(rows[b], want)
        return self._reserve(rows) or grown

    def _widen(self, capacity: int) -> None:
        """A table of `capacity` rows; where every sequence owns its pages, the pool with it."""
        blocks, old = capacity // PAGE, self.table
        with self._allocation_scope():
            self.table = torch.full((self.batch, blocks), -1, device=self.device, dtype=torch.int32)
        self.table[:, : old.shape[1]].copy_(old)
        self.generation += 1
        if self.own and self._rows == [PAGE * old.shape[1]] * self.batch:
            have, new = self.pages, self.batch * (blocks - old.shape[1])
            self._grow_pool(have + new)
            self.table[:, old.shape[1]:].copy_(torch.arange(have, have + new, dtype=torch.int32).view(self.batch, -1))
            self.refs[have:].fill_(1)
            self._rows = [capacity] * self.batch

    def _grow_pool(self, pages: int) -> None:
        """A pool of `pages`, the pages that there are at their numbers."""
        have = self.pages
        with self._allocation_scope():
            store, scales, refs = self._pool(pages)
        store[:, :, :have].copy_(self.store)
        scales[:, :, :have].copy_(self.scales)
        refs[:have].copy_(self.refs)
        self.store, self.scales, self.refs = store, scales, refs
        self.generation += 1

    def _reserve(self, rows: List[int]) -> bool:
        if all(new // PAGE <= old // PAGE for new, old in zip(rows, self._rows)):
            self._rows = rows
            return False
        want = torch.tensor(rows, device=self.device)
        missing = int(pages_reserve(self.refs, self.table, want))
        if missing:
            self._grow_pool(max(2 * self.pages, self.pages + missing))
            if int(pages_reserve(self.refs, self.table, want)):
                raise RuntimeError("the grown pool has too few pages")  # its counts do not fit its table
        self._rows = rows
        return bool(missing)

    def fork(self, src: int, dst: Sequence[int], S: torch.Tensor) -> bool:
        """The sequences `dst` continue `src`, which holds S[src] rows: they share its whole blocks, its newest rows are
        copied in every layer, S[dst] = S[src], and they get pages for as many rows as src has. Their own are released.
        Returns True when a tensor of the arena was reallocated for those pages, as `ensure` does."""
        planes = self.tails.view(2 * self.n_layers, *self.tails.shape[2:])
        pages_fork(self.refs, self.table, S, src, dst, planes)
        if len(dst):
            self._shared = max(self._shared, min(int(S[src]), self.capacity) // PAGE * PAGE)
        rows = list(self._rows)
        for b in dst:
            rows[b], self._rows[b] = rows[src], 0
        return self._reserve(rows)

    def release(self, seqs: Sequence[int]) -> None:
        """The sequences have ended: their pages are free. An `ensure` that names them, or nobody, gives them pages again."""
        pages_free(self.refs, self.table, seqs)
        for b in seqs:
            self._rows[b] = 0

    def compact(self, pages: Optional[int] = None) -> int:
        """The pages in use at the front of a pool of `pages` (by default as many as are in use); returns how many are in
        use. Reads their number on the host."""
        live = int((self.refs > 0).sum())
        pages = max(live, 1) if pages is None else int(pages)
        if pages < max(live, 1):
            raise ValueError(f"a pool of {pages} pages for {live} in use")
        with self._allocation_scope():
            store, scales, refs = self._pool(pages)
        flat = lambda codes, sc, n: PagePool(codes.view(2 * self.n_layers, codes.shape[2], -1), sc.view(2 * self.n_layers, codes.shape[2], -1), n)
        table, _ = pages_compact(flat(self.store, self.scales, self.refs), self.table, flat(store, scales, refs))
        self.table.copy_(table)
        self.store, self.scales, self.refs = store, scales, refs
        self.generation += 1
        return live

    def _reallocate(self, capacity: int) -> None:
        self._widen(-(-int(capacity) // PAGE) * PAGE)


class ArenaLayer8(ArenaLayer):
    """A layer of the state: `write` appends rows, whole blocks in 8 bits; `views` reads rows back."""

    __slots__ = ()

    def _room(self, T: int) -> None:
        a, n = self.arena, self.state.n
        if n + T > a.capacity:
            raise RuntimeError(f"arena overflow: rows up to {n + T} in a capacity of {a.capacity}")
        if any((n + T) // PAGE > r // PAGE for r in a._rows):
            raise RuntimeError(f"no pages for rows up to {n + T}: ensure({n + T}) gives them out")
        if n % PAGE and n < a._held[self.layer]:
            raise ValueError(f"rows up to {a._held[self.layer]} are stored: a state goes back to a whole block of {PAGE}, not to {n}")
        if n < a._shared:
            first, pages = n // PAGE, a.table[:, n // PAGE : a._shared // PAGE]
            shared = (a.refs[pages.clamp(min=0).long()] > 1).logical_and(pages >= 0).any(0).nonzero().flatten().tolist()
            # the record goes down to what the counts still say, so that a window asks them only while there is more
            a._shared = PAGE * (first + shared[-1] + 1) if shared else PAGE * first
            if shared and first + shared[0] < (n + T) // PAGE:
                raise ValueError(f"rows {n} to {n + T} lie in blocks that forks share: release them first")

    def _cast(self, p2: torch.Tensor, info: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        return p2.to(self.arena.dtype), info.to(self.arena.dtype)

    def write(self, p2: torch.Tensor, info: torch.Tensor) -> None:
        """Append T rows [n, n + T) to every sequence; p2 / info are [batch, H, T, dh]."""
        n, T = self.state.n, p2.shape[2]
        self._room(T)
        cache8_write(self.arena.cache(self.layer), *self._cast(p2, info), n)
        self.arena._held[self.layer] = n + T

    def views(self, upto: int) -> Tuple[torch.Tensor, torch.Tensor]:
        """(P2, I~) rows [0, upto) of sequences that hold `upto` rows, as new [batch, H, upto, dh] tensors in the arena's
        dtype: whole blocks at their 8-bit values, the rest as it is."""
        return cache8_read(self.arena.cache(self.layer), upto, 0, upto, dtype=self.arena.dtype)

    def extend(self, p2: torch.Tensor, info: torch.Tensor) -> Tuple[torch.Tensor, torch.Tensor]:
        """Append T rows as `write` does; rows [0, n + T) for their own queries: those that were held as they were held
        before the call, the new ones as they are."""
        a, n, T = self.arena, self.state.n, p2.shape[2]
        new = self._cast(p2, info)
        if n == 0:
            self.write(*new)
            return new
        self._room(T)
        out = tuple(torch.empty(a.batch, a.n_heads, n + T, a.d_head, device=a.device, dtype=a.dtype) for _ in range(2))
        cache8_read(a.cache(self.layer), n, 0, n, out=tuple(t[:, :, :n] for t in out))
        for t, rows in zip(out, new):
            t[:, :, n:].copy_(rows)
        self.write(*new)
        return out
