"""RelationArena8 on the host: sizes, views that it does not give, growth and the host record of pages."""

from __future__ import annotations

import pytest
import torch

from mote_amd.arena import ArenaState, RelationArena
from mote_amd.arena8 import ArenaLayer8, RelationArena8
from mote_amd.prefix import ArenaPages, Branch


def test_sizes_and_layers():
    a = RelationArena8(3, 4, 100, 40, "cpu", torch.bfloat16, batch=2)
    assert a.capacity == 128 and a.pages == 4 and a.chunks == 3
    assert a.store.shape == (3, 2, 4, 4, 64 * 48) and a.scales.shape == (3, 2, 4, 4) and a.tails.shape == (3, 2, 2, 4, 64, 40)
    assert a.table.tolist() == [[0, 1], [2, 3]] and a.refs.tolist() == [1] * 4
    assert a.bytes_per_chunk == 3 * 2 * 2 * 4 * (64 * 48 + 4) // 64 + (3 * 2 * 2 * 4 * 4 % 64 > 0)
    assert a.nbytes() == 3 * 2 * 4 * 4 * (64 * 48 + 4) + 3 * 2 * 2 * 4 * 64 * 40 * 2 + 4 * 4 + 4 * 4
    rows = RelationArena(3, 4, 12800, 96, "cpu", torch.bfloat16)
    pages = RelationArena8(3, 4, 12800, 96, "cpu", torch.bfloat16)
    assert pages.nbytes() < 0.51 * rows.nbytes()
    c = a.cache(1)
    assert [tuple(t.shape) for t in c] == [(4, 4, 3, 64, 16), (4, 4), (4, 4, 48, 64), (4, 4), (2, 4, 64, 40), (2, 4, 64, 40), (2, 2)]
    assert a.cache(1) is c
    c.info[3, 2, 47] = 7
    assert (a.store[1, 1, 3, 2, 47 * 64:] == 7).all()
    st = ArenaState(a, 5)
    assert isinstance(st[2], ArenaLayer8) and st[2].n == 5 and len(list(st)) == 3
    few = RelationArena8(1, 2, 640, 64, "cpu", batch=4, pages=7)
    assert few.capacity == 640 and few.pages == 7 and (few.table == -1).all() and (few.refs == 0).all()


def test_what_it_refuses():
    with pytest.raises(ValueError, match="head dim"):
        RelationArena8(1, 2, 64, 132, "cpu")
    with pytest.raises(TypeError, match="8 bits"):
        RelationArena8(1, 2, 64, 32, "cpu", torch.float16)
    with pytest.raises(ValueError, match="capacity"):
        RelationArena8(1, 2, 0, 32, "cpu")
    with pytest.raises(ValueError, match="0 pages"):
        RelationArena8(1, 2, 64, 32, "cpu", pages=0)
    a = RelationArena8(1, 2, 64, 32, "cpu")
    for view in (lambda: a.buf, lambda: a.p2(0), lambda: a.info(0), lambda: a.rows(0, 4)):
        with pytest.raises(TypeError, match="no rows to view"):
            view()
    with pytest.raises(TypeError, match="pages"):
        ArenaPages(pin=False).store_rows(Branch(), a, 0, 4)
    x = torch.zeros(1, 2, 60, 32)
    with pytest.raises(RuntimeError, match="overflow"):
        ArenaState(a, 5)[0].write(x, x)
    few = RelationArena8(1, 2, 640, 32, "cpu", pages=7)
    with pytest.raises(RuntimeError, match="no pages for rows up to 65"):
        ArenaState(few, 5)[0].write(x, x)
    a._held[0] = 40
    with pytest.raises(ValueError, match="goes back to a whole block"):
        ArenaState(a, 3)[0].extend(x[:, :, :4], x[:, :, :4])


def test_growth_keeps_every_sequence():
    a = RelationArena8(2, 2, 128, 32, "cpu", batch=3)
    for t in (a.store, a.scales, a.tails):
        t.copy_(torch.rand(t.shape) * 100)
    before = [t.clone() for t in (a.store, a.scales, a.tails, a.table)]
    c = a.cache(0)
    assert not a.ensure(128) and a.ensure(129)
    assert a.capacity == 256 and a.pages == 12 and a.generation > 0
    assert torch.equal(a.store[:, :, :6], before[0]) and torch.equal(a.scales[:, :, :6], before[1])
    assert torch.equal(a.tails, before[2]) and torch.equal(a.table[:, :2], before[3])
    assert sorted(a.table.flatten().tolist()) == list(range(12)) and a.refs.tolist() == [1] * 12
    assert (a.store[:, :, 6:] == 0).all() and a.cache(0) is not c
    assert a.ensure(1000) and a.capacity == 1024 and a.pages == 48
    few = RelationArena8(1, 2, 64, 32, "cpu", batch=2, pages=3)
    assert not few.ensure(63)  # no whole block yet: no page, no launch
    with pytest.raises(RuntimeError, match="MI355X"):
        few.ensure(64)
    with pytest.raises(RuntimeError, match="MI355X"):
        a.release([1])
    with pytest.raises(ValueError, match="in use"):
        a.compact(47)


def test_a_window_leaves_shared_blocks_alone():
    """Back to a whole block that a fork shares: refused while it does, before anything is stored."""
    a = RelationArena8(1, 2, 256, 32, "cpu", batch=2)
    a.table[1, :2] = a.table[0, :2]
    a.refs[a.table[0, :2].long()] = 2
    a._shared = 128  # what a fork of 150 rows leaves
    x = torch.zeros(2, 2, 70, 32)
    for n in (0, 64):
        with pytest.raises(ValueError, match="forks share"):
            ArenaState(a, n)[0].write(x, x)
    for n, T in ((128, 70), (64, 63)):  # behind them; no block of them becomes whole
        with pytest.raises(RuntimeError, match="MI355X"):
            ArenaState(a, n)[0].write(x[:, :, :T], x[:, :, :T])
    a.refs[a.table[0, :2].long()] = 1  # released
    with pytest.raises(RuntimeError, match="MI355X"):
        ArenaState(a, 0)[0].write(x, x)
