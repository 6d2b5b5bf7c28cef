"""The life of a RelationArena8 on the host: its calls over plain loops in the place of the pages' kernels (which have
tests of their own against such loops), so that what it gives out, records and reports can be followed step by step."""

from __future__ import annotations

import pytest
import torch

from mote_amd import arena8
from mote_amd.arena8 import RelationArena8


def _free(refs, table, seqs):
    for s in list(seqs):
        for t in table[s].tolist():
            if 0 <= t < len(refs):
                refs[t] -= 1
        table[s] = -1


def _fork(refs, table, S, src, dst, tails=None):
    n = min(max(int(S[src]), 0) // 64, table.shape[1])
    for s in list(dst):
        _free(refs, table, [s])
        table[s, :n] = table[src, :n]
        for t in table[s].tolist():
            if t >= 0:
                refs[t] += 1
        S[s] = S[src]
        if tails is not None:
            tails[:, s, :, : int(S[src]) % 64] = tails[:, src, :, : int(S[src]) % 64]


def _reserve(refs, table, rows):
    missing = 0
    free = iter([p for p, n in enumerate(refs.tolist()) if n == 0])
    per = rows.tolist() if torch.is_tensor(rows) else [rows] * table.shape[0]
    for b, row in enumerate(table):
        for j in range(min(max(per[b], 0) // 64, len(row))):
            if row[j] < 0:
                row[j] = next(free, -1)
                if row[j] < 0:
                    missing += 1
                else:
                    refs[row[j]] = 1
    return torch.tensor([missing], dtype=torch.int32)


def _compact(pool, table, into):
    live = (pool.refs > 0).nonzero().flatten().tolist()
    number = {old: new for new, old in enumerate(live)}
    for old, new in number.items():
        into.codes[:, new], into.scales[:, new], into.refs[new] = pool.codes[:, old], pool.scales[:, old], pool.refs[old]
    into.refs[len(live):] = 0
    return torch.tensor([[number.get(t, -1) for t in row] for row in table.tolist()], dtype=torch.int32), torch.tensor([0])


@pytest.fixture
def on_host(monkeypatch):
    for name, body in (("pages_free", _free), ("pages_fork", _fork), ("pages_reserve", _reserve), ("pages_compact", _compact)):
        monkeypatch.setattr(arena8, name, body)


def _sound(a):
    """Counts are the table's entries, and every sequence has the pages that the host's record says."""
    counts = torch.zeros(a.pages, dtype=torch.int32)
    for t in a.table[a.table >= 0].tolist():
        counts[t] += 1
    assert torch.equal(counts, a.refs)
    for b, rows in enumerate(a._rows):
        assert (a.table[b, : rows // 64] >= 0).all(), (b, rows)


def test_a_fork_that_grows_the_pool_says_so(on_host):
    """True when a tensor of the arena was reallocated, as `ensure` answers: what was captured over it is void."""
    a = RelationArena8(1, 2, 640, 32, "cpu", batch=4, pages=20)
    S = torch.full((4,), 200)
    assert not a.ensure(320) and (a.refs > 0).sum() == 20
    a.release([1, 2, 3])
    store, generation = a.store, a.generation
    assert a.fork(0, [1], S) is False  # two pages for the blocks after the three that are shared
    assert a.store is store and a.generation == generation and (a.refs > 0).sum() == 7
    _sound(a)
    a.compact(8)
    store, generation = a.store, a.generation
    assert a.fork(0, [], S) is False and a.generation == generation
    assert a.fork(0, [2, 3], S) is True
    assert a.store is not store and a.generation > generation and (a.refs > 0).sum() == 11
    assert a.cache(0).p2.data_ptr() == a.store.data_ptr()
    _sound(a)


def test_the_ended_stay_without_pages(on_host):
    """`ensure` for the sequences that run: the ended ones, and shorter ones, hold no pages for the longest's rows."""
    a = RelationArena8(1, 2, 1024, 32, "cpu", batch=4, pages=16)
    assert not a.ensure(256) and (a.refs > 0).sum() == 16
    a.release([1, 2, 3])
    assert a.compact() == 4 and a.pages == 4
    assert a.ensure(320, [0]) is True and a.pages == 8  # a growth at least doubles the pool
    assert (a.table[1:] == -1).all() and (a.refs > 0).sum() == 5
    assert a.ensure(512, range(1)) is False and (a.refs > 0).sum() == 8 and a.pages == 8
    _sound(a)
    S = torch.full((4,), 130)
    assert a.fork(0, [2], S) is True  # eight blocks as its source, two of them shared
    assert a.ensure(128, [1]) is False and (a.table[1, :2] >= 0).all() and (a.table[1, 2:] == -1).all()
    assert (a.table[3] == -1).all()
    _sound(a)
    assert a.ensure(128, []) is False
    a.ensure(128)  # all of them, as without a list
    assert (a.table[3, :2] >= 0).all()
    assert a.ensure(1025, [3]) is True and a.capacity == 2048 and (a.table[3, :16] >= 0).all() and (a.table[1, 2:] == -1).all()
    _sound(a)
    for bad in ([4], [-1], [0, 9]):
        with pytest.raises(ValueError, match="no sequence"):
            a.ensure(64, bad)


def test_pages_of_their_own_for_the_named(on_host):
    """Without a pool size every sequence owns pages for its whole capacity, the ended ones once they are named again."""
    a = RelationArena8(2, 2, 128, 32, "cpu", batch=3)
    a.release([1])
    assert a.ensure(129, [0, 2]) is True and a.capacity == 256
    assert (a.table[[0, 2]] >= 0).all() and (a.table[1] == -1).all()
    _sound(a)
    a.ensure(1, [1])
    assert (a.table >= 0).all() and a._rows == [256] * 3
    assert a.ensure(257) is True and a.capacity == 512 and (a.table >= 0).all()
    _sound(a)


def test_windows_wait_for_the_device_only_while_blocks_are_shared(on_host, monkeypatch):
    """What a window asks of the counts is asked once: the record of shared rows goes down with the answer."""
    from mote_amd.arena import ArenaState

    monkeypatch.setattr(arena8, "cache8_write", lambda *a: None)
    a = RelationArena8(2, 2, 512, 32, "cpu", batch=3)
    S = torch.full((3,), 300)
    a.fork(0, [1], S)
    assert a._shared == 256
    x = torch.zeros(3, 2, 70, 32)
    for n in (0, 64, 190):
        with pytest.raises(ValueError, match="forks share"):
            ArenaState(a, n)[0].write(x, x)
    assert a._shared == 256
    ArenaState(a, 256)[0].write(x, x)  # behind them: nothing to ask
    a.fork(2, [1], torch.full((3,), 64))  # one shared block in the place of four
    a._held = [0, 0]
    ArenaState(a, 128)[0].write(x, x)
    assert a._shared == 128  # nothing is shared from there on; the rows before were not asked about
    with pytest.raises(ValueError, match="forks share"):
        ArenaState(a, 0)[0].write(x, x)
    assert a._shared == 64
    a.release([1])
    a.ensure(512)
    ArenaState(a, 0)[1].write(x, x)
    assert a._shared == 0
    a.fork(0, [2], torch.full((3,), 130))
    assert a._shared == 128
