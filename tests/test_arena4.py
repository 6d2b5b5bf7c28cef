"""RelationArena4 on the host: sizes, views that it does not give, growth and residency."""

from __future__ import annotations

import pytest
import torch

from mote_amd.arena import ArenaState, RelationArena
from mote_amd.arena4 import ArenaLayer4, RelationArena4
from mote_amd.prefix import ArenaPages, Branch


def test_sizes_and_layers():
    a = RelationArena4(3, 4, 64, 48, "cpu", torch.bfloat16, batch=2)
    assert a.capacity == 64 and a.store.shape == (3, 2, 2, 4, 64, 32) and a.scales.shape == (3, 2, 2, 4, 64, 2)
    assert a.nbytes() == 64 * a.bytes_per_chunk == 3 * 2 * 2 * 4 * 64 * (32 + 4)
    assert a.nbytes() * 8 == RelationArena(3, 4, 64, 64, "cpu", torch.bfloat16, batch=2).nbytes() * 9 // 4
    c = a.cache(1)
    assert [tuple(t.shape) for t in c] == [(2, 4, 64, 32), (2, 4, 64, 2)] * 2
    c.info[1, 2, 3] = 7
    assert (a.store[1, 1, 1, 2, 3] == 7).all()
    st = ArenaState(a, 5)
    assert isinstance(st[2], ArenaLayer4) and st[2].n == 5 and len(list(st)) == 3
    with pytest.raises(IndexError):
        st[3]
    assert isinstance(ArenaState(RelationArena(1, 2, 8, 32, "cpu", torch.float32))[0], type(st[0]).__mro__[1])


def test_what_it_refuses():
    with pytest.raises(ValueError, match="head dim"):
        RelationArena4(1, 2, 64, 132, "cpu")
    with pytest.raises(TypeError, match="4 bits"):
        RelationArena4(1, 2, 64, 32, "cpu", torch.float16)
    with pytest.raises(ValueError, match="capacity"):
        RelationArena4(1, 2, 0, 32, "cpu")
    a = RelationArena4(1, 2, 64, 32, "cpu")
    for view in (lambda: a.buf, lambda: a.p2(0), lambda: a.info(0), lambda: a.rows(0, 4)):
        with pytest.raises(TypeError, match="no rows to view"):
            view()
    with pytest.raises(TypeError, match="pages"):
        ArenaPages(pin=False).store_rows(Branch(), a, 0, 4)
    with pytest.raises(TypeError, match="pages"):
        ArenaPages(pin=False).hydrate(Branch(), 0, a)
    x = torch.zeros(1, 2, 60, 32)
    with pytest.raises(RuntimeError, match="overflow"):
        ArenaState(a, 5)[0].write(x, x)


@pytest.mark.parametrize("batch", [1, 2])
def test_growth_keeps_live_rows(batch):
    a = RelationArena4(2, 2, 16, 32, "cpu", batch=batch)
    a.store[...] = torch.randint(0, 256, a.store.shape, dtype=torch.uint8)
    a.scales[...] = torch.rand(a.scales.shape).to(torch.bfloat16)
    store, scales = a.store.clone(), a.scales.clone()
    if batch == 1:
        a.claim(9, 10)
    live = 10 if batch == 1 else 16
    assert not a.ensure(16) and a.ensure(17)
    assert a.capacity == 32 and a.generation == 1
    assert torch.equal(a.store[..., :live, :], store[..., :live, :]) and torch.equal(a.scales[..., :live, :], scales[..., :live, :])
    assert (a.store[..., live:, :] == 0).all() and (a.scales[..., live:, :] == 0).all()
    if batch == 1:
        assert (a.owner, a.n_valid) == (9, 10)
        a.invalidate()
        assert a.ensure(100) and a.capacity == 128 and (a.store == 0).all() and (a.scales == 0).all()
