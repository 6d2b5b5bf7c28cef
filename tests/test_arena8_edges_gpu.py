"""Calls of the paged arena that move its tensors, between steps that are captured."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16


def test_a_fork_into_a_pool_that_is_too_small(cuda):
    """Between replays of a captured step a fork finds too few pages: it answers True, the step is captured again, and
    every sequence equals, bit for bit, the same rows in an arena with pages of its own."""
    from mote_amd.arena import ArenaState
    from mote_amd.arena8 import RelationArena8
    from mote_amd.graph import RelationMainStep
    from mote_amd.relation import FullRelation

    d, H, L, B = 256, 4, 2, 3
    torch.manual_seed(0)
    mixers = [FullRelation(d, H, i, device=cuda).to(BF16) for i in range(L)]
    x0 = torch.randn(B, 100, d, device=cuda).to(BF16)
    shared, alone = (RelationArena8(L, H, 256, d // H, cuda, BF16, batch=B, pages=p) for p in (9, None))
    shared.ensure(192)
    with torch.no_grad():
        for a in (shared, alone):
            h, state = x0, ArenaState(a)
            for i, m in enumerate(mixers):
                h = m(h, cache=state[i])
    S, Sa = torch.full((B,), 100, device=cuda), torch.full((B,), 100, device=cuda)
    shared.release([2])
    shared.compact()
    assert shared.pages == 6
    ours, theirs = RelationMainStep(shared, S), RelationMainStep(alone, Sa)
    x = torch.zeros(B, 1, d, device=cuda, dtype=BF16)

    def through(step, h):
        for i, m in enumerate(mixers):
            h = step(m, h, li=i)
        return h

    def capture():
        keep = [t.clone() for t in (shared.store, shared.scales, shared.tails, S)]
        through(ours, x)
        for a, b in zip((shared.store, shared.scales, shared.tails, S), keep):
            a.copy_(b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = through(ours, x)
        return graph, out

    graph, out = capture()
    moved = 0
    for t in range(60):
        x.copy_(torch.randn(B, 1, d, device=cuda))
        if t == 20:  # row 120: block 1 becomes whole, in a page of the grown pool, for each of them
            generation, store = shared.generation, shared.store
            assert shared.fork(0, [2], S) is True
            assert shared.generation > generation and shared.store.data_ptr() != store.data_ptr()
            alone.store[:, :, alone.table[2].long()] = alone.store[:, :, alone.table[0].long()]
            alone.scales[:, :, alone.table[2].long()] = alone.scales[:, :, alone.table[0].long()]
            alone.tails[:, :, 2] = alone.tails[:, :, 0]
            graph, out = capture()
            moved = 1
        graph.replay()
        want = through(theirs, x)
        torch.cuda.synchronize()
        live = [0, 1, 2] if moved else [0, 1]
        assert torch.equal(out[live], want[live]), t
        assert torch.equal(S, Sa)
    assert moved
    for layer in range(L):
        c, w = shared.cache(layer), alone.cache(layer)
        for b in range(B):
            for j in range(2):
                for a, e in zip(c[:4], w[:4]):
                    assert torch.equal(a[int(c.table[b, j])], e[int(w.table[b, j])])
