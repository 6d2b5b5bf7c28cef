"""Serving from pages of 8-bit values as a user runs it: prompt windows, forks, decode steps, the draw of the next token,
sequences that end, the pool compacted. Every piece is tested against 64 bits on its own; here the path has to equal
those pieces put together by hand, bit for bit."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _mixer(cuda, d, H, layer=0, dtype=BF16, **kw):
    from mote_amd.relation import FullRelation

    torch.manual_seed(d + layer)
    m = FullRelation(d, H, layer, device=cuda, **kw).to(dtype)
    with torch.no_grad():
        m.lam.fill_(0.4)
        m.theta.copy_(torch.rand(H // 2) * 0.6 - 0.3)
    return m


def _x(seed, *shape, dtype=BF16):
    return torch.randn(*shape, generator=torch.Generator().manual_seed(seed)).to(dtype)


def _hand(B, H, blocks, D, cuda, dtype):
    from mote_amd.cache8 import cache8_zeros

    c = cache8_zeros(B, H, B * blocks, 64 * blocks, D, cuda, dtype)
    c.table.copy_(torch.arange(B * blocks).view(B, blocks).int())
    return c


@pytest.mark.parametrize("d,H,B,dtype,kw", [(192, 4, 1, BF16, {}), (768, 8, 2, BF16, dict(qk_norm=True, out_gate=True)),
                                            (192, 4, 2, F32, {}), (512, 8, 1, BF16, dict(out_gate=True))])
def test_prompt_windows(cuda, d, H, B, dtype, kw):
    """The first window equals the layer without a cache; the second reads the first's whole blocks at their 8-bit values
    and its open block and itself as they are; the arena then holds both."""
    from mote_amd.arena import ArenaState
    from mote_amd.arena8 import RelationArena8
    from mote_amd.cache8 import cache8_read, cache8_write
    from mote_amd.flash_relation import flash_relation

    m = _mixer(cuda, d, H, 1, dtype, **kw)
    arena = RelationArena8(2, H, 256, d // H, cuda, dtype, batch=B)
    state = ArenaState(arena)
    x1, x2 = _x(1, B, 140, d, dtype=dtype).to(cuda), _x(2, B, 67, d, dtype=dtype).to(cuda)
    with torch.no_grad():
        out1, g1 = m(x1, cache=state[1], return_gates=True)
        want1, gw1 = m(x1, return_gates=True)
        state.advance(140)
        assert torch.equal(out1, want1) and torch.equal(g1, gw1)
        p1, p2, info = m.heads(x1, 0)
        hand = _hand(B, H, 4, d // H, cuda, dtype)
        cache8_write(hand, p2, info, 0)
        for a, b in zip(arena.cache(1), hand):
            assert torch.equal(a, b)
        assert (arena.store[0] == 0).all() and (arena.tails[0] == 0).all()
        out2, g2 = m(x2, cache=state[1], return_gates=True)
        q, k, v = m.heads(x2, 140)
        held = cache8_read(hand, 140, dtype=dtype)
        assert torch.equal(held[0][:, :, 128:], p2[:, :, 128:]) and not torch.equal(held[0][:, :, :128], p2[:, :, :128])
        y, g = flash_relation(q, torch.cat([held[0], k], 2), torch.cat([held[1], v], 2), m.lam, m.tau_s, q_start=140)
        assert torch.equal(out2, m._out(y, x2)) and torch.equal(g2, g)
        cache8_write(hand, k, v, 140)
        state.advance(67)
        for a, b in zip(arena.cache(1), hand):
            assert torch.equal(a, b)
        for a, b in zip(state[1].views(207), cache8_read(hand, 207, dtype=dtype)):
            assert torch.equal(a, b)
        state.n = 150
        with pytest.raises(ValueError, match="goes back to a whole block"):
            m(x2, cache=state[1])
        state.n = 128  # a whole block: what was behind it is replaced
        m(x2[:, :5], cache=state[1])
        assert torch.equal(arena.tails[1, 0, :, :, :5], m.heads(x2[:, :5], 128)[1])
        state.n = 200
        with pytest.raises(RuntimeError, match="overflow"):
            m(x1, cache=state[1])
    state.n = 207
    with pytest.raises(RuntimeError, match="no backward"):
        m(x2[:, :20], cache=state[1])


@pytest.mark.parametrize("d,H,B,x_dtype,arena_dtype,kw,int8", [
    (192, 4, 3, BF16, BF16, {}, False), (768, 8, 2, BF16, BF16, dict(qk_norm=True, out_gate=True), True),
    (192, 4, 1, F32, F32, {}, True), (512, 8, 4, F32, BF16, {}, False)])
def test_steps_over_a_growing_arena(cuda, d, H, B, x_dtype, arena_dtype, kw, int8):
    """A padded batch of prompts, then steps through RelationMainStep over two layers, by hand beside it; the table and the
    pool grow on the way and pages go out as rows come."""
    from mote_amd.arena8 import RelationArena8
    from mote_amd.cache8 import cache8_write, relation_decode8
    from mote_amd.decode import skinny_linear
    from mote_amd.graph import RelationMainStep
    from mote_amd.int8 import int8_linear, int8_weight

    mixers = [_mixer(cuda, d, H, i, x_dtype, **kw) for i in range(2)]
    dh = d // H
    arena = RelationArena8(2, H, 64, dh, cuda, arena_dtype, batch=B, pages=2)
    arena.ensure(64)
    assert arena.pages >= B
    lens = (torch.arange(B) * 7 % 50 + 10).to(cuda)
    S = lens.clone()
    twins = [_hand(B, H, 4, dh, cuda, arena_dtype) for _ in range(2)]
    for i in range(2):
        k, v = _x(i, B, H, 60, dh, dtype=arena_dtype).to(cuda), _x(i + 9, B, H, 60, dh, dtype=arena_dtype).to(cuda)
        for c in (arena.cache(i), twins[i]):
            cache8_write(c, k, v, torch.zeros_like(lens), lens)
    St, xm = S.clone(), torch.empty(2, B, device=cuda)
    step = RelationMainStep(arena, S, xm, int8=int8)
    skinny = x_dtype == BF16 and d % 128 == 0
    lin = lambda x, w: int8_linear(x, int8_weight(w)) if int8 else skinny_linear(x, w) if skinny else torch.nn.functional.linear(x, w)
    with torch.no_grad():
        for t in range(75):
            arena.ensure(int(lens.max()) + t + 1)
            x = xt = _x(100 + t, B, 1, d, dtype=x_dtype).to(cuda)
            for i, m in enumerate(mixers):
                x = step(m, x, li=i)
                qkv = lin(xt.reshape(B, d), torch.cat([m.w1.weight, m.w2.weight, m.wi.weight])).view(B, 3, H, dh).to(arena_dtype)
                if m.qk_norm:
                    qkv = torch.stack([m.p1_norm(qkv[:, 0]), m.p2_norm(qkv[:, 1]), qkv[:, 2]], 1)
                # a table as wide as the arena's: splits follow its width, and sums their order
                twin = twins[i]._replace(table=twins[i].table[:, : arena.capacity // 64])
                y, g = relation_decode8(qkv[:, 0], qkv[:, 1], qkv[:, 2], St, twin, m.lam, m.tau_s, m.inv_freq, m.theta, m.layer_idx,
                                        rope_f32=x_dtype == F32 and arena_dtype != F32)
                y = y.to(x_dtype).reshape(B, d)
                if m.out_gate:
                    y = y * torch.sigmoid(lin(xt.reshape(B, d), m.wg.weight))
                xt = lin(y, m.wo.weight).view(B, 1, d)
                assert torch.equal(x, xt), (t, i)
            St += 1
            assert torch.equal(S, St)
    rows = S.tolist()
    for i in range(2):
        c, tw = arena.cache(i), twins[i]
        for b in range(B):
            for j in range(rows[b] // 64):
                for x, y in zip(c[:4], tw[:4]):
                    assert torch.equal(x[int(c.table[b, j])], y[int(tw.table[b, j])])
            r = rows[b] % 64
            for x, y in zip(c[4:6], tw[4:6]):
                assert torch.equal(x[b, :, :r], y[b, :, :r])
    assert max(rows) <= arena.capacity < 2 * max(max(rows), 64) and (arena.refs.sum() == (arena.table >= 0).sum())


def test_a_group_of_continuations(cuda):
    """Together, as they are used: one prompt read, five continuations forked from it, tokens drawn and fed back through a
    captured step, one sequence ended and another forked in its place, the pool compacted on the way. Each sequence has
    to equal, bit for bit, the same tokens fed through an arena in which it is alone with pages of its own."""
    from mote_amd.arena import ArenaState
    from mote_amd.arena8 import RelationArena8
    from mote_amd.decode import skinny_linear
    from mote_amd.graph import RelationMainStep
    from mote_amd.sample import sample_tokens

    d, H, L, B, V = 256, 4, 2, 6, 272
    mixers = [_mixer(cuda, d, H, i) for i in range(L)]
    embed, head = _x(1, V, d).to(cuda), (_x(2, V, d) / 4).to(cuda)
    prompt = _x(3, 1, 100, d).to(cuda)
    g = torch.Generator().manual_seed(5)
    us = torch.rand(60, B, generator=g).to(cuda)
    mk = lambda pages: RelationArena8(L, H, 256, d // H, cuda, BF16, batch=B, pages=pages)

    def read_prompt(arena):
        state = ArenaState(arena)
        h = prompt.expand(arena.batch, -1, -1).contiguous()
        with torch.no_grad():
            for i, m in enumerate(mixers):
                h = m(h, cache=state[i])
        return h[:, -1]

    shared, alone = mk(8), mk(None)  # 8 pages: too few at first, the pool grows
    shared.ensure(100)
    last = read_prompt(shared)   # every slot reads the prompt; all but the first are released and forked from it
    assert torch.equal(last, read_prompt(alone))
    S, Sa = torch.full((B,), 100, device=cuda), torch.full((B,), 100, device=cuda)
    shared.release([1, 2, 3, 4, 5])
    assert int((shared.refs > 0).sum()) == 1
    shared.fork(0, [1, 2, 3, 4, 5], S)
    assert shared.refs.max() == 6 and int((shared.refs > 0).sum()) == 1 and S.tolist() == [100] * B
    with pytest.raises(ValueError, match="forks share"):  # a window over a block that several sequences read
        ArenaState(shared)[0].write(torch.zeros(B, H, 64, d // H, device=cuda, dtype=BF16), torch.zeros(B, H, 64, d // H, device=cuda, dtype=BF16))
    for t in shared.tails.flatten(0, 1):
        assert torch.equal(t[:, :, :36], t[:1, :, :36].expand(B, -1, -1, -1))

    def token_step(step, token, u, T, k):
        h = embed[token].view(B, 1, d)
        for i, m in enumerate(mixers):
            h = step(m, h, li=i)
        logits = skinny_linear(h.view(B, d), head)
        return logits, sample_tokens(logits, u, T, k, top_p=0.95, min_p=0.001)

    T, k = torch.tensor([0.7, 1.0, 1.3, 0.0, 1.0, 0.9], device=cuda), torch.tensor([0, 40, 5, 0, 271, 100], device=cuda)
    shared.ensure(160)
    first = sample_tokens(skinny_linear(last, head), us[0], T, k)
    token, u = first.clone(), us[0].clone()
    ours, theirs = RelationMainStep(shared, S), RelationMainStep(alone, Sa)

    def capture():
        keep = [t.clone() for t in (shared.store, shared.scales, shared.tails, S, token)]
        token_step(ours, token, u, T, k)
        for a, b in zip((shared.store, shared.scales, shared.tails, S, token), keep):
            a.copy_(b)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            logits, drawn = token_step(ours, token, u, T, k)
            token.copy_(drawn)
        return graph, logits

    graph, logits = capture()
    other = first.clone()
    for t in range(1, 60):
        u.copy_(us[t])
        graph.replay()
        theirs_logits, other = token_step(theirs, other, us[t], T, k)
        torch.cuda.synchronize()
        assert torch.equal(logits, theirs_logits) and torch.equal(token, other), t
        assert torch.equal(S, Sa)
        if t == 30:  # sequence 2 ends; 4 continues there too: the same rows copied by hand in the other arena
            shared.release([2])
            shared.fork(4, [2], S)
            alone.store[:, :, alone.table[2].long()] = alone.store[:, :, alone.table[4].long()]
            alone.scales[:, :, alone.table[2].long()] = alone.scales[:, :, alone.table[4].long()]
            alone.tails[:, :, 2] = alone.tails[:, :, 4]
            for tok in (token, other):
                tok[2] = tok[4]
        if t == 40:
            before = int((shared.refs > 0).sum())
            assert shared.compact() == before and shared.pages == before
            shared.ensure(200)
            graph, logits = capture()
    assert len(set(token.tolist())) > 1
    shared.release(range(B))
    assert (shared.refs == 0).all() and (shared.table == -1).all()
