"""The quantised decode path as a user runs it: prompt windows into an arena in 4 bits, then decode steps over
it with the projections in 8-bit integers, eager and captured. Every piece is tested against 64 bits on its own;
here the path has to equal those pieces put together by hand, bit for bit."""

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


@pytest.mark.parametrize("d,H,B,dtype,kw", [(192, 4, 1, BF16, {}), (768, 8, 2, BF16, dict(qk_norm=True, out_gate=True)),
                                            (192, 4, 2, F32, {}), (512, 8, 1, BF16, dict(out_gate=True))])
def test_prompt_windows(cuda, d, H, B, dtype, kw):
    """The first window equals the layer without a cache; the second reads the first's rows at their 4-bit values
    and its own as they are; the arena then holds both."""
    from mote_amd.arena import ArenaState
    from mote_amd.arena4 import RelationArena4
    from mote_amd.cache4 import cache4_read, cache4_write, cache4_zeros
    from mote_amd.flash_relation import flash_relation

    m = _mixer(cuda, d, H, 1, dtype, **kw)
    arena = RelationArena4(2, H, 256, d // H, cuda, dtype, batch=B)
    state = ArenaState(arena)
    x1, x2 = _x(1, B, 130, d, dtype=dtype).to(cuda), _x(2, B, 37, d, dtype=dtype).to(cuda)
    with torch.no_grad():
        out1, g1 = m(x1, cache=state[1], return_gates=True)
        want1, gw1 = m(x1, return_gates=True)
        state.advance(130)
        assert torch.equal(out1, want1) and torch.equal(g1, gw1)
        p1, p2, info = m.heads(x1, 0)
        hand = cache4_zeros(B, H, 256, d // H, cuda)
        cache4_write(hand, p2, info, 0)
        for a, b in zip(arena.cache(1), hand):
            assert torch.equal(a, b)
        assert (arena.store[0] == 0).all()
        out2, g2 = m(x2, cache=state[1], return_gates=True)
        q, k, v = m.heads(x2, 130)
        held = cache4_read(hand, d // H, 0, 130, dtype=dtype)
        y, g = flash_relation(q, torch.cat([held[0], k], 2), torch.cat([held[1], v], 2), m.lam, m.tau_s, q_start=130)
        assert torch.equal(out2, m._out(y, x2)) and torch.equal(g2, g)
        cache4_write(hand, k, v, 130)
        state.advance(37)
        for a, b in zip(arena.cache(1), hand):
            assert torch.equal(a, b)
        for a, b in zip(state[1].views(167), cache4_read(hand, d // H, 0, 167, dtype=dtype)):
            assert torch.equal(a, b)
    with pytest.raises(RuntimeError, match="no backward"):
        m(x2, cache=state[1])
    with torch.no_grad(), pytest.raises(RuntimeError, match="overflow"):
        m(x1, cache=state[1])


def _by_hand(m, x, S, cache, arena_dtype, w8, y_dtype, in_place_rows=None):
    """One decode step from the public operators."""
    from mote_amd.cache4 import relation_decode4
    from mote_amd.decode import relation_decode
    from mote_amd.int8 import int8_linear

    B, _, Dm = x.shape
    H, dh = m.n_heads, m.d_head
    qkv = int8_linear(x.reshape(B, Dm), w8["qkv"]).view(B, 3, H, dh).to(arena_dtype)
    if m.qk_norm:
        qkv = torch.stack([m.p1_norm(qkv[:, 0]), m.p2_norm(qkv[:, 1]), qkv[:, 2]], 1)
    rope32 = x.dtype == F32 and arena_dtype != F32
    args = (m.lam, m.tau_s, m.inv_freq, m.theta, m.layer_idx)
    if in_place_rows is None:
        y, g = relation_decode4(qkv[:, 0], qkv[:, 1], qkv[:, 2], S, cache, *args, rope_f32=rope32)
    else:
        y, g = relation_decode(qkv[:, 0], qkv[:, 1], qkv[:, 2], S, *in_place_rows, *args, rope_f32=rope32)
    y = y.to(y_dtype).reshape(B, H * dh)
    if m.out_gate:
        y = y * torch.sigmoid(int8_linear(x.reshape(B, Dm), w8["wg"]))
    return int8_linear(y, w8["wo"]).view(B, 1, Dm), g


@pytest.mark.parametrize("d,H,B,x_dtype,arena_dtype,kw", [
    (192, 4, 3, BF16, BF16, {}), (768, 8, 2, BF16, BF16, dict(qk_norm=True, out_gate=True)), (192, 4, 1, F32, F32, {}),
    (512, 8, 16, F32, BF16, {})])
@pytest.mark.parametrize("four", [True, False])
def test_prompt_then_steps(cuda, d, H, B, x_dtype, arena_dtype, kw, four):
    """A padded batch of prompts (each sequence at its own length), then steps through RelationMainStep over two
    layers with 8-bit projections, over an arena in 4 bits or in the model's dtype; the arena grows on the way."""
    from mote_amd.arena import RelationArena
    from mote_amd.arena4 import RelationArena4
    from mote_amd.cache4 import Cache4, cache4_write
    from mote_amd.graph import RelationMainStep
    from mote_amd.int8 import int8_weight

    mixers = [_mixer(cuda, d, H, i, x_dtype, **kw) for i in range(2)]
    dh = d // H
    arena = (RelationArena4 if four else RelationArena)(2, H, 64, dh, cuda, arena_dtype, batch=B)
    arena.claim(1, 64) if B == 1 else None
    lens = (torch.arange(B) * 7 % 50 + 3).to(cuda)
    S = lens.clone()
    for i in range(2):
        k, v = _x(i, B, H, 60, dh, dtype=arena_dtype).to(cuda), _x(i + 9, B, H, 60, dh, dtype=arena_dtype).to(cuda)
        if four:
            cache4_write(arena.cache(i), k, v, torch.zeros_like(lens), lens)
        else:
            arena.p2(i)[:, :, :60], arena.info(i)[:, :, :60] = k, v
    twin = [Cache4(*(t.clone() for t in arena.cache(i))) for i in range(2)] if four else [None, None]
    rows = [None, None] if four else [(arena.p2(i).clone(), arena.info(i).clone()) for i in range(2)]
    St, xm = S.clone(), torch.empty(2, B, device=cuda)
    w8 = [{"qkv": int8_weight(torch.cat([m.w1.weight, m.w2.weight, m.wi.weight])), "wo": int8_weight(m.wo.weight),
           **({"wg": int8_weight(m.wg.weight)} if m.out_gate else {})} for m in mixers]
    step = RelationMainStep(arena, S, xm, int8=True)
    with torch.no_grad():
        for t in range(5):
            if t == 3:
                arena.ensure(100)  # the store moves and grows
                grow = lambda t_: torch.cat([t_, torch.zeros_like(t_)], 2)
                twin = [Cache4(*(grow(t_) for t_ in c)) if four else None for c in twin]
                rows = [None if four else tuple(grow(t_) for t_ in r) for r in rows]
            x = xt = _x(100 + t, B, 1, d, dtype=x_dtype).to(cuda)
            for i, m in enumerate(mixers):
                x = step(m, x, li=i)
                xt, g = _by_hand(m, xt, St, twin[i], arena_dtype, w8[i], x_dtype, rows[i])
                assert torch.equal(x, xt), (t, i)
                assert torch.allclose(xm[i], g.mean(1), rtol=16 * 2.0 ** -24, atol=0)
            St += 1
            assert torch.equal(S, St)
    if four:
        for i in range(2):
            for a, b in zip(arena.cache(i), twin[i]):
                assert torch.equal(a, b)


def test_captured_token_with_a_predicate(cuda):
    """One graph of a two-layer token (4-bit arena, 8-bit projections) replayed with the router's bit on and off,
    other work in between, against the eager steps; new weights reach it through sync_params."""
    from mote_amd.arena4 import RelationArena4
    from mote_amd.graph import RelationMainStep

    d, H, B = 512, 8, 2
    mixers = [_mixer(cuda, d, H, i) for i in range(2)]
    mk = lambda: RelationArena4(2, H, 128, d // H, cuda, BF16, batch=B)
    a, b = mk(), mk()
    Sa, Sb = torch.tensor([0, 5], device=cuda), torch.tensor([0, 5], device=cuda)
    run, x = torch.ones(1, dtype=torch.bool, device=cuda), _x(0, B, 1, d).to(cuda)
    sa, sb = RelationMainStep(a, Sa, run=run, int8=True), RelationMainStep(b, Sb, int8=True)

    def token(step, h):
        for i, m in enumerate(mixers):
            h = step(m, h, li=i)
        return h

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        token(sa, x)
    torch.cuda.current_stream().wait_stream(side)
    a.store.zero_(), a.scales.zero_(), Sa.copy_(Sb)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token(sa, x)
    want = None
    for t in range(8):
        x.copy_(_x(50 + t, B, 1, d))
        run.fill_(t % 3 != 1)
        if t == 5:
            with torch.no_grad():
                mixers[0].w2.weight.mul_(1.25)
            sa.sync_params(), sb.sync_params()
        graph.replay()
        if t % 3 != 1:
            want = token(sb, x)
        torch.cuda.synchronize()
        assert torch.equal(Sa, Sb) and torch.equal(a.store, b.store) and torch.equal(a.scales, b.scales)
        assert torch.equal(out, want)


def test_what_the_step_refuses(cuda):
    from mote_amd.arena import RelationArena
    from mote_amd.decode import RelationDecodeStep

    m = _mixer(cuda, 192, 4)
    with pytest.raises(ValueError, match="64 sequences"):
        RelationDecodeStep(m, RelationArena(1, 4, 64, 48, cuda, BF16, batch=65), 0, int8=True)
    step = RelationDecodeStep(m, RelationArena(1, 4, 64, 48, cuda, BF16, batch=2), 0, int8=True)
    S = torch.zeros(2, dtype=torch.int64, device=cuda)
    for shape in ((2, 2, 192), (1, 1, 192)):
        with pytest.raises(ValueError, match="takes x"):
            step(torch.zeros(shape, device=cuda, dtype=BF16), S)
