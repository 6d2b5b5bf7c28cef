"""The quantised operators on the GPU at the edges of what a call may pass: workspaces and layers' objects that
several calls share, sizes at a launch's limit, every kernel form that a rule on sizes selects."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _step_inputs(cuda, seed, B, H, D, cap):
    """(new chunk [B, 3, H, D], S, a cache of ordinary random rows) with every position in the cache's second half."""
    from mote_amd.cache4 import Cache4, groups

    g, G = _gen(seed), groups(D)
    codes = lambda: torch.randint(0, 256, (B, H, cap, 16 * G), generator=g, dtype=torch.uint8).to(cuda)
    scales = lambda: (0.2 + 0.3 * torch.rand(B, H, cap, G, generator=g)).to(BF16).to(cuda)
    x = torch.randn(B, 3, H, D, generator=g).to(BF16).to(cuda)
    return x, torch.randint(cap // 2, cap, (B,), generator=g).to(cuda), Cache4(codes(), scales(), codes(), scales())


def _raw_step(x, S, cache, lam, ws):
    """relation_decode4 through the C entry point, on the workspace as it is; y, g and the S that it advanced."""
    from mote_amd import _lib as L

    B, _, H, D = x.shape
    y = torch.full((B, H, D), 7.0, device=x.device, dtype=BF16)
    g, S = torch.full((B, H), 7.0, device=x.device), S.clone()
    a = L.Decode4Args()
    a.dtype, a.B, a.H, a.D, a.capacity, a.flags, a.tau_s = L.MOTE_BF16, B, H, D, cache.p2.shape[2], L.MOTE_DECODE_ADVANCE, 2.0
    a.lam, a.S, a.in_sb = lam.data_ptr(), S.data_ptr(), x.stride(0)
    a.p1, a.p2, a.info = (x[:, i].data_ptr() for i in range(3))
    a.cache.p2, a.cache.p2_scale, a.cache.info, a.cache.info_scale = (t.data_ptr() for t in cache)
    a.cache.codes_sb, a.cache.codes_sh, a.cache.scale_sb, a.cache.scale_sh = (*cache.p2.stride()[:2], *cache.p2_scale.stride()[:2])
    a.y, a.y_sb, a.g = y.data_ptr(), H * D, g.data_ptr()
    a.workspace, a.workspace_bytes = ws.data_ptr(), ws.numel()
    assert ws.numel() >= int(L.lib().mote_relation_decode4_workspace(a))
    L.check(L.lib().mote_relation_decode4(a, L.stream_of(x)), "mote_relation_decode4")
    return y, g, S


@pytest.mark.parametrize("first,second", [
    ((1, 4, 40, 5120), (4, 4, 48, 768)), ((1, 8, 64, 4096), (3, 4, 40, 4096)), ((1, 8, 64, 8192), (16, 8, 64, 768)),
    ((1, 8, 96, 5376), (16, 8, 96, 512)), ((16, 8, 128, 512), (1, 8, 128, 4096)), ((2, 4, 48, 2560), (4, 4, 40, 1280))])
def test_calls_of_other_sizes_on_one_workspace(cuda, first, second):
    """A workspace that calls of several batches and heads take in turn: each finds its counters at zero, so y, g
    and S are those of a workspace of its own, bit for bit."""
    from mote_amd.cache4 import decode4_workspace, relation_decode4

    n = max(decode4_workspace(*sizes, cuda).numel() for sizes in (first, second))
    ws, lam = torch.zeros(n, dtype=torch.uint8, device=cuda), torch.tensor(0.5, device=cuda)
    for turn in range(3):
        for sizes in (first, second):
            x, S, cache = _step_inputs(cuda, 31 + turn, *sizes)
            y, g, advanced = _raw_step(x, S, cache, lam, ws)
            want = relation_decode4(x[:, 0], x[:, 1], x[:, 2], S, cache, lam)
            assert torch.equal(y, want[0]) and torch.equal(g, want[1]) and torch.equal(advanced, S + 1), (turn, sizes)
            if decode4_workspace(*sizes, cuda).numel() == n:
                got = relation_decode4(x[:, 0], x[:, 1], x[:, 2], S, cache, lam, workspace=ws)
                assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1]), (turn, sizes)


@pytest.mark.parametrize("capacities", [(512, 5376, 1024), (5376, 300)])
def test_one_batch_on_a_workspace_of_any_bytes(cuda, capacities):
    """Calls of one B and H may be given another number of a workspace's bytes each time (a cache that grows)."""
    from mote_amd.cache4 import decode4_workspace, relation_decode4

    B, H, D = 2, 8, 96
    need = {cap: decode4_workspace(B, H, D, cap, cuda).numel() for cap in capacities}
    ws, lam = torch.zeros(max(need.values()), dtype=torch.uint8, device=cuda), torch.tensor(0.5, device=cuda)
    for turn in range(2):
        for cap in capacities:
            x, S, cache = _step_inputs(cuda, 41 + turn, B, H, D, cap)
            y, g, _ = _raw_step(x, S, cache, lam, ws[:need[cap]])
            want = relation_decode4(x[:, 0], x[:, 1], x[:, 2], S, cache, lam)
            assert torch.equal(y, want[0]) and torch.equal(g, want[1]), (turn, cap)


# ---- the arena's layers ----------------------------------------------------------------------------
def test_a_layer_that_is_kept_reads_what_the_arena_holds(cuda):
    """An ArenaLayer4 object gives the rows that are stored, whoever stored them last: another object of the layer,
    a decode step, or itself from tensors that have changed since."""
    from mote_amd.arena import ArenaState
    from mote_amd.arena4 import RelationArena4
    from mote_amd.cache4 import cache4_read, relation_decode4

    B, H, D, T = 2, 4, 48, 20
    state = ArenaState(RelationArena4(1, H, 64, D, cuda, BF16, batch=B), 5)
    cache = state.arena.cache(0)
    k, v, k2, v2 = (torch.randn(B, H, T, D, generator=_gen(50 + i)).to(BF16).to(cuda) for i in range(4))
    layer = state[0]
    held = lambda: cache4_read(cache, D, 0, 5 + T)
    same = lambda: all(torch.equal(a, b) for a, b in zip(layer.views(5 + T), held()))
    layer.write(k, v)
    assert same() and same()
    k.mul_(2.0)
    assert same()
    state[0].write(k2, v2)
    assert same()
    x = torch.randn(B, 3, H, D, generator=_gen(60)).to(BF16).to(cuda)
    relation_decode4(x[:, 0], x[:, 1], x[:, 2], torch.full((B,), 5, device=cuda), cache, torch.tensor(0.5, device=cuda))
    assert same()
    state.advance(T)
    state.n -= T
    assert same()


def test_a_window_reads_its_own_rows_as_they_are(cuda):
    """What `extend` gives a window: the rows before it as they are stored, its own as they were given; the layer
    that a forward hands back holds no rows of its own."""
    from mote_amd.arena import ArenaState, RelationArena
    from mote_amd.arena4 import RelationArena4
    from mote_amd.cache4 import cache4_read
    from mote_amd.relation import FullRelation

    B, H, D = 2, 4, 48
    for arena in (RelationArena4(1, H, 64, D, cuda, BF16, batch=B), RelationArena(1, H, 64, D, cuda, BF16, batch=B)):
        state = ArenaState(arena)
        for T in (11, 1, 30):
            k, v = (torch.randn(B, H, T, D, generator=_gen(T + i)).to(cuda) for i in range(2))
            before = [t.clone() for t in state[0].views(state.n)]
            rows = state[0].extend(k, v)
            for r, old, new in zip(rows, before, (k, v)):
                assert r.shape == (B, H, state.n + T, D) and r.dtype == BF16
                assert torch.equal(r[:, :, : state.n], old) and torch.equal(r[:, :, state.n:], new.to(BF16))
            state.advance(T)
    mixer = FullRelation(H * D, H, 0, device=cuda).to(BF16)
    state = ArenaState(RelationArena4(1, H, 64, D, cuda, BF16, batch=B))
    with torch.no_grad():
        _, layer = mixer(torch.randn(B, 9, H * D, generator=_gen(70)).to(BF16).to(cuda), cache=state[0], return_cache=True)
    assert not any(torch.is_tensor(getattr(layer, n, None)) for c in type(layer).__mro__ for n in getattr(c, "__slots__", ()))
    assert all(torch.equal(a, b) for a, b in zip(layer.views(9), cache4_read(state.arena.cache(0), D, 0, 9)))


# ---- sizes at a launch's limit -----------------------------------------------------------------------
def test_more_rows_than_one_launch_quantises(cuda):
    """Past 2^28 rows: the codes and scales of every row, and products of the first rows, the last ones and those
    beside the borders between launches."""
    from mote_amd.int8 import int8_linear, int8_weight, quantize_rows

    M = (1 << 28) + 5
    x = torch.empty(M, 1, device=cuda, dtype=BF16)
    for a in range(0, M, 1 << 25):  # whole numbers up to 125: exact in bf16
        n = min(1 << 25, M - a)
        x[a: a + n, 0] = (torch.arange(a, a + n, device=cuda) % 251 - 125).to(BF16)
    q, s = quantize_rows(x)
    for a in range(0, M, 1 << 25):
        part, b = x[a: a + (1 << 25), 0].float(), min(a + (1 << 25), M)
        assert torch.equal(q[a:b, 0].float(), 127 * part.sign()), a
        assert torch.equal(s[a:b], torch.div(part.abs(), torch.full_like(part, 127.0))), a
        assert (q[a: a + 1000, 1:] == 0).all() and (q[b - 1000: b, 1:] == 0).all()
    del q, s
    w8 = int8_weight(torch.tensor([[3.0]], device=cuda))
    y = int8_linear(x, w8)
    for a in (0, *range((1 << 25) - 8, M, 1 << 25), M - 16):
        assert torch.equal(y[a: a + 16], int8_linear(x[a: a + 16], w8)), a


# ---- every form that a rule on sizes selects ------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,N,K", [
    (200, 300, 900),     # 32 x 16 tiles, a ring of four
    (515, 1111, 1000),   # 64 x 32, four
    (1010, 1990, 1500),  # 128 x 64, four
    (2000, 2000, 1100),  # 128 x 128, four
    (2040, 2300, 520),   # 128 x 64, two
    (2890, 2290, 600),   # 128 x 128, two
    (4961, 2290, 700),   # 256 x 192
    (16370, 2300, 640),  # 192 x 256
    (16384, 2304, 768),  # 192 x 256, no tail
    (8100, 4090, 1000),  # 256 x 256
])
def test_every_tile_in_its_steady_state(cuda, dtype, M, N, K):
    """Each tile that the rule picks (at 256 CUs), with more stages than its ring has, so that slots are filled
    again, and with tails of tokens and channels. y is the exact sum of the codes' products, converted to fp32,
    times the two scales, each step rounded once: nothing is left open, so every value is compared bit for bit."""
    from mote_amd.int8 import int8_linear, int8_weight, quantize_rows

    x = (torch.randn(M, K, generator=_gen(M)) * (1 + 5 * (torch.arange(K) % 97 == 0))).to(dtype).to(cuda)
    w = int8_weight((torch.randn(N, K, generator=_gen(N)) * 0.05).to(cuda))
    q, s = quantize_rows(x)
    y = int8_linear(x, w)
    wd = w.q.double().t().contiguous()
    for a in range(0, M, 4096):
        acc = torch.mm(q[a: a + 4096].double(), wd).float()
        assert torch.equal(y[a: a + 4096], (acc * s[a: a + 4096, None] * w.scale).to(dtype)), a
    buf = torch.full((M, N + 33), 9.0, device=cuda, dtype=dtype)  # rows that share cache lines
    int8_linear(x, w, out=buf[:, 5: N + 5])
    assert torch.equal(buf[:, 5: N + 5], y) and (buf[:, :5] == 9).all() and (buf[:, N + 5:] == 9).all()


@pytest.mark.parametrize("dtype,T", [(BF16, 4300), (F32, 2200)])
def test_rows_that_pass_the_caches_by(cuda, dtype, T):
    """100 MB and more of rows in one call (read past the caches) store what smaller calls store, bit for bit."""
    from mote_amd.cache4 import cache4_write, cache4_zeros

    B, H, D = 8, 8, 96
    assert 2 * B * H * T * D * (2 if dtype == BF16 else 4) >= 100e6
    k, v = (torch.randn(B, T, H, D, generator=torch.Generator(device=cuda).manual_seed(i), device=cuda).to(dtype).transpose(1, 2)
            for i in range(2))
    v[3, 2, 7, 11] = float("inf")
    once, parts = cache4_zeros(B, H, T + 9, D, cuda), cache4_zeros(B, H, T + 9, D, cuda)
    start, lens = torch.arange(B, device=cuda), T - 100 * torch.arange(B, device=cuda)
    cache4_write(once, k, v, start, lens)
    for a in range(0, T, 1000):
        cache4_write(parts, k[:, :, a: a + 1000], v[:, :, a: a + 1000], start + a, lens - a)
    for x, y in zip(once, parts):
        assert torch.equal(x.view(torch.uint8), y.view(torch.uint8)) and x.view(torch.uint8).any()


# ---- the decode step over an arena in 4 bits with its projections as they are --------------------------------
def _mixer(cuda, d, H, layer, dtype, **kw):
    from mote_amd.relation import FullRelation

    torch.manual_seed(d + layer)
    m = FullRelation(d, H, layer, device=cuda, **kw).to(dtype)
    with torch.no_grad():
        m.lam.fill_(0.4)
        m.theta.copy_(torch.rand(H // 2) * 0.6 - 0.3)
    return m


def _token_by_hand(m, x, S, cache, arena_dtype):
    """One step from the public operators: the skinny product where it applies, else F.linear."""
    import torch.nn.functional as F

    from mote_amd.cache4 import relation_decode4
    from mote_amd.decode import skinny_linear

    B, _, d = x.shape
    H, dh = m.n_heads, m.d_head
    w = torch.cat([m.w1.weight, m.w2.weight, m.wi.weight])
    skinny = x.dtype == BF16 and B <= 16 and d % 128 == 0
    qkv = (skinny_linear(x.reshape(B, d), w) if skinny else F.linear(x, w)).view(B, 3, H, dh).to(arena_dtype)
    if m.qk_norm:
        qkv = torch.stack([m.p1_norm(qkv[:, 0]), m.p2_norm(qkv[:, 1]), qkv[:, 2]], 1)
    y, g = relation_decode4(qkv[:, 0], qkv[:, 1], qkv[:, 2], S, cache, m.lam, m.tau_s, m.inv_freq, m.theta, m.layer_idx,
                            rope_f32=x.dtype == F32 and arena_dtype != F32)
    y = y.to(x.dtype)
    if not skinny:
        return m._out(y.view(B, H, 1, dh), x), g
    y = y.reshape(B, H * dh)
    if m.out_gate:
        y = y * torch.sigmoid(skinny_linear(x.reshape(B, d), m.wg.weight))
    return skinny_linear(y, m.wo.weight).view(B, 1, d), g


@pytest.mark.parametrize("d,H,B,x_dtype,arena_dtype,kw", [
    (512, 8, 2, BF16, BF16, dict(qk_norm=True, out_gate=True)), (768, 8, 16, BF16, BF16, {}), (192, 4, 3, BF16, BF16, {}),
    (512, 8, 20, BF16, BF16, dict(out_gate=True)), (192, 4, 1, F32, F32, {}), (512, 8, 2, F32, BF16, {})])
def test_steps_over_four_bits_with_the_layers_own_projections(cuda, d, H, B, x_dtype, arena_dtype, kw):
    """Prompts of two layers, then steps through RelationMainStep, the arena growing on the way: the tokens, the
    exchange masses and the arena are those of the operators put together by hand."""
    from mote_amd.arena import ArenaState
    from mote_amd.arena4 import RelationArena4
    from mote_amd.cache4 import Cache4
    from mote_amd.graph import RelationMainStep

    mixers = [_mixer(cuda, d, H, i, x_dtype, **kw) for i in range(2)]
    arena = RelationArena4(2, H, 64, d // H, cuda, arena_dtype, batch=B)
    state = ArenaState(arena)
    with torch.no_grad():
        h = torch.randn(B, 60, d, generator=_gen(1)).to(x_dtype).to(cuda)
        for i, m in enumerate(mixers):
            h = m(h, cache=state[i])
        state.advance(60)
        arena.claim(1, 60) if B == 1 else None
        S = torch.full((B,), 60, device=cuda)
        twin, St, xm = [Cache4(*(t.clone() for t in arena.cache(i))) for i in range(2)], S.clone(), torch.empty(2, B, device=cuda)
        step = RelationMainStep(arena, S, xm)
        for t in range(5):
            if t == 2:
                arena.claim(1, 62) if B == 1 else None
                arena.ensure(100)
                grow = lambda c: torch.cat([c, torch.zeros_like(c)], 2)
                twin = [Cache4(*(grow(c) for c in layer)) for layer in twin]
            x = xt = torch.randn(B, 1, d, generator=_gen(100 + t)).to(x_dtype).to(cuda)
            for i, m in enumerate(mixers):
                x = step(m, x, li=i)
                xt, g = _token_by_hand(m, xt, St, twin[i], arena_dtype)
                assert torch.equal(x, xt), (t, i)
                # H additions and a division of numbers up to 1
                assert torch.allclose(xm[i], g.mean(1), rtol=2 * (H + 1) * 2.0 ** -24, atol=0)
            St += 1
            assert torch.equal(S, St)
    for i in range(2):
        assert all(torch.equal(a, b) for a, b in zip(arena.cache(i), twin[i]))


def test_captured_token_over_four_bits(cuda):
    """One graph of a two-layer token with bf16 projections, replayed with the router's bit on and off and other work
    in between, against eager steps."""
    from mote_amd.arena4 import RelationArena4
    from mote_amd.graph import RelationMainStep

    d, H, B = 512, 8, 2
    mixers = [_mixer(cuda, d, H, i, BF16, out_gate=True) for i in range(2)]
    a, b = (RelationArena4(2, H, 128, d // H, cuda, BF16, batch=B) for _ in range(2))
    Sa, Sb = torch.tensor([0, 5], device=cuda), torch.tensor([0, 5], device=cuda)
    run, x = torch.ones(1, dtype=torch.bool, device=cuda), torch.randn(B, 1, d, generator=_gen(0)).to(BF16).to(cuda)
    sa, sb = RelationMainStep(a, Sa, run=run), RelationMainStep(b, Sb)

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
        x.copy_(torch.randn(B, 1, d, generator=_gen(50 + t)).to(BF16))
        run.fill_(t % 3 != 1)
        graph.replay()
        if t % 3 != 1:
            want = token(sb, x)
        torch.cuda.synchronize()
        assert torch.equal(Sa, Sb) and torch.equal(a.store, b.store) and torch.equal(a.scales, b.scales)
        assert torch.equal(out, want)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_both_outputs_in_one_buffer(cuda, dtype):
    """The two outputs of a read as columns, as alternate rows and as halves of one buffer."""
    from mote_amd.cache4 import cache4_read

    B, H, T, D = 2, 4, 10, 48
    _, _, cache = _step_inputs(cuda, 80, B, H, D, 64)
    want = cache4_read(cache, D, 3, T, dtype=dtype)
    new = lambda *s: torch.full(s, 9.0, device=cuda, dtype=dtype)
    side, turned, long, inner = new(B, H, T, 2 * D), new(B, T, H, 2 * D).transpose(1, 2), new(B, H, 2 * T, D), new(B, 3, H, T, D)
    for out in ((side[..., :D], side[..., D:]), (turned[..., D:], turned[..., :D]), (long[:, :, ::2], long[:, :, 1::2]),
                (inner[:, 0], inner[:, 2])):
        got = cache4_read(cache, D, 3, T, out=out)
        assert all(torch.equal(a, b) for a, b in zip(got, want)) and all(torch.equal(a, b) for a, b in zip(out, want))
    assert (inner[:, 1] == 9).all()


def test_windows_of_another_type_than_the_arena(cuda):
    """An fp32 layer over an arena of bf16 rows in 4 bits: two windows, against the operators put together by hand."""
    from mote_amd.arena import ArenaState
    from mote_amd.arena4 import RelationArena4
    from mote_amd.cache4 import cache4_read
    from mote_amd.flash_relation import flash_relation

    d, H, B = 192, 4, 2
    m = _mixer(cuda, d, H, 1, F32)
    arena = RelationArena4(1, H, 128, d // H, cuda, BF16, batch=B)
    state = ArenaState(arena)
    with torch.no_grad():
        for T in (50, 1, 30):
            x, n = torch.randn(B, T, d, generator=_gen(T)).to(cuda), state.n
            held = cache4_read(arena.cache(0), d // H, 0, n)
            q, k, v = (t.to(BF16) for t in m.heads(x, n))
            y, g = flash_relation(q, torch.cat([held[0], k], 2), torch.cat([held[1], v], 2), m.lam, m.tau_s, q_start=n)
            out, gates = m(x, cache=state[0], return_gates=True)
            assert torch.equal(out, m._out(y.to(F32), x)) and torch.equal(gates, g)
            state.advance(T)
