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
