"""What the quantised operators' entry points refuse at the edges of what a call may pass, on the CPU: calls that
would write one place twice, sizes beyond a launch, derivatives that they do not carry, growth that fails."""

from __future__ import annotations

import pytest
import torch

from mote_amd import _lib as L

pytestmark = pytest.mark.skipif(not L.available(), reason="libmote_relation.so not built")

BF16 = torch.bfloat16


def _cache(B=2, H=4, cap=64, D=48):
    from mote_amd.cache4 import cache4_zeros

    return cache4_zeros(B, H, cap, D, "cpu")


def _layouts(B, H, T, D):
    """Pairs of views [B, H, T, D] for the two outputs, and whether they may be written together."""
    new = lambda *s: torch.zeros(*s, dtype=BF16)
    flat = new(4 * B * H * T * D)
    view = lambda strides, at=0: flat.as_strided((B, H, T, D), strides, at)
    dense = (H * T * D, T * D, D, 1)
    two = new(2, B, H, T, D)
    side = new(B, H, T, 2 * D)
    inner = new(B, 2, H, T, D)
    turned = new(B, T, H, 2 * D).transpose(1, 2)
    long = new(B, H, 2 * T, D)
    yield (two[0], two[1]), True
    yield (side[..., :D], side[..., D:]), True
    yield (side[..., D:], side[..., :D]), True
    yield (inner[:, 0], inner[:, 1]), True
    yield (turned[..., :D], turned[..., D:]), True
    yield (long[:, :, :T], long[:, :, T:]), True
    yield (long[:, :, ::2], long[:, :, 1::2]), True
    yield (view(dense), view((T * D, B * T * D, D, 1), B * H * T * D)), True
    yield (two[0], two[0]), False                                          # one tensor twice
    yield (long[:, :, :T], long[:, :, 8: 8 + T]), False                    # some rows twice
    yield (view(dense), view(dense, 8)), False                             # a chunk apart
    yield (view(dense), view((T * D, B * T * D, D, 1))), False             # the same range in another order
    yield (view((H * T * 8, T * 8, 8, 1)), two[0]), False                  # rows closer than they are long
    yield (two[0], view((H * T * D, 8, H * D, 1))), False                  # heads closer than they are wide
    yield (two[0], view((T * D, T * D, D, 1))), False                      # sequences over heads


def test_read_refuses_outputs_that_share_places():
    from mote_amd.cache4 import Cache4, cache4_read

    c = _cache()
    for out, fine in _layouts(2, 4, 10, 48):
        with pytest.raises(RuntimeError if fine else ValueError, match="MI355X" if fine else "out"):
            cache4_read(c, 48, 0, 10, out=out)
    pool = torch.zeros(2 * 4 * 64 * 64 * 2, dtype=torch.uint8)
    over = c._replace(p2=pool[: c.p2.numel()].view(c.p2.shape))
    out = pool[c.p2.numel() // 2:][: 2 * 4 * 10 * 48 * 2].view(BF16).view(2, 4, 10, 48)
    with pytest.raises(ValueError, match="over the cache"):
        cache4_read(Cache4(*over), 48, 0, 10, out=(out, torch.zeros_like(out)))
    after = pool[c.p2.numel():][: 2 * 4 * 10 * 48 * 2].view(BF16).view(2, 4, 10, 48)
    with pytest.raises(RuntimeError, match="MI355X"):
        cache4_read(Cache4(*over), 48, 0, 10, out=(after, torch.zeros_like(out)))
    none = torch.zeros(2, 4, 0, 48, dtype=BF16)
    with pytest.raises(RuntimeError, match="MI355X"):
        cache4_read(c, 48, 0, 0, out=(none, none))


def test_caches_that_share_rows_are_not_written():
    from mote_amd.arena4 import RelationArena4
    from mote_amd.cache4 import Cache4, cache4_write, relation_decode4

    B, H, cap, D = 2, 4, 64, 48
    rows = torch.zeros(B, H, 8, D, dtype=BF16)
    x, S, lam = torch.zeros(B, H, D, dtype=BF16), torch.zeros(B, dtype=torch.int64), torch.tensor(0.5)

    def refused(cache, match):
        for call in (lambda: cache4_write(cache, rows, rows), lambda: relation_decode4(x, x, x, S, cache, lam)):
            with pytest.raises(RuntimeError if match == "MI355X" else ValueError, match=match):
                call()

    c = _cache(B, H, cap, D)
    close = torch.zeros(B * H * cap * 32, dtype=torch.uint8).as_strided(c.p2.shape, (H * cap * 32, 32, 32, 1))
    refused(c._replace(p2=close, info=close.clone().as_strided(c.p2.shape, close.stride())), "several heads")
    over = torch.zeros(3, H, cap, 32, dtype=torch.uint8)
    refused(c._replace(p2=over[:2], info=over[1:]), "same rows")
    scales = torch.zeros(B, H + 1, cap, 2, dtype=BF16)
    refused(c._replace(p2_scale=scales[:, :H], info_scale=scales[:, 1:]), "same rows")
    # disjoint parts of one store
    refused(RelationArena4(2, H, cap, D, "cpu", batch=B).cache(1), "MI355X")
    both = [torch.zeros(B, 2, H, cap, w, dtype=dt) for w, dt in ((32, torch.uint8), (2, BF16))]
    refused(Cache4(both[0][:, 0], both[1][:, 0], both[0][:, 1], both[1][:, 1]), "MI355X")


def test_c_entry_points_refuse_caches_that_share_rows():
    lib = L.lib()
    B, H, cap, D, G = 3, 4, 64, 48, 2

    def rows(cache):
        r = L.Cache4RowsArgs()
        r.dtype, r.B, r.H, r.T, r.D, r.capacity = L.MOTE_BF16, B, H, 4, D, cap
        r.p2.data = r.info.data = 16
        r.p2.stride_r = r.info.stride_r = D
        r.cache = cache
        return lib.mote_cache4_write(r, None)

    def step(cache):
        a = L.Decode4Args()
        a.dtype, a.B, a.H, a.D, a.capacity = L.MOTE_BF16, B, H, D, cap
        a.lam = a.S = a.p1 = a.p2 = a.info = a.y = a.g = a.workspace = 16
        a.workspace_bytes = int(lib.mote_relation_decode4_workspace(a))
        a.cache = cache
        return lib.mote_relation_decode4(a, None)

    block, head = 16 * G * cap, G * cap
    for sb, sh in ((0, block), (H * block, block - 16), (H * block - 16, block), (block, B * block - 16), (block - 16, H * block)):
        for codes in (True, False):
            c = L.Cache4View()
            c.p2 = c.info = c.p2_scale = c.info_scale = 16
            c.codes_sb, c.codes_sh = (sb, sh) if codes else (H * block, block)
            c.scale_sb, c.scale_sh = (H * head, head) if codes else (sb // 16, sh // 16)
            for call in (rows, step):
                assert call(c) == 1 and b"share rows" in lib.mote_last_error(), (sb, sh, codes, call)


def test_sizes_beyond_a_launch_are_refused():
    """A grid holds fewer than 2^32 threads: what needs more is refused before anything is launched."""
    lib = L.lib()
    w = L.Int8LinearArgs()
    w.dtype, w.x, w.wq, w.w_scale, w.y, w.workspace, w.workspace_bytes = L.MOTE_BF16, *(16,) * 5, 1 << 62
    for M, N, K in ((1, 1 << 28, 128), (16, 1 << 27, 2048), (1 << 20, 1 << 19, 64), (1 << 30, 1 << 13, 1)):
        w.M, w.N, w.K, w.x_sr, w.y_sr = M, N, K, K, N
        assert lib.mote_int8_linear(w, None) == 2 and b"for one launch" in lib.mote_last_error(), (M, N, K)
    a = L.Decode4Args()
    a.dtype, a.B, a.H, a.D, a.capacity = L.MOTE_BF16, 1 << 23, 2, 8, 1
    a.lam = a.S = a.p1 = a.p2 = a.info = a.y = a.g = a.workspace = 16
    a.workspace_bytes = int(lib.mote_relation_decode4_workspace(a))
    a.cache.p2 = a.cache.info = a.cache.p2_scale = a.cache.info_scale = 16
    a.cache.codes_sb, a.cache.codes_sh, a.cache.scale_sb, a.cache.scale_sh = 32, 16, 2, 1
    assert lib.mote_relation_decode4(a, None) == 2 and b"for one launch" in lib.mote_last_error()


def test_more_rows_than_32_bits_count_are_refused():
    """With device positions the capacity does not bound the number of rows: one that 32 bits cannot hold is
    refused, not cut."""
    from mote_amd.cache4 import cache4_read, cache4_write

    c, start = _cache(1, 2, 64, 48), torch.zeros(1, dtype=torch.int64)
    for T in (1 << 31, (1 << 32) + 4):
        rows = torch.zeros(1, 2, 1, 48, dtype=BF16).expand(1, 2, T, 48)
        with pytest.raises(ValueError, match="32 bits"):
            cache4_write(c, rows, rows, start)
        with pytest.raises(ValueError, match="32 bits"):
            cache4_read(c, 48, start, T)
    one = [t[:1, :1, :1, :].expand(1 << 32, 1, 1, t.shape[3]) for t in c]
    with pytest.raises(ValueError, match="32 bits"):
        cache4_read(type(c)(*one), 48)


def test_tangents_are_refused():
    """Forward-mode derivatives are not dropped in silence, under no_grad neither (which leaves forward mode on)."""
    from mote_amd.cache4 import cache4_read, cache4_write, relation_decode4
    from mote_amd.int8 import Int8Weight, int8_linear, quantize_rows

    fwd = torch.autograd.forward_ad
    c, S, lam = _cache(), torch.zeros(2, dtype=torch.int64), torch.tensor(0.5)
    rows, x = torch.zeros(2, 4, 8, 48, dtype=BF16), torch.zeros(2, 4, 48, dtype=BF16)
    w, t = Int8Weight(torch.zeros(16, 128, dtype=torch.int8), torch.zeros(16), 48), torch.zeros(4, 48)
    with fwd.dual_level():
        dual = lambda v: fwd.make_dual(v, torch.ones_like(v))
        calls = [lambda: cache4_write(c, dual(rows), rows), lambda: cache4_write(c, rows, dual(rows)),
                 lambda: relation_decode4(dual(x), x, x, S, c, lam), lambda: relation_decode4(x, x, dual(x), S, c, lam),
                 lambda: cache4_read(c, 48, 0, 8, out=(dual(rows), rows.clone())),
                 lambda: quantize_rows(dual(t)), lambda: int8_linear(dual(t), w)]
        for grad in (True, False):
            for call in calls:
                with torch.set_grad_enabled(grad), pytest.raises(RuntimeError, match="forward-mode"):
                    call()
        with pytest.raises(RuntimeError, match="MI355X"):
            int8_linear(t, w)
        with fwd._set_fwd_grad_enabled(False), pytest.raises(RuntimeError, match="MI355X"):
            int8_linear(dual(t), w)


def test_parameters_and_outputs_that_want_a_gradient_are_refused():
    from mote_amd.cache4 import relation_decode4
    from mote_amd.int8 import Int8Weight, int8_linear

    c, S = _cache(), torch.zeros(2, dtype=torch.int64)
    x, want = torch.zeros(2, 4, 48, dtype=BF16), lambda *s, dt=torch.float32: torch.zeros(*s, dtype=dt, requires_grad=True)
    args = dict(lam=torch.tensor(0.5))
    w, t = Int8Weight(torch.zeros(16, 128, dtype=torch.int8), torch.zeros(16), 48), torch.zeros(2, 48)
    calls = [(lambda **kw: relation_decode4(x, x, x, S, c, **{**args, **kw}), name, value) for name, value in
             (("lam", want(())), ("inv_freq", want(24)), ("theta", want(2)), ("y", want(2, 4, 48, dt=BF16)),
              ("g", want(2, 4)), ("xm", want(2)))]
    calls += [(lambda **kw: int8_linear(t, **{"w": w, **kw}), name, value) for name, value in
              (("w", w._replace(scale=want(16))), ("out", want(2, 16)))]
    calls += [(lambda **kw: int8_linear(t, w, **{"g": torch.zeros(2, 4), "xm": torch.zeros(2), **kw}), name, value) for name, value in
              (("g", want(2, 4)), ("xm", want(2)))]
    for call, name, value in calls:
        with pytest.raises(RuntimeError, match="no backward"):
            call(**{name: value})
        with torch.no_grad(), pytest.raises(RuntimeError, match="MI355X"):
            call(**{name: value})


@pytest.mark.parametrize("batch", [1, 2])
@pytest.mark.parametrize("fails", [torch.uint8, torch.bfloat16])
def test_a_growth_that_fails_leaves_the_arena_as_it_was(monkeypatch, batch, fails):
    from mote_amd import arena4

    a = arena4.RelationArena4(2, 2, 16, 32, "cpu", batch=batch)
    a.store.random_(0, 256)
    a.scales.copy_(torch.rand(a.scales.shape))
    a.claim(9, 10) if batch == 1 else None
    before = [t.clone() for t in (*a.cache(0), *a.cache(1))]
    zeros = torch.zeros

    def no_memory(*size, **kw):
        if kw.get("dtype") == fails:
            raise torch.OutOfMemoryError("out of memory")
        return zeros(*size, **kw)

    with monkeypatch.context() as m:
        m.setattr(torch, "zeros", no_memory)
        with pytest.raises(torch.OutOfMemoryError):
            a.ensure(17)
    assert a.capacity == 16 and a.generation == 0
    assert all(torch.equal(x, y) for x, y in zip((*a.cache(0), *a.cache(1)), before))
    assert a.ensure(17) and a.capacity == 32 and a.scales.shape[4] == 32
    assert all(torch.equal(x[:, :, :10], y[:, :, :10]) for x, y in zip((*a.cache(0), *a.cache(1)), before))


def test_the_steps_of_the_model_type_refuse_tangents_too():
    from mote_amd.decode import relation_decode, skinny_linear

    fwd = torch.autograd.forward_ad
    x, S, lam = torch.zeros(2, 4, 48, dtype=BF16), torch.zeros(2, dtype=torch.int64), torch.tensor(0.5)
    rows, w = torch.zeros(2, 4, 64, 48, dtype=BF16), torch.zeros(16, 128, dtype=BF16)
    with fwd.dual_level(), torch.no_grad():
        dual = lambda v: fwd.make_dual(v, torch.ones_like(v))
        for call in (lambda: relation_decode(dual(x), x, x, S, rows, rows, lam), lambda: relation_decode(x, x, x, S, rows, rows, dual(lam)),
                     lambda: skinny_linear(dual(w[:4]), w), lambda: skinny_linear(w[:4], dual(w))):
            with pytest.raises(RuntimeError, match="forward-mode"):
                call()
        with pytest.raises(RuntimeError, match="MI355X"):
            relation_decode(x, x, x, S, rows, rows, lam)
