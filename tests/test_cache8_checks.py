"""What the paged 8-bit cache's, its pages' and the draw's entry points refuse, on the CPU: a bad call raises before
anything could be launched."""

from __future__ import annotations

import ctypes as C

import pytest
import torch

from mote_amd import _lib as L

pytestmark = pytest.mark.skipif(not L.available(), reason="libmote_relation.so not built")

BF16 = torch.bfloat16


def _cache(B=2, H=4, pages=5, rows=128, D=48, dtype=BF16):
    from mote_amd.cache8 import cache8_zeros

    return cache8_zeros(B, H, pages, rows, D, "cpu", dtype)


def _rows(B=2, H=4, T=8, D=48, dtype=BF16):
    return torch.zeros(B, H, T, D, dtype=dtype), torch.zeros(B, H, T, D, dtype=dtype)


def test_layout():
    c = _cache(D=40, rows=100)
    assert [tuple(t.shape) for t in c] == [(5, 4, 3, 64, 16), (5, 4), (5, 4, 48, 64), (5, 4), (2, 4, 64, 40), (2, 4, 64, 40), (2, 2)]
    assert (c.table == -1).all()
    for D in (0, 4, 50, 136):
        with pytest.raises(ValueError, match="head dim"):
            _cache(D=D)
    with pytest.raises(ValueError, match="0 pages"):
        _cache(pages=0)


def test_write_refuses():
    from mote_amd.cache8 import cache8_write

    c = _cache()
    k, v = _rows()
    with pytest.raises(ValueError, match="p2 and info"):
        cache8_write(c, k, v[:, :, :4])
    with pytest.raises(TypeError):
        cache8_write(c, k, v.float())
    with pytest.raises(TypeError):
        cache8_write(c, k.half(), v.half())
    with pytest.raises(TypeError, match="tails"):
        cache8_write(c, k.float(), v.float())
    with pytest.raises(ValueError, match="head dim"):
        cache8_write(c, *_rows(D=44))
    with pytest.raises(ValueError, match="pages of P2"):
        cache8_write(c, *_rows(D=96))
    with pytest.raises(ValueError, match="pages of P2"):
        cache8_write(c, *_rows(H=2))
    with pytest.raises(ValueError, match="tails of P2"):
        cache8_write(c, *_rows(B=3))
    for start in (-1, 121, 128):
        with pytest.raises(RuntimeError, match="table of 128"):
            cache8_write(c, k, v, start)
    for bad in (torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)):
        with pytest.raises(ValueError, match="start"):
            cache8_write(c, k, v, bad)
        with pytest.raises(ValueError, match="lens"):
            cache8_write(c, k, v, 0, bad)
    with pytest.raises(RuntimeError, match="no backward"):
        cache8_write(c, k.requires_grad_(True), v)
    with pytest.raises(RuntimeError, match="MI355X"):
        cache8_write(c, k.detach(), v)
    with pytest.raises(ValueError, match="over the cache"):
        cache8_write(c, c.p2_tail[:, :, :8], v)


def test_cache_layouts_that_are_refused():
    from mote_amd.cache8 import cache8_read, cache8_write

    c = _cache()
    k, v = _rows()
    bad = dict(
        p2=[torch.zeros(5, 4, 3, 64, 32, dtype=torch.uint8)[..., :16], c.p2[:1].expand(5, -1, -1, -1, -1), c.info.view(5, 4, 3, 64, 16)],
        info=[c.p2, torch.zeros(10, 4, 48, 64, dtype=torch.uint8)[::2]],
        p2_scale=[c.p2_scale[:3], c.info_scale, torch.zeros(4, 5).t()],
        info_tail=[c.p2_tail, c.info_tail[:, :2], torch.zeros(2, 64, 4, 48, dtype=BF16).transpose(1, 2), c.info_tail[:1].expand(2, -1, -1, -1)],
        table=[c.table[0], torch.zeros(2, 2, 2, dtype=torch.int32), torch.zeros(3, 2, dtype=torch.int32),
               torch.zeros(2, 4, dtype=torch.int32)[:, ::2], torch.zeros(2, 0, dtype=torch.int32)])
    for name, values in bad.items():
        for value in values:
            with pytest.raises(ValueError):
                cache8_write(c._replace(**{name: value}), k, v)
    for name, value in dict(p2=c.p2.to(torch.int8), p2_scale=c.p2_scale.to(BF16), table=c.table.long(), info_tail=c.info_tail.float(),
                            p2_tail=c.p2_tail.half()).items():
        with pytest.raises(TypeError):
            cache8_write(c._replace(**{name: value}), k, v)
    with pytest.raises(ValueError, match="seven"):
        L.native().cache8_write(list(c)[:6], k, v, 0, None, None)
    one = c._replace(p2=c.p2[:1].expand(5, -1, -1, -1, -1), info=c.info[:1].expand(5, -1, -1, -1))
    with pytest.raises(RuntimeError, match="MI355X"):
        cache8_read(one, 10)  # reading shared rows is fine: only the device is missing


def test_read_refuses():
    from mote_amd.cache8 import cache8_read

    c = _cache()
    for held in (-1, 129):
        with pytest.raises(RuntimeError, match="held"):
            cache8_read(c, held)
    with pytest.raises(RuntimeError, match="rows from -1"):
        cache8_read(c, 10, -1)
    with pytest.raises(ValueError, match="rows"):
        cache8_read(c, 10, 0, -1)
    dev = torch.zeros(2, dtype=torch.int64)
    for args in ((dev,), (10, dev)):
        with pytest.raises(ValueError, match="number of rows"):
            cache8_read(c, *args)
    for args in ((dev.int(), 0), (10, dev[:1])):
        with pytest.raises(ValueError, match="contiguous int64"):
            cache8_read(c, *args, rows=4)
    with pytest.raises(TypeError):
        cache8_read(c, 10, dtype=torch.float16)
    with pytest.raises(ValueError, match="out"):
        cache8_read(c, 10, 0, 8, out=_rows(T=9))
    with pytest.raises(ValueError, match="several places"):
        cache8_read(c, 10, 0, 8, out=tuple(t[:, :, :1].expand(t.shape) for t in _rows()))
    with pytest.raises(ValueError, match="over the cache"):
        cache8_read(c, 10, 0, 8, out=(c.p2_tail[:, :, :8], _rows()[0]))
    x = _rows()[0]
    with pytest.raises(ValueError, match="over one another"):
        cache8_read(c, 10, 0, 8, out=(x, x))
    with pytest.raises(RuntimeError, match="gradient"):
        cache8_read(c, 10, 0, 8, out=tuple(t.requires_grad_(True) for t in _rows()))
    with pytest.raises(RuntimeError, match="no backward"):
        cache8_read(c._replace(p2_tail=c.p2_tail.clone().requires_grad_(True)), 10)
    with pytest.raises(RuntimeError, match="MI355X"):
        cache8_read(c, 10)


def test_decode8_refuses():
    from mote_amd.cache8 import relation_decode8

    c = _cache()
    x = torch.zeros(2, 4, 48, dtype=BF16)
    S, lam = torch.zeros(2, dtype=torch.int64), torch.tensor(0.5)
    with pytest.raises(ValueError, match="head stride"):
        relation_decode8(x, x, x.transpose(1, 2).contiguous().transpose(1, 2), S, c, lam)
    with pytest.raises(ValueError, match="head stride"):
        relation_decode8(x, x[:1], x, S, c, lam)
    with pytest.raises(TypeError):
        relation_decode8(x, x, x.float(), S, c, lam)
    with pytest.raises(TypeError):
        relation_decode8(x.half(), x.half(), x.half(), S, c, lam)
    with pytest.raises(TypeError, match="tails"):
        relation_decode8(x.float(), x.float(), x.float(), S, c, lam)
    for s in (S.int(), S[:1], torch.zeros(4, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError, match="S must"):
            relation_decode8(x, x, x, s, c, lam)
    with pytest.raises(ValueError, match="tails of P2"):
        relation_decode8(x, x, x, S, _cache(B=1), lam)
    y3 = torch.zeros(2, 3, 48, dtype=BF16)
    with pytest.raises(ValueError, match="even"):
        relation_decode8(y3, y3, y3, S, _cache(H=3), lam)
    bad = dict(inv_freq=torch.zeros(23), theta=torch.zeros(4), xm=torch.zeros(3), run=torch.zeros(2, dtype=torch.bool),
               y=torch.zeros(2, 4, 48), g=torch.zeros(2, 4, dtype=BF16), workspace=torch.zeros(64, dtype=torch.uint8)[::2])
    for name, value in bad.items():
        with pytest.raises(ValueError, match=name):
            relation_decode8(x, x, x, S, c, lam, **{name: value})
    qkv = torch.zeros(2, 3, 4, 48, dtype=BF16)
    with pytest.raises(ValueError, match="lies over an input"):
        relation_decode8(qkv[:, 0], qkv[:, 1], qkv[:, 2], S, c, lam, y=qkv[:, 2])
    with pytest.raises(ValueError, match="over the cache"):
        relation_decode8(x, x, x, S, c, lam, y=c.p2_tail[0].view(-1)[: 2 * 4 * 48].view(2, 4, 48))
    with pytest.raises(RuntimeError, match="no backward"):
        relation_decode8(x, x, x, S, c, torch.nn.Parameter(torch.tensor(0.5)))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="dual"):
        relation_decode8(torch.autograd.forward_ad.make_dual(x, x), x, x, S, c, lam)
    with pytest.raises(RuntimeError, match="MI355X"):
        relation_decode8(x, x, x, S, c, lam)


def test_the_c_entries_refuse():
    """Sizes, pointers and strides that a kernel could not walk, from the library itself."""
    lib = L.lib()
    a = L.Decode8Args()
    a.dtype, a.B, a.H, a.D, a.tau_s = L.MOTE_BF16, 2, 4, 48, 2.0
    for f in ("lam", "S", "p1", "p2", "info", "y", "g", "workspace"):
        setattr(a, f, 16)
    c = a.cache
    for f in ("p2", "p2_scale", "info", "info_scale", "p2_tail", "info_tail", "table"):
        setattr(c, f, 16)
    c.pages, c.blocks, c.codes_sp, c.scale_sp, c.tail_sb, c.table_sb = 5, 2, 4 * 64 * 48, 4, 4 * 64 * 48, 2
    need = int(lib.mote_relation_decode8_workspace(a))
    assert need > 0 and need % 32 == 0
    a.workspace_bytes = need - 1
    assert lib.mote_relation_decode8(a, None) == 3
    for f, v, rc in (("codes_sp", 4 * 64 * 48 - 16, 1), ("codes_sp", 4 * 64 * 48 + 8, 1), ("scale_sp", 3, 1), ("tail_sb", 100, 1),
                     ("table_sb", 1, 1), ("pages", 0, 1), ("blocks", 0, 1), ("p2", 24, 1), ("table", None, 1)):
        old = getattr(c, f)
        setattr(c, f, v)
        assert lib.mote_relation_decode8(a, None) == rc, f
        setattr(c, f, old)
    for f, v in (("D", 44), ("D", 136), ("H", 3), ("B", 0)):
        old = getattr(a, f)
        setattr(a, f, v)
        assert lib.mote_relation_decode8(a, None) == 2, f
        setattr(a, f, old)
    r = L.Cache8RowsArgs()
    r.dtype, r.tail_dtype, r.B, r.H, r.T, r.D, r.cache = L.MOTE_BF16, L.MOTE_F32, 2, 4, 8, 48, c
    assert lib.mote_cache8_write(r, None) == 1  # rows and tails of two types
    r.tail_dtype = L.MOTE_BF16
    assert lib.mote_cache8_write(r, None) == 1 and b"null" in lib.mote_last_error()
    r.p2.data = r.info.data = 16
    r.p2.stride_r = 4
    assert lib.mote_cache8_write(r, None) == 1 and b"16-byte" in lib.mote_last_error()
    r.T = 0
    assert lib.mote_cache8_write(r, None) == 0  # nothing to do, nothing launched
    assert lib.mote_cache8_read(r, None) == 0
    s = L.SampleArgs()
    s.dtype, s.B, s.V, s.logits, s.u, s.tokens = L.MOTE_F32, 1, 100000, 16, 16, 16
    assert lib.mote_sample(s, None) == 3 and int(lib.mote_sample_workspace(s)) > 0
    s.V = (1 << 20) + 1
    assert lib.mote_sample(s, None) == 2
    s.V, s.B = 100, 0
    assert lib.mote_sample(s, None) == 0 and int(lib.mote_sample_workspace(s)) == 0
    p = L.PagesArgs()
    p.B, p.blocks, p.pages, p.table_sb, p.table, p.refs = 9, 4, 5, 4, 16, 16
    for seqs, word in (([3, 9], b"no sequence 9"), ([2, 5, 2], b"sequence 2 twice"), ([-1], b"no sequence -1")):
        held = (C.c_int32 * len(seqs))(*seqs)
        p.seqs, p.n = C.addressof(held), len(seqs)
        assert lib.mote_pages_free(p, None) == 1 and word in lib.mote_last_error()
    held = (C.c_int32 * 1)(4)
    p.seqs, p.n, p.src, p.S = C.addressof(held), 1, 4, 16
    assert lib.mote_pages_fork(p, None) == 1 and b"is the source" in lib.mote_last_error()
    p.n = 0
    assert lib.mote_pages_free(p, None) == 0 and lib.mote_pages_fork(p, None) == 0  # nothing to do, nothing launched
    assert lib.mote_sample(None, None) == 1 and lib.mote_pages_free(None, None) == 1 and lib.mote_cache8_read(None, None) == 1


def test_pages_refuse():
    from mote_amd.pages import PagePool, pages_compact, pages_fork, pages_free, pages_reserve

    refs, table, S = torch.zeros(6, dtype=torch.int32), torch.full((3, 4), -1, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)
    for seqs, word in (([3], "no sequence 3"), ([-1], "no sequence -1"), ([0, 0], "twice")):
        with pytest.raises(ValueError, match=word):
            pages_free(refs, table, seqs)
        with pytest.raises(ValueError, match=word):
            pages_fork(refs, table, S, 1, seqs)
    with pytest.raises(ValueError, match="source"):
        pages_fork(refs, table, S, 1, [0, 1])
    with pytest.raises(ValueError, match="no sequence 7"):
        pages_fork(refs, table, S, 7, [0])
    for bad in (S[:2], S.int()):
        with pytest.raises(ValueError, match="S must"):
            pages_fork(refs, table, bad, 1, [0])
        with pytest.raises(ValueError, match="rows must"):
            pages_reserve(refs, table, bad)
    tails = torch.zeros(2, 3, 2, 64, 16)
    for bad in (tails[0], tails[:, :2], tails[..., :12], tails.transpose(0, 2), tails[:1].expand(2, -1, -1, -1, -1),
                torch.zeros(2, 3, 2, 64, 136)):
        with pytest.raises(ValueError):
            pages_fork(refs, table, S, 1, [0], bad)
    with pytest.raises(TypeError):
        pages_fork(refs, table, S, 1, [0], tails.half())
    with pytest.raises(RuntimeError, match="no backward"):
        pages_fork(refs, table, S, 1, [0], tails.clone().requires_grad_(True))
    for rows in (-1, 4 * 64 + 64):
        with pytest.raises(RuntimeError, match="table of 256"):
            pages_reserve(refs, table, rows)
    for r, t in ((refs.view(2, 3), table), (torch.zeros(12, dtype=torch.int32)[::2], table), (refs, table[0]), (refs, table[:, ::2]),
                 (refs, table[:1].expand(3, -1)), (table.view(-1), table)):
        with pytest.raises(ValueError):
            pages_free(r, t, [0])
    for r, t in ((refs.long(), table), (refs, table.long())):
        with pytest.raises(TypeError):
            pages_free(r, t, [0])
    for call in (lambda: pages_free(refs, table, [0]), lambda: pages_fork(refs, table, S, 1, [0], tails), lambda: pages_reserve(refs, table, S)):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()
    mk = lambda P, n=32, H=2, planes=2: PagePool(torch.zeros(planes, P, n, dtype=torch.uint8), torch.zeros(planes, P, H), torch.zeros(P, dtype=torch.int32))
    pool = mk(6)
    for into in (mk(6, n=48), mk(6, H=3), mk(6, planes=3), mk(6)._replace(refs=torch.zeros(5, dtype=torch.int32)), pool,
                 mk(6)._replace(codes=torch.zeros(2, 32, 6, dtype=torch.uint8).transpose(1, 2)), mk(6)._replace(refs=pool.refs)):
        with pytest.raises(ValueError):
            pages_compact(pool, table, into)
    with pytest.raises(ValueError, match="multiple of 16"):
        pages_compact(mk(6, n=24), table, mk(6, n=24))
    with pytest.raises(TypeError):
        pages_compact(pool, table, mk(6)._replace(scales=torch.zeros(2, 6, 2, dtype=BF16)))
    with pytest.raises(RuntimeError, match="MI355X"):
        pages_compact(pool, table, mk(3))


def test_sample_refuses():
    from mote_amd.sample import sample_tokens

    x, u = torch.zeros(3, 50), torch.zeros(3)
    for bad in (x[0], x[:, :0], torch.zeros(1, (1 << 20) + 1)):
        with pytest.raises(ValueError):
            sample_tokens(bad, u[: bad.shape[0]] if bad.dim() == 2 else u)
    for dt in (torch.float16, torch.float64, torch.int32):
        with pytest.raises(TypeError):
            sample_tokens(x.to(dt), u)
    for bad in (u[:2], torch.zeros(6)[::2], u[:, None]):
        with pytest.raises(ValueError, match="u must"):
            sample_tokens(x, bad)
    with pytest.raises(TypeError, match="u must"):
        sample_tokens(x, u.double())
    for name in ("temperature", "top_p", "min_p"):
        for bad in (-0.5, float("nan")):
            with pytest.raises(ValueError, match=name):
                sample_tokens(x, u, **{name: bad})
        with pytest.raises(TypeError, match=name):
            sample_tokens(x, u, **{name: "1"})
        with pytest.raises(TypeError, match=name):
            sample_tokens(x, u, **{name: u.double()})
        with pytest.raises(ValueError, match=name):
            sample_tokens(x, u, **{name: u[:2]})
    with pytest.raises(ValueError, match="top_k"):
        sample_tokens(x, u, top_k=-1)
    with pytest.raises(TypeError, match="top_k"):
        sample_tokens(x, u, top_k=2.5)
    with pytest.raises(TypeError, match="top_k"):
        sample_tokens(x, u, top_k=torch.zeros(3, dtype=torch.int32))
    for bad in (torch.zeros(2, dtype=torch.int64), torch.zeros(3, dtype=torch.int32)):
        with pytest.raises(ValueError, match="out must"):
            sample_tokens(x, u, out=bad)
    with pytest.raises(ValueError, match="run must"):
        sample_tokens(x, u, run=torch.zeros(2, dtype=torch.bool))
    with pytest.raises(RuntimeError, match="no backward"):
        sample_tokens(x.clone().requires_grad_(True), u)
    with pytest.raises(RuntimeError, match="no backward"):
        sample_tokens(x, u, temperature=torch.ones(3, requires_grad=True))
    with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="dual"):
        sample_tokens(torch.autograd.forward_ad.make_dual(x, x), u)
    with pytest.raises(RuntimeError, match="MI355X"):
        sample_tokens(x, u)
