"""What the 4-bit cache's and the 8-bit products' entry points refuse, on the CPU: a bad call raises before
anything could be launched."""

from __future__ import annotations

import pytest
import torch

from mote_amd import _lib as L

pytestmark = pytest.mark.skipif(not L.available(), reason="libmote_relation.so not built")


def _cache(B=2, H=4, cap=64, D=48):
    from mote_amd.cache4 import cache4_zeros

    return cache4_zeros(B, H, cap, D, "cpu")


def _rows(B=2, H=4, T=8, D=48, dtype=torch.bfloat16):
    return torch.zeros(B, H, T, D, dtype=dtype), torch.zeros(B, H, T, D, dtype=dtype)


def test_cache4_zeros_layout():
    c = _cache(D=40)
    assert c.p2.shape == (2, 4, 64, 32) and c.p2_scale.shape == (2, 4, 64, 2)
    assert c.p2.dtype == torch.uint8 and c.info_scale.dtype == torch.bfloat16
    for D in (0, 4, 50, 136):
        with pytest.raises(ValueError, match="head dim"):
            _cache(D=D)


def test_write_refuses():
    from mote_amd.cache4 import cache4_write

    c = _cache()
    k, v = _rows()
    with pytest.raises(ValueError, match="p2 and info"):
        cache4_write(c, k, v[:, :, :4])
    with pytest.raises(TypeError):
        cache4_write(c, k, v.float())
    with pytest.raises(TypeError):
        cache4_write(c, k.half(), v.half())
    with pytest.raises(ValueError, match="head dim"):
        cache4_write(c, *_rows(D=44))
    with pytest.raises(ValueError, match="codes of P2"):
        cache4_write(c, *_rows(D=96))
    with pytest.raises(ValueError, match="codes of P2"):
        cache4_write(c, *_rows(H=2))
    for start in (-1, 57, 64):
        with pytest.raises(RuntimeError, match="capacity of 64"):
            cache4_write(c, k, v, start)
    for bad in (torch.zeros(2, dtype=torch.int32), torch.zeros(3, dtype=torch.int64)):
        with pytest.raises(ValueError, match="start"):
            cache4_write(c, k, v, bad)
        with pytest.raises(ValueError, match="lens"):
            cache4_write(c, k, v, 0, bad)
    with pytest.raises(RuntimeError, match="no backward"):
        cache4_write(c, k.requires_grad_(True), v)
    with pytest.raises(RuntimeError, match="MI355X"):
        cache4_write(c, k.detach(), v)


def test_cache_layouts_that_are_refused():
    from mote_amd.cache4 import Cache4, cache4_read, cache4_write

    c = _cache()
    k, v = _rows()
    with pytest.raises(ValueError, match="back to back"):
        cache4_write(c._replace(p2=torch.zeros(2, 4, 64, 64, dtype=torch.uint8)[..., :32],
                                info=torch.zeros(2, 4, 64, 64, dtype=torch.uint8)[..., :32]), k, v)
    with pytest.raises(ValueError, match="same strides"):
        cache4_write(c._replace(info=torch.zeros(2, 4, 128, 32, dtype=torch.uint8)[:, :, :64]), k, v)
    with pytest.raises(TypeError):
        cache4_write(c._replace(p2_scale=c.p2_scale.float()), k, v)
    with pytest.raises(TypeError):
        cache4_write(c._replace(p2=c.p2.to(torch.int8)), k, v)
    one = [t[:, :1].expand(t.shape) for t in c]
    with pytest.raises(ValueError, match="several heads"):
        cache4_write(Cache4(*one), k, v)
    with pytest.raises(ValueError, match="same rows"):
        cache4_write(c._replace(info=c.p2), k, v)
    with pytest.raises(RuntimeError, match="MI355X"):
        cache4_read(Cache4(*one), 48)  # reading shared rows is fine: only the device is missing


def test_read_refuses():
    from mote_amd.cache4 import cache4_read

    c = _cache()
    with pytest.raises(ValueError, match="codes of P2"):
        cache4_read(c, 96)
    with pytest.raises(RuntimeError, match="capacity of 64"):
        cache4_read(c, 48, 60, 5)
    with pytest.raises(ValueError, match="rows"):
        cache4_read(c, 48, 0, -1)
    with pytest.raises(ValueError, match="number of rows"):
        cache4_read(c, 48, torch.zeros(2, dtype=torch.int64))
    with pytest.raises(TypeError):
        cache4_read(c, 48, dtype=torch.float16)
    with pytest.raises(ValueError, match="out"):
        cache4_read(c, 48, 0, 8, out=_rows(T=9))
    with pytest.raises(ValueError, match="several places"):
        cache4_read(c, 48, 0, 8, out=tuple(t[:, :, :1].expand(t.shape) for t in _rows()))
    with pytest.raises(RuntimeError, match="gradient"):
        cache4_read(c, 48, 0, 8, out=tuple(t.requires_grad_(True) for t in _rows()))
    with pytest.raises(RuntimeError, match="MI355X"):
        cache4_read(c, 48)


def test_decode4_refuses():
    from mote_amd.cache4 import relation_decode4

    c = _cache()
    x = torch.zeros(2, 4, 48, dtype=torch.bfloat16)
    S, lam = torch.zeros(2, dtype=torch.int64), torch.tensor(0.5)
    with pytest.raises(ValueError, match="head stride"):
        relation_decode4(x, x, x.transpose(1, 2).contiguous().transpose(1, 2), S, c, lam)
    with pytest.raises(ValueError, match="head stride"):
        relation_decode4(x, x[:1], x, S, c, lam)
    with pytest.raises(TypeError):
        relation_decode4(x, x, x.float(), S, c, lam)
    with pytest.raises(TypeError):
        relation_decode4(x.half(), x.half(), x.half(), S, c, lam)
    for s in (S.int(), S[:1], torch.zeros(4, dtype=torch.int64)[::2]):
        with pytest.raises(ValueError, match="S must"):
            relation_decode4(x, x, x, s, c, lam)
    with pytest.raises(ValueError, match="codes of P2"):
        relation_decode4(x, x, x, S, _cache(B=1), lam)
    y3 = torch.zeros(2, 3, 48, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="even"):
        relation_decode4(y3, y3, y3, S, _cache(H=3), lam)
    bad = dict(inv_freq=torch.zeros(23), theta=torch.zeros(4), xm=torch.zeros(3), run=torch.zeros(2, dtype=torch.bool),
               y=torch.zeros(2, 4, 48), g=torch.zeros(2, 4, dtype=torch.bfloat16),
               workspace=torch.zeros(64, dtype=torch.uint8)[::2])
    for name, value in bad.items():
        with pytest.raises(ValueError, match=name):
            relation_decode4(x, x, x, S, c, lam, **{name: value})
    qkv = torch.zeros(2, 3, 4, 48, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="lies over an input"):
        relation_decode4(qkv[:, 0], qkv[:, 1], qkv[:, 2], S, c, lam, y=qkv[:, 2])
    with pytest.raises(ValueError, match="lam"):
        relation_decode4(x, x, x, S, c, torch.zeros(2))
    with pytest.raises(RuntimeError, match="no backward"):
        relation_decode4(x.clone().requires_grad_(True), x, x, S, c, lam)
    with pytest.raises(RuntimeError, match="MI355X"):
        relation_decode4(x, x, x, S, c, lam)


def test_int8_refuses():
    from mote_amd.int8 import Int8Weight, int8_linear, quantize_rows

    w = Int8Weight(torch.zeros(16, 128, dtype=torch.int8), torch.zeros(16), 100)
    x = torch.zeros(4, 100, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="x must be"):
        int8_linear(x[:, :64], w)
    with pytest.raises(TypeError):
        int8_linear(x.half(), w)
    with pytest.raises(ValueError, match="codes"):
        int8_linear(x, w._replace(q=w.q[:, :100]))
    with pytest.raises(ValueError, match="codes"):
        int8_linear(x, w._replace(scale=torch.zeros(15)))
    with pytest.raises(TypeError):
        int8_linear(x, w._replace(q=w.q.to(torch.uint8)))
    with pytest.raises(ValueError, match="out must be"):
        int8_linear(x, w, out=torch.zeros(4, 17, dtype=torch.bfloat16))
    square = Int8Weight(torch.zeros(100, 128, dtype=torch.int8), torch.zeros(100), 100)
    wide = torch.zeros(4, 150, dtype=torch.bfloat16)
    for inp, out in ((x, x), (wide[:, :100], wide[:, 50:])):
        with pytest.raises(ValueError, match="lies over an input"):
            int8_linear(inp, square, out=out)
    with pytest.raises(ValueError, match="run"):
        int8_linear(x, w, run=torch.zeros(1))
    with pytest.raises(ValueError, match="xm"):
        int8_linear(x, w, xm=torch.zeros(4))
    with pytest.raises(RuntimeError, match="no backward"):
        int8_linear(x.clone().requires_grad_(True), w)
    with pytest.raises(RuntimeError, match="MI355X"):
        int8_linear(x, w)
    with pytest.raises(ValueError, match=r"\[M, K\]"):
        quantize_rows(torch.zeros(4))
    with pytest.raises(RuntimeError, match="MI355X"):
        quantize_rows(x)


def test_c_entry_points_refuse_without_a_gpu():
    """The C ABI's own checks: sizes, alignment, workspace; nothing is launched and nothing thrown."""
    lib = L.lib()
    for call in (lib.mote_cache4_write, lib.mote_cache4_read):
        r = L.Cache4RowsArgs()
        assert call(None, None) == 1
        r.dtype, r.B, r.H, r.T, r.D, r.capacity = 7, 1, 2, 4, 48, 64
        assert call(r, None) == 1
        r.dtype, r.D = L.MOTE_BF16, 100
        assert call(r, None) == 2 and b"head dim" in lib.mote_last_error()
        r.D = 48
        assert call(r, None) == 1  # null pointers
        r.T = 0
        assert call(r, None) == 0
        r.T = 4
        r.p2.data = r.info.data = r.cache.p2 = r.cache.info = r.cache.p2_scale = r.cache.info_scale = 16
        r.p2.stride_r = 44
        assert call(r, None) == 1 and b"16-byte" in lib.mote_last_error()
        r.p2.stride_r, r.cache.codes_sh = 48, 24
        assert call(r, None) == 1 and b"codes" in lib.mote_last_error()
        r.cache.codes_sh = 32
        for r.H, r.T in ((65536, 4), (2, 1 << 28)):
            assert call(r, None) == 2 and b"too many" in lib.mote_last_error()
    a = L.Decode4Args()
    assert lib.mote_relation_decode4(None, None) == 1
    a.dtype, a.B, a.H, a.D, a.capacity = L.MOTE_BF16, 1, 3, 96, 256
    assert lib.mote_relation_decode4(a, None) == 2  # an odd number of heads
    a.H = 2
    assert lib.mote_relation_decode4(a, None) == 1  # null pointers
    a.lam = a.S = a.p1 = a.p2 = a.info = a.y = a.g = 16
    a.cache.p2 = a.cache.info = a.cache.p2_scale = a.cache.info_scale = 16
    need = int(lib.mote_relation_decode4_workspace(a))
    assert need > 0
    a.workspace, a.workspace_bytes = 16, need - 1
    assert lib.mote_relation_decode4(a, None) == 3
    a.workspace, a.workspace_bytes = 24, need  # off a 16-byte boundary
    assert lib.mote_relation_decode4(a, None) == 3
    w = L.Int8LinearArgs()
    assert lib.mote_int8_linear(None, None) == 1 and lib.mote_quantize_rows(None, None) == 1
    w.dtype, w.M, w.N, w.K = L.MOTE_BF16, 4, 16, 200000
    assert lib.mote_int8_linear(w, None) == 2
    w.K, w.M = 128, (1 << 30) + 1
    assert lib.mote_int8_linear(w, None) == 2
    w.M = 0
    assert lib.mote_int8_linear(w, None) == 0
    w.M = 65
    assert lib.mote_int8_linear(w, None) == 1
    w.x = w.wq = w.w_scale = w.y = 16
    w.x_sr, w.y_sr = 128, 16
    assert int(lib.mote_int8_linear_workspace(w)) >= 65 * 128 + 65 * 4
    assert lib.mote_int8_linear(w, None) == 3
    w.run = 16
    assert lib.mote_int8_linear(w, None) == 2  # the predicate belongs to the one-launch form
