"""The cache in 4 bits on the GPU: rows written and read back bit for bit, and the decode step over them
against the Relation oracle in 64 bits on the stored values."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import quant as Q
from oracle import relation as O

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _rows(seed, B, H, T, D, dtype, scale=1.0):
    x = torch.randn(B, H, T, D, generator=_gen(seed)) * scale
    x[..., :: max(1, D // 3)] *= 5.0
    return x.to(dtype)


def _stored(codes, scales, D):
    return Q.unpack_codes(codes.cpu(), D) * scales.cpu().double().repeat_interleave(Q.GROUP, -1)[..., :D]


def _random_cache(seed, B, H, cap, D, cuda):
    """A cache whose every byte is random (padding included) with scales of ordinary size."""
    from mote_amd.cache4 import Cache4, groups

    G, g = groups(D), _gen(seed)
    codes = lambda: torch.randint(0, 256, (B, H, cap, 16 * G), generator=g, dtype=torch.uint8).to(cuda)
    scales = lambda: (0.2 + 0.3 * torch.rand(B, H, cap, G, generator=g)).to(BF16).to(cuda)
    return Cache4(codes(), scales(), codes(), scales())


# ---- rows ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,T,D", [(1, 2, 1, 8), (2, 3, 5, 40), (1, 4, 67, 48), (3, 2, 33, 64), (2, 8, 130, 96),
                                     (1, 2, 9, 120), (2, 2, 64, 128)])
def test_rows_are_the_formats_bit_for_bit(cuda, dtype, B, H, T, D):
    from mote_amd.cache4 import cache4_read, cache4_write

    cap, start = T + 7, 3
    cache = _random_cache(1, B, H, cap, D, cuda)
    before = [t.clone() for t in cache]
    k, v = _rows(2, B, H, T, D, dtype), _rows(3, B, H, T, D, dtype, 1e-3)
    cache4_write(cache, k.to(cuda), v.to(cuda), start)
    for codes, scales, x in ((cache.p2, cache.p2_scale, k), (cache.info, cache.info_scale, v)):
        vals, s = Q.encode4(x)
        assert torch.equal(scales[:, :, start: start + T].cpu(), s)
        assert torch.equal(Q.unpack_codes(codes[:, :, start: start + T].cpu(), D), vals)
    for now, old in zip(cache, before):  # the rows around them
        assert torch.equal(now[:, :, :start], old[:, :, :start])
        assert torch.equal(now[:, :, start + T:], old[:, :, start + T:])
    for out_dtype in (BF16, F32):
        got = cache4_read(cache, D, 0, dtype=out_dtype)
        for g, codes, scales in zip(got, (cache.p2, cache.info), (cache.p2_scale, cache.info_scale)):
            assert g.shape == (B, H, cap, D)
            # a code has two significant bits and a scale eight: the product is exact in fp32
            assert torch.equal(g.cpu(), _stored(codes, scales, D).float().to(out_dtype))


def test_every_border_and_every_special_value(cuda):
    """Codes at the borders between e2m1 values (on them and one step of fp32 beside), and groups that hold
    infinities, NaNs, zeros and magnitudes near the smallest and largest numbers."""
    from mote_amd.cache4 import cache4_read, cache4_write, cache4_zeros

    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0])
    near = torch.cat([mids, mids * (1 + 2.0 ** -23), mids * (1 - 2.0 ** -23), torch.tensor([6.0])])
    x = torch.zeros(1, 2, 12, 64)
    x[0, 0, 0, : near.numel()], x[0, 1, 0, : near.numel()] = near, -near
    x[0, 0, 1, : near.numel()] = near * 3.0  # a scale that is no power of two
    x[0, 0, 1, 40] = 17.9
    for r, val in enumerate((float("inf"), -float("inf"), float("nan"), 1e-44, 5.9 * 2.0 ** -126, 6.0 * 2.0 ** -126, 3.38e38, -0.0)):
        x[0, 0, 2 + r, 5], x[0, 1, 2 + r, 40] = val, val
        x[0, 0, 2 + r, 6] = -0.75
    cache = cache4_zeros(1, 2, 12, 64, cuda)
    cache4_write(cache, x.to(cuda), (-x).to(cuda))
    for codes, scales, t in ((cache.p2, cache.p2_scale, x), (cache.info, cache.info_scale, -x)):
        vals, s = Q.encode4(t)
        assert torch.equal(scales.cpu().isnan(), s.isnan())
        assert torch.equal(scales.cpu().nan_to_num(-1.0), s.nan_to_num(-1.0))
        assert torch.equal(Q.unpack_codes(codes.cpu(), 64), vals)
    k, _ = cache4_read(cache, 64, dtype=F32)
    assert k[0, 0, 2, :32].isnan().all() and (k[0, 0, 2, 32:] == 0).all()
    assert k[0, 1, 4, 32:].isnan().all() and (k[0, 1, 4, :32] == 0).all()


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_scales_and_codes_of_every_magnitude(cuda, dtype):
    """Groups whose maximum has every exponent a float has, every mantissa of a bf16 (and random ones of fp32):
    the scale and its inverse are those of the divisions, whatever the kernel computes them with."""
    from mote_amd.cache4 import cache4_write, cache4_zeros

    e = torch.arange(-140, 128).double()[:, None]
    m = 1.0 + torch.arange(128).double() / 128
    if dtype == F32:
        m = torch.cat([m, 1.0 + torch.rand(128, generator=_gen(5)).double()])
    top = torch.ldexp(m, e.int()).reshape(-1)
    border = (6.0 * 2.0 ** -126) * (1 + torch.arange(-64, 64).double() * (2.0 ** -23 if dtype == F32 else 2.0 ** -7))
    top = torch.cat([top, border]).float().to(dtype)
    top = top[top.isfinite()]
    x = (torch.rand(1, 2, top.numel(), 32, generator=_gen(6)) * 2 - 1) * top[:, None].float()
    x[..., 7] = top.float()
    x = x.to(dtype)
    cache = cache4_zeros(1, 2, top.numel(), 32, cuda)
    cache4_write(cache, x.to(cuda), (-x).to(cuda))
    for codes, scales, t in ((cache.p2, cache.p2_scale, x), (cache.info, cache.info_scale, -x)):
        vals, s = Q.encode4(t)
        assert torch.equal(scales.cpu(), s)
        assert torch.equal(Q.unpack_codes(codes.cpu(), 32), vals)


def test_more_sequences_than_one_launch_takes(cuda):
    from mote_amd.cache4 import cache4_read, cache4_write, cache4_zeros

    B, D = 70001, 8
    cache = cache4_zeros(B, 1, 3, D, cuda)
    x = _rows(11, B, 1, 1, D, BF16)
    start, lens = (torch.arange(B) % 3), (torch.arange(B) % 5 > 0).long()
    cache4_write(cache, x.to(cuda), (-x).to(cuda), start.to(cuda), lens.to(cuda))
    vals, s = Q.encode4(x)
    want = torch.zeros(B, 1, 3, D, dtype=torch.double)
    want[torch.arange(B), 0, start] = (Q.values4(vals, s) * lens[:, None, None, None])[:, 0, 0]
    for dtype in (BF16, F32):
        k, v = cache4_read(cache, D, 0, dtype=dtype)
        assert torch.equal(k.cpu(), want.float().to(dtype)) and torch.equal(v.cpu(), -want.float().to(dtype))


def test_positions_lengths_and_strides(cuda):
    """Device positions, padded batches, rows outside the capacity, transposed and misaligned inputs,
    caches that are slices of a larger store, views as outputs."""
    from mote_amd.cache4 import Cache4, cache4_read, cache4_write

    B, H, T, D, cap = 5, 2, 11, 96, 40
    big = _random_cache(5, 2 * B, H + 1, cap, D, cuda)
    cache = Cache4(*(t[::2, 1:] for t in big))
    before = [t.clone() for t in big]
    x = _rows(6, B, T, H, 2 * D + 1, BF16).to(cuda)
    k, v = x[..., :D].transpose(1, 2), x[..., D + 1:].transpose(1, 2)  # v's rows start off a chunk
    start = torch.tensor([0, 7, 35, -4, 40], device=cuda)
    lens = torch.tensor([11, 0, 11, 11, 3], device=cuda)
    cache4_write(cache, k, v, start, lens)
    want = [t.clone() for t in before]
    for i, (codes, scales, t) in enumerate(((0, 1, k), (2, 3, v))):
        vals, s = Q.encode4(t.cpu())
        for b in range(B):
            for r in range(int(lens[b])):
                row = int(start[b]) + r
                if 0 <= row < cap:
                    got = Q.unpack_codes(cache[codes][b, :, row].cpu(), D)
                    assert torch.equal(got, vals[b, :, r]) and torch.equal(cache[scales][b, :, row].cpu(), s[b, :, r])
                    want[codes][2 * b, 1:, row] = cache[codes][b, :, row]
                    want[scales][2 * b, 1:, row] = cache[scales][b, :, row]
    for now, w in zip(big, want):
        assert torch.equal(now, w)
    out = torch.full((B, T + 2, H, D), 7.0, device=cuda, dtype=BF16).transpose(1, 2)
    outs = (out[:, :, 1: T + 1], torch.empty(B, H, T, D, device=cuda, dtype=BF16))
    got = cache4_read(cache, D, start, T, out=outs)
    assert got[0].data_ptr() == outs[0].data_ptr()
    for g, codes, scales in zip(got, cache[::2], cache[1::2]):
        full = _stored(codes, scales, D).float().to(BF16)
        for b in range(B):
            for r in range(T):
                row = int(start[b]) + r
                if 0 <= row < cap:
                    assert torch.equal(g[b, :, r].cpu(), full[b, :, row])
                else:
                    assert g[b, :, r].isnan().all()
    assert (out[:, :, 0] == 7).all() and (out[:, :, T + 1] == 7).all()
    cache4_write(cache, k[:, :, :0], v[:, :, :0], 0)  # no rows: nothing launched
    assert cache4_read(cache, D, 5, 0)[0].shape == (B, H, 0, D)
    for now, w in zip(big, want):
        assert torch.equal(now, w)


# ---- the decode step -------------------------------------------------------------------------------
def _tolerance(q, kvals, vvals, new, S, D, dtype):
    """What fp32 arithmetic can move y and g by, from the formula (per sequence and head, absolute).

    U: D products summed in any order, the scale and 1 / sqrt(D): (D + 4) half steps of sum |q k| / sqrt(D);
    a bf16 dot instruction may also truncate instead of rounding, twice that. e = SiLU(U): slope at most 1.1,
    and a few steps of exp and rcp (2 ulp each): 8 half steps of |U|. A weight exp(e - LSE) is off by twice
    that bound (numerator and denominator) and the sums over n rows run in chains of at most n / 64 + 64 + 64
    terms. Both scale |I~| in the mean; y is rounded once to its dtype."""
    h = 2.0 ** -24
    if S == 0:
        e_w = torch.zeros(q.shape[0], dtype=torch.float64)
        vmax = new.abs().amax(-1)
    else:
        mag = (q[:, None].abs() * kvals[:, :S].abs()).sum(-1) / math.sqrt(D)
        e_u = 2 * (D + 4) * h * mag.amax(-1) + 8 * h * mag.amax(-1)
        e_w = 2 * 1.1 * e_u + (S / 64 + 128 + 16) * h
        vmax = torch.maximum(vvals[:, :S].abs().amax((-1, -2)), new.abs().amax(-1))
    self_mag = (q.abs() * new.abs()).sum(-1) / math.sqrt(D)
    # g = sigma(.): slope at most 1/4; its argument is off by e_w and a few steps of ln(S + 1) and the Self score
    e_g = 0.25 * (e_w + 16 * h * (2 + math.log(S + 2.0)) + 2 * (D + 4) * h * self_mag * 0.25) + 4 * h
    e_y = (e_w + 2 * e_g + 8 * h) * vmax
    return e_y, e_g, torch.finfo(dtype).eps / 2


def _decode_case(cuda, seed, dtype, B, H, D, cap, S, layer=0, rope=False, givens=False, cache=None):
    g = _gen(seed)
    x = torch.randn(B, 3, H, D, generator=g).to(dtype)
    cache = _random_cache(seed + 1, B, H, cap, D, cuda) if cache is None else cache
    inv = O.rope_inv_freq(D, 10000.0).float() if rope else None
    theta = (torch.rand(H // 2, generator=g) * 0.6 - 0.3) if givens else None
    return x, cache, inv, theta, torch.tensor(0.5), torch.tensor(S)


def _check_step(x, cache, inv, theta, lam, S, layer, dtype, y, g, kstored, vstored):
    B, _, H, D = x.shape
    q, kn, new = O.decode_rows_ref(x[:, 0], x[:, 1], x[:, 2], S.tolist(), inv, theta, layer, dtype)
    for b in range(B):
        s = int(S[b])
        kb, vb = kstored[b].clone(), vstored[b].clone()
        kb[:, s], vb[:, s] = kn[b].double(), new[b].double()
        yr, gr = O.relation_decode_ref(q[b: b + 1].double(), kb[None], vb[None], [s], lam.double(), 2.0, dtype=torch.float64)
        e_y, e_g, half = _tolerance(q[b].double(), kb, vb, new[b].double(), s, D, dtype)
        dy, dg = (y[b].cpu().double() - yr[0]).abs(), (g[b].cpu().double() - gr[0]).abs()
        assert (dy <= e_y[:, None] + half * yr[0].abs() * (1 + 2.0 ** -7)).all(), (b, s, float(dy.max()))
        assert (dg <= e_g).all(), (b, s, float(dg.max()), float(e_g.min()))
    return kn, new


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,D,cap,S", [
    (1, 2, 8, 64, [5]), (2, 4, 48, 300, [0, 299]), (1, 2, 32, 1100, [1024]), (3, 2, 40, 130, [1, 63, 129]),
    (2, 8, 96, 700, [64, 65]), (1, 8, 96, 4200, [4099]), (4, 2, 64, 600, [127, 128, 129, 511]),
    (2, 2, 128, 520, [519, 2]), (1, 6, 112, 333, [300]), (20, 8, 96, 256, list(range(0, 240, 12)))])
def test_decode_step_against_64_bits(cuda, dtype, B, H, D, cap, S):
    """y and g against the oracle on the stored values (no rotation: the query is the input itself), the new
    row stored in the format's own codes, every other row untouched."""
    from mote_amd.cache4 import relation_decode4

    x, cache, _, _, lam, S = _decode_case(cuda, 10 + D, dtype, B, H, D, cap, S)
    kst, vst = _stored(cache.p2, cache.p2_scale, D), _stored(cache.info, cache.info_scale, D)
    before = [t.clone() for t in cache]
    xd, Sd = x.to(cuda), S.to(cuda)
    y, g = relation_decode4(xd[:, 0], xd[:, 1], xd[:, 2], Sd, cache, lam.to(cuda))
    assert y.dtype == dtype and g.dtype == F32 and torch.equal(Sd.cpu(), S)
    kn, new = _check_step(x, cache, None, None, lam, S, 0, dtype, y, g, kst, vst)
    for b in range(B):
        s = int(S[b])
        for codes, scales, row in ((cache.p2, cache.p2_scale, kn), (cache.info, cache.info_scale, new)):
            vals, sc = Q.encode4(row[b])
            assert torch.equal(Q.unpack_codes(codes[b, :, s].cpu(), D), vals)
            assert torch.equal(scales[b, :, s].cpu(), sc)
        for now, old in zip(cache, before):
            now[b, :, s] = old[b, :, s]
    for now, old in zip(cache, before):
        assert torch.equal(now, old)


@pytest.mark.parametrize("layer", [0, 1])
@pytest.mark.parametrize("dtype,rope_f32", [(BF16, False), (BF16, True), (F32, False)])
def test_decode_step_with_rope_and_givens(cuda, dtype, rope_f32, layer):
    """RoPE at far positions and Givens: the step's own convention, as in the step over a bf16 cache. A table
    entry one rounding step off (the GPU's and the CPU's cos differ in the last bit of fp32) moves one query
    element by a step of its dtype; the bound is the reference's own for such steps (2e-2 in bf16, 1e-5 in
    fp32, relative to the largest value)."""
    from conftest import rel_err
    from mote_amd.cache4 import relation_decode4

    B, H, D, cap, S = 3, 4, 96, 4000, [3999, 17, 2500]
    x, cache, inv, theta, lam, S = _decode_case(cuda, 77, dtype, B, H, D, cap, S, layer, True, True)
    kst, vst = _stored(cache.p2, cache.p2_scale, D), _stored(cache.info, cache.info_scale, D)
    xd = x.to(cuda)
    y, g = relation_decode4(xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), cache, lam.to(cuda), 2.0, inv.to(cuda),
                            theta.to(cuda), layer, rope_f32=rope_f32)
    q, kn, new = O.decode_rows_ref(x[:, 0], x[:, 1], x[:, 2], S.tolist(), inv, theta, layer, dtype,
                                   rope_dtype=F32 if rope_f32 else None)
    for b in range(B):
        s = int(S[b])
        kst[b, :, s], vst[b, :, s] = kn[b].double(), new[b].double()
    yr, gr = O.relation_decode_ref(q.double(), kst, vst, S.tolist(), lam.double(), 2.0, dtype=torch.float64)
    bound = 2e-2 if dtype == BF16 else 1e-5
    assert rel_err(y, yr) < bound and rel_err(g, gr) < bound
    got_k = torch.stack([_stored(cache.p2[b, :, int(S[b])], cache.p2_scale[b, :, int(S[b])], D) for b in range(B)])
    vals, sc = Q.encode4(kn)
    # a flipped table entry may move a value by one code: at most a gap of 2 codes' scale
    assert ((got_k - Q.values4(vals, sc)).abs() <= 2.01 * sc.double().repeat_interleave(32, -1)).all()
    got_v = torch.stack([_stored(cache.info[b, :, int(S[b])], cache.info_scale[b, :, int(S[b])], D) for b in range(B)])
    vals, sc = Q.encode4(new)
    assert torch.equal(got_v, Q.values4(vals, sc))


def test_rows_past_the_fill_never_count(cuda):
    """NaN scales in every row at and past S change nothing."""
    from mote_amd.cache4 import Cache4, relation_decode4

    for D, S in ((48, [70, 0]), (96, [1, 193]), (64, [128, 129]), (32, [255, 256])):
        x, cache, _, _, lam, S = _decode_case(cuda, 5, BF16, 2, 2, D, 600, S)
        poisoned = Cache4(*(t.clone() for t in cache))
        for b in range(2):
            poisoned.p2_scale[b, :, int(S[b]):] = float("nan")
            poisoned.info_scale[b, :, int(S[b]):] = float("nan")
        xd = x.to(cuda)
        a = relation_decode4(xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), cache, lam.to(cuda))
        b_ = relation_decode4(xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), poisoned, lam.to(cuda))
        assert torch.equal(a[0], b_[0]) and torch.equal(a[1], b_[1])


def test_a_nan_row_shows_and_a_bad_position_stores_nothing(cuda):
    from mote_amd.cache4 import relation_decode4

    x, cache, _, _, lam, S = _decode_case(cuda, 6, BF16, 4, 2, 64, 300, [200, 300, -1, 200])
    cache.info_scale[0, 1, 57, 1] = float("nan")   # dims 32..63 of one head's mean
    cache.p2_scale[3, 0, 57, 0] = float("nan")     # a score: the whole head
    before = [t.clone() for t in cache]
    xd = x.to(cuda)
    y, g = relation_decode4(xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), cache, lam.to(cuda))
    assert y[0, 1, 32:].isnan().all() and not y[0, 1, :32].isnan().any() and not y[0, 0].isnan().any()
    assert y[3, 0].isnan().all() and g[3, 0].isnan() and not y[3, 1].isnan().any()
    assert y[1:3].isnan().all() and g[1:3].isnan().all()
    for now, old in zip(cache, before):
        assert torch.equal(now[1:3].nan_to_num(-1.0) if now.is_floating_point() else now[1:3],
                           old[1:3].nan_to_num(-1.0) if old.is_floating_point() else old[1:3])


def test_advance_xm_run_and_given_outputs(cuda):
    from mote_amd.cache4 import decode4_workspace, relation_decode4

    B, H, D, cap = 3, 4, 96, 512
    x, cache, _, _, lam, S = _decode_case(cuda, 8, BF16, B, H, D, cap, [100, 0, 511])
    xd, Sd = x.to(cuda), S.to(cuda)
    ws = decode4_workspace(B, H, D, cap, cuda)
    y, g, xm = torch.full((B, H, D), 3.0, device=cuda, dtype=BF16), torch.full((B, H), 3.0, device=cuda), torch.full((B,), 3.0, device=cuda)
    before = [t.clone() for t in cache]
    off = torch.zeros(1, dtype=torch.bool, device=cuda)
    args = (xd[:, 0], xd[:, 1], xd[:, 2], Sd, cache, lam.to(cuda))
    kw = dict(workspace=ws, y=y, g=g, xm=xm, advance=True)
    relation_decode4(*args, run=off, **kw)
    assert (y == 3).all() and (g == 3).all() and (xm == 3).all() and torch.equal(Sd.cpu(), S)
    assert all(torch.equal(a, b) for a, b in zip(cache, before))
    out = relation_decode4(*args, run=~off, **kw)
    assert out[0].data_ptr() == y.data_ptr() and torch.equal(Sd.cpu(), S + 1)
    want = torch.stack([g[:, i] for i in range(H)]).cumsum(0)[-1] / H
    assert torch.allclose(xm, want, rtol=4 * 2.0 ** -24, atol=0)  # four additions and a division
    n = decode4_workspace(B, H, D, cap, cuda).numel()
    assert n == ws.numel()
    for bad in (ws[:-1], decode4_workspace(B + 1, H, D, cap, cuda)):
        with pytest.raises(ValueError, match="workspace"):
            relation_decode4(*args, workspace=bad)


def test_many_steps_in_a_graph(cuda):
    """Steps captured with the device position moving, replayed between eager work, against the same steps
    one by one; two graphs and eager calls share the workspace in turn."""
    from mote_amd.cache4 import Cache4, decode4_workspace, relation_decode4

    B, H, D, cap = 2, 4, 64, 700
    x, cache, inv, theta, lam, S = _decode_case(cuda, 9, BF16, B, H, D, cap, [120, 3], 0, True, True)
    twin = Cache4(*(t.clone() for t in cache))
    xd, Sd, St = x.to(cuda), S.to(cuda), S.to(cuda)
    lamd, invd, thd = lam.to(cuda), inv.to(cuda), theta.to(cuda)
    ws = decode4_workspace(B, H, D, cap, cuda)
    y, g = torch.empty(B, H, D, device=cuda, dtype=BF16), torch.empty(B, H, device=cuda)
    step = lambda c, s, **kw: relation_decode4(xd[:, 0], xd[:, 1], xd[:, 2], s, c, lamd, 2.0, invd, thd, 1, advance=True, **kw)
    graph = torch.cuda.CUDAGraph()
    warm = Cache4(*(t.clone() for t in cache))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, S.to(cuda), workspace=ws, y=y, g=g)
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        step(cache, Sd, workspace=ws, y=y, g=g)
    other, So = Cache4(*(t.clone() for t in warm)), torch.tensor([640, 0], device=cuda)
    third, S3 = Cache4(*(t.clone() for t in warm)), So.clone()
    second = torch.cuda.CUDAGraph()
    with torch.cuda.graph(second):
        yo, go = step(other, So, workspace=ws)
    for i in range(5):
        graph.replay()
        yt, gt = step(twin, St)
        torch.cuda.synchronize()
        assert torch.equal(y, yt) and torch.equal(g, gt) and torch.equal(Sd, St)
        second.replay()
        y3, g3 = step(third, S3, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(yo, y3) and torch.equal(go, g3)
    for a, b in zip(cache, twin):
        assert torch.equal(a, b)
    assert Sd.tolist() == [125, 8]


def test_another_stream_and_strided_stores(cuda):
    """On a side stream, over the layer slices of one store whose sequences are far apart."""
    from mote_amd.cache4 import Cache4, relation_decode4

    B, H, D, cap = 2, 2, 96, 300
    x, cache, _, _, lam, S = _decode_case(cuda, 12, F32, B, H, D, cap, [299, 40])
    store = [torch.zeros(B, 3, H, *t.shape[2:], dtype=t.dtype, device=cuda) for t in cache]
    for s, t in zip(store, cache):
        s[:, 1] = t
    view = Cache4(*(s[:, 1] for s in store))
    xd, lamd, Sd = x.to(cuda), lam.to(cuda), S.to(cuda)
    want = relation_decode4(xd[:, 0], xd[:, 1], xd[:, 2], Sd, cache, lamd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = relation_decode4(xd[:, 0], xd[:, 1], xd[:, 2], Sd, view, lamd)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    four = torch.cat([xd, xd[:, :1]], 1)  # y in the rows of the projections' own buffer
    relation_decode4(four[:, 0], four[:, 1], four[:, 2], Sd, cache, lamd, y=four[:, 3])
    assert torch.equal(four[:, 3], want[0]) and torch.equal(four[:, :3], xd)
    for s, t in zip(store, cache):
        assert torch.equal(s[:, 1], t) and (s[:, 0] == 0).all() and (s[:, 2] == 0).all()


def test_offsets_past_32_bits(cuda):
    """A cache of more than 2^32 code bytes: the last sequence's rows are written, read and swept there."""
    from mote_amd.cache4 import Cache4, cache4_read, cache4_write, relation_decode4

    B, H, D, cap = 9, 2, 128, 4 << 20
    codes = lambda: torch.empty(B, H, cap, 64, dtype=torch.uint8, device=cuda)
    scales = lambda: torch.empty(B, H, cap, 4, dtype=BF16, device=cuda)
    cache = Cache4(codes(), scales(), codes(), scales())
    assert cache.p2.numel() > 1 << 32
    small = _random_cache(20, B, H, 96, D, cuda)
    lo = cap - 96
    for big, s in zip(cache, small):
        big[:, :, lo:] = s
    k, v = _rows(21, B, H, 20, D, BF16).to(cuda), _rows(22, B, H, 20, D, BF16).to(cuda)
    cache4_write(cache, k, v, cap - 30)
    cache4_write(small, k, v, 66)
    for big, s in zip(cache, small):
        assert torch.equal(big[:, :, lo:], s)
    for a, b in zip(cache4_read(cache, D, lo, 96), cache4_read(small, D)):
        assert torch.equal(a, b)
    for big in (cache.p2, cache.p2_scale, cache.info, cache.info_scale):
        big[-1, :, :lo] = 0  # zero rows score e = 0 and carry nothing
    x = torch.randn(B, 3, H, D, generator=_gen(23)).to(BF16).to(cuda)
    S = torch.zeros(B, dtype=torch.int64, device=cuda)
    S[-1] = cap - 1
    lam = torch.tensor(0.0, device=cuda)
    y, g = relation_decode4(x[:, 0], x[:, 1], x[:, 2], S, cache, lam)
    q = x[-1, 0].double()
    kd, vd = (_stored(c[-1], s[-1], D)[:, :95].to(cuda) for c, s in ((small.p2, small.p2_scale), (small.info, small.info_scale)))
    u = (kd * q[:, None]).sum(-1) / math.sqrt(D)
    e = torch.exp(u * torch.sigmoid(u))
    total = e.sum(-1) + lo
    mean = (e[..., None] * vd).sum(1) / total[:, None]
    self_score = torch.sigmoid((q * x[-1, 1].double()).sum(-1) / math.sqrt(D) / 2.0)
    gate = torch.sigmoid(torch.log(total) - self_score)
    want = (1 - gate)[:, None] * x[-1, 2].double() + gate[:, None] * mean
    # chains of cap / 64 / 128 terms and the formula's own steps, then one rounding
    assert (g[-1].double() - gate).abs().max() < 1e-5
    assert ((y[-1].double() - want).abs() <= 2.0 ** -8 * want.abs() + 1e-5).all()
