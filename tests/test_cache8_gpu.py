"""The paged cache in 8 bits against plain implementations in 64 bits: rows appended and read back bit for bit, the
decode step within bounds derived from the formula."""

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


def _rows(seed, B, H, T, D, dtype):
    """Rows with channels of unlike size and a few large ones."""
    g = _gen(seed)
    amp = (0.5 + torch.rand(H, 1, D, generator=g)) * torch.where(torch.rand(H, 1, D, generator=g) < 0.1, 8.0, 1.0)
    return (torch.randn(B, H, T, D, generator=g) * amp).to(dtype)


def _empty(B, H, D, blocks, dtype, cuda, spare=3, seed=0):
    """A cache whose table names pages of its own for every block, in no order."""
    from mote_amd.cache8 import cache8_zeros

    c = cache8_zeros(B, H, B * blocks + spare, blocks * 64, D, cuda, dtype)
    order = torch.randperm(B * blocks + spare, generator=_gen(seed))[: B * blocks]
    c.table.copy_(order.view(B, blocks).int())
    return c


def _filled(seed, B, H, D, blocks, dtype, cuda, held):
    """(cache, rows of P2, rows of I~) with held[b] rows in sequence b."""
    from mote_amd.cache8 import cache8_write

    c = _empty(B, H, D, blocks, dtype, cuda, seed=seed)
    T = max(max(held), 1)
    k, v = _rows(seed, B, H, T, D, dtype), _rows(seed + 1, B, H, T, D, dtype)
    cache8_write(c, k.to(cuda), v.to(cuda), torch.zeros(B, dtype=torch.int64, device=cuda), torch.tensor(held, device=cuda))
    return c, k, v


def _values(codes):
    return codes.cpu().view(torch.float8_e4m3fn).double()


def _page(c, D, b, j):
    """(codes of P2 [H, 64, D], scales, codes of I~, scales) of block j of sequence b."""
    t = int(c.table[b, j])
    k = _values(c.p2[t]).transpose(1, 2).flatten(2)
    v = _values(c.info[t]).transpose(1, 2)
    assert (k[..., D:] == 0).all() and (v[..., D:] == 0).all()
    return k[..., :D], c.p2_scale[t].cpu().double(), v[..., :D], c.info_scale[t].cpu().double()


# ---- rows ------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,D,held,new", [
    (1, 2, 96, [0], [64]), (2, 4, 48, [0, 60], [63, 4]), (3, 2, 40, [1, 64, 127], [190, 0, 66]), (2, 8, 128, [130, 0], [1, 300]),
    (1, 2, 8, [63], [1]), (2, 6, 112, [10, 50], [53, 15]), (1, 1, 16, [200], [500]), (2, 2, 120, [5, 100], [120, 29]),
    (1, 3, 64, [64], [64]), (1, 2, 72, [0], [1])])
def test_append_and_read(cuda, dtype, B, H, D, held, new):
    """Codes and scales are the format's own bit for bit; pages and tail rows that no new row belongs to are left as
    they were; rows read back are the values, each rounded once, zeros behind the end."""
    from mote_amd.cache8 import cache8_read, cache8_write

    T, blocks = max(new), (max(h + n for h, n in zip(held, new)) + 63) // 64 + 1
    c, k0, v0 = _filled(3, B, H, D, blocks, dtype, cuda, held)
    before = [t.clone() for t in c]
    k1, v1 = _rows(5, B, H, T, D, dtype), _rows(6, B, H, T, D, dtype)
    k1d = k1.transpose(1, 2).contiguous().transpose(1, 2).to(cuda)  # the projections' own layout
    cache8_write(c, k1d, v1.to(cuda), torch.tensor(held, device=cuda), torch.tensor(new, device=cuda))
    fresh = set()
    for b in range(B):
        end = held[b] + new[b]
        rows = [torch.cat([x0[b, :, : held[b]], x1[b, :, : new[b]]], 1) for x0, x1 in ((k0, k1), (v0, v1))]
        for j in range(held[b] // 64, end // 64):
            ck, sk, cv, sv = _page(c, D, b, j)
            for got, s, x in ((ck, sk, rows[0]), (cv, sv, rows[1])):
                codes, scale = Q.block8(x[:, 64 * j: 64 * j + 64])
                assert torch.equal(got, codes) and torch.equal(s, scale), (b, j)
            fresh.add(int(c.table[b, j]))
        for tail, x, old in ((c.p2_tail, rows[0], before[4]), (c.info_tail, rows[1], before[5])):
            rest = end % 64
            assert torch.equal(tail[b, :, :rest].cpu(), x[:, end - rest: end])
            assert torch.equal(tail[b, :, rest:], old[b, :, rest:])
    rest = [p for p in range(c.p2.shape[0]) if p not in fresh]
    for now, old in zip(c[:4], before[:4]):
        assert torch.equal(now[rest], old[rest])
    assert torch.equal(c.table, before[6])
    end = [h + n for h, n in zip(held, new)]
    for out in (BF16, F32):
        got = cache8_read(c, torch.tensor(end, device=cuda), 0, blocks * 64, dtype=out)
        for b in range(B):
            for g, x0, x1 in zip(got, (k0, v0), (k1, v1)):
                want = Q.held8(torch.cat([x0[b, :, : held[b]], x1[b, :, : new[b]]], 1))
                assert torch.equal(g[b, :, : end[b]].cpu(), want.float().to(out))
                assert (g[b, :, end[b]:] == 0).all()


def test_reads_at_any_position(cuda):
    """A row a sequence at device positions, before the first and behind the last, ranges that begin inside a block,
    into views of a larger buffer; pages that are not there read as NaN."""
    from mote_amd.cache8 import cache8_read

    B, H, D, held = 4, 2, 40, [100, 256, 0, 63]
    c, k, v = _filled(11, B, H, D, 5, BF16, cuda, held)
    hd = torch.tensor(held, device=cuda)
    want = [torch.stack([torch.nn.functional.pad(Q.held8(x[b, :, : held[b]]), (0, 0, 0, 400 - held[b])) for b in range(B)]).float()
            for x in (k, v)]
    for start in ([0, 64, 0, 62], [99, 255, 1, 63], [-5, 200, -64, 300], [1 << 50, -(1 << 60), 5, 60]):
        buf = torch.full((B, 9, H, D), 7.0, device=cuda, dtype=BF16).transpose(1, 2)
        out = (buf[:, :, 1:8], torch.empty(B, H, 7, D, device=cuda, dtype=BF16))
        got = cache8_read(c, hd, torch.tensor(start, device=cuda), 7, out=out)
        assert got[0].data_ptr() == out[0].data_ptr()
        for g, w in zip(got, want):
            for b in range(B):
                for r in range(7):
                    pos = start[b] + r
                    x = w[b, :, pos] if 0 <= pos < held[b] else torch.zeros(H, D)
                    assert torch.equal(g[b, :, r].cpu(), x.to(BF16)), (b, pos)
        assert (buf[:, :, 0] == 7).all() and (buf[:, :, 8] == 7).all()
    for start, rows in ((37, 150), (64, 64), (0, 1), (300, 20)):
        for g, w in zip(cache8_read(c, hd, start, rows, dtype=F32), want):
            x = torch.nn.functional.pad(w, (0, 0, 0, 64))[:, :, start: start + rows]
            assert torch.equal(g.cpu(), x)
    table = c.table.clone()
    c.table[1, 1], c.table[1, 3] = -1, c.p2.shape[0]
    got = cache8_read(c, hd, 0, 256)
    for g, w in zip(got, want):
        for j in range(4):
            x = g[1, :, 64 * j: 64 * j + 64].cpu()
            assert x.isnan().all() if j in (1, 3) else torch.equal(x, w[1, :, 64 * j: 64 * j + 64].to(BF16))
        assert torch.equal(g[0].cpu(), w[0, :, :256].to(BF16))
    c.table.copy_(table)
    assert cache8_read(c, 100, 100)[0].shape == (B, H, 0, D)
    far = cache8_read(c, torch.full((B,), 1 << 60, device=cuda), 320, 3)  # positions that no block of the table holds
    assert far[0].isnan().all() and far[1].isnan().all()


def test_rows_without_a_page_and_past_the_table(cuda):
    """Blocks that become whole without a page are dropped, rows past the table's end too; a start that the table does
    not reach stores nothing."""
    from mote_amd.cache8 import cache8_write

    B, H, D = 4, 2, 48
    c = _empty(B, H, D, 2, F32, cuda)
    c.table[0, 0], c.table[0, 1] = -7, c.p2.shape[0]
    before = [t.clone() for t in c]
    k, v = _rows(1, B, H, 200, D, F32).to(cuda), _rows(2, B, H, 200, D, F32).to(cuda)
    start = torch.tensor([0, 0, 129, -1], device=cuda)
    cache8_write(c, k, v, start, torch.tensor([130, 200, 9, 9], device=cuda))
    mine = c.table[1].long()
    for i, (codes, x) in enumerate(((c.p2, k), (c.info, v))):
        for j in range(2):
            want, _ = Q.block8(x[1, :, 64 * j: 64 * j + 64].cpu())
            assert torch.equal(_page(c, D, 1, j)[2 * i], want)
    others = [p for p in range(c.p2.shape[0]) if p not in mine.tolist()]
    for now, old in zip(c[:4], before[:4]):
        assert torch.equal(now[others], old[others])
    assert torch.equal(c.p2_tail, before[4]) and torch.equal(c.info_tail, before[5])  # 64 blocks end the table: no tail
    cache8_write(c, k[:, :, :0], v[:, :, :0], 128)
    cache8_write(c, k, v, torch.zeros_like(start), torch.tensor([0, -3, 0, 0], device=cuda))  # 200 rows: more than the table
    assert torch.equal(c.p2_tail, before[4])


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_extreme_blocks(cuda, dtype):
    """Zeros, the smallest scales, the largest values, NaN and infinities, ties between codes."""
    from mote_amd.cache8 import cache8_read, cache8_write

    H, D = 2, 32
    x = torch.randn(8, H, 64, D, generator=_gen(4))
    x[0] = 0.0
    x[1] *= 2.0 ** -118          # below the smallest scale: zeros
    x[2] = 0.0
    x[2, :, 5, 3] = 2.0 ** -112  # the smallest scale itself
    x[3] *= 2.0 ** 120
    x[4, 0, 63, 31], x[4, 1, 0, 0] = float("nan"), float("inf")
    x[5, 0, 7, 7] = -float("inf")
    # the maximum 448 makes codes of the values themselves: every midpoint between neighbours, and below the normals
    n = torch.arange(126)
    mag = lambda i: torch.where(i < 8, i * 2.0 ** -9, (1 + (i % 8) / 8.0) * 2.0 ** (i // 8 - 7).float())
    mid = (mag(n) + mag(n + 1)) / 2
    x[6] = 0.0
    x[6].view(H, -1)[:, :126], x[6].view(H, -1)[:, 126:252], x[6, :, 63, 31] = mid, -mid, 448.0
    x = x.to(dtype)
    c = _empty(8, H, D, 1, dtype, cuda)
    cache8_write(c, x.to(cuda), x.flip(3).contiguous().to(cuda), 0)
    for b in range(8):
        ck, sk, cv, sv = _page(c, D, b, 0)
        for got, s, r in ((ck, sk, x[b]), (cv, sv, x[b].flip(2))):
            codes, scale = Q.block8(r)
            assert torch.equal(s.nan_to_num(-1.0), scale.nan_to_num(-1.0)), b
            assert torch.equal(torch.where(scale.isnan()[:, None, None], 0.0, codes), got), b
    k, _ = cache8_read(c, 64, dtype=F32)
    assert k[4].isnan().all() and k[5, 0].isnan().all() and not k[5, 1].isnan().any() and (k[:2] == 0).all()


# ---- the decode step -------------------------------------------------------------------------------
def _tolerance(q, kvals, vvals, new, S, D, dtype):
    """What fp32 arithmetic can move y and g by, from the formula (per sequence and head, absolute).

    U: D products summed in any order, the scale, 1 / sqrt(D) and the value's own rounding: (D + 6) half steps of
    sum |q k| / sqrt(D); a bf16 dot instruction may also truncate instead of rounding, twice that. e = SiLU(U): slope
    at most 1.1, and a few steps of exp and rcp (2 ulp each): 8 half steps of |U|. A weight exp(e - LSE) is off by
    twice that bound (numerator and denominator); a lane adds 16 rows of a page, of a quarter of the pages at most,
    and 16 of the tail: chains of S / 16 + 32 terms, then lanes, waves, splits: 128 more. Both scale |I~| in the
    mean; y is rounded once to its dtype."""
    h = 2.0 ** -24
    if S == 0:
        e_w = torch.zeros(q.shape[0], dtype=torch.float64)
        vmax = new.abs().amax(-1)
    else:
        mag = (q[:, None].abs() * kvals[:, :S].abs()).sum(-1) / math.sqrt(D)
        e_u = 2 * (D + 6) * h * mag.amax(-1) + 8 * h * mag.amax(-1)
        e_w = 2 * 1.1 * e_u + (S / 16 + 160) * h
        vmax = torch.maximum(vvals[:, :S].abs().amax((-1, -2)), new.abs().amax(-1))
    self_mag = (q.abs() * new.abs()).sum(-1) / math.sqrt(D)
    # g = sigma(.): slope at most 1/4; its argument is off by e_w and a few steps of ln(S + 1) and the Self score
    e_g = 0.25 * (e_w + 16 * h * (2 + math.log(S + 2.0)) + 2 * (D + 4) * h * self_mag * 0.25) + 4 * h
    e_y = (e_w + 2 * e_g + 8 * h) * vmax
    return e_y, e_g, torch.finfo(dtype).eps / 2


def _step_case(cuda, seed, dtype, B, H, D, blocks, S):
    c, k, v = _filled(seed, B, H, D, blocks, dtype, cuda, S)
    x = torch.randn(B, 3, H, D, generator=_gen(seed + 2)).to(dtype)
    return c, k, v, x, torch.tensor(0.5), torch.tensor(S)


def _check_step(x, k, v, lam, S, dtype, y, g):
    B, _, H, D = x.shape
    for b in range(B):
        s = int(S[b])
        q, kn, new = x[b].double()
        kb = torch.cat([Q.held8(k[b, :, :s]), kn[:, None]], 1)
        vb = torch.cat([Q.held8(v[b, :, :s]), new[:, None]], 1)
        yr, gr = O.relation_decode_ref(q[None], kb[None], vb[None], [s], lam.double(), 2.0, dtype=torch.float64)
        e_y, e_g, half = _tolerance(q, kb, vb, new, s, D, dtype)
        dy, dg = (y[b].cpu().double() - yr[0]).abs(), (g[b].cpu().double() - gr[0]).abs()
        assert (dy <= e_y[:, None] + half * yr[0].abs() * (1 + 2.0 ** -7)).all(), (b, s, float(dy.max()))
        assert (dg <= e_g).all(), (b, s, float(dg.max()), float(e_g.min()))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,H,D,blocks,S", [
    (1, 2, 8, 1, [5]), (2, 4, 48, 5, [0, 319]), (1, 2, 32, 18, [1024]), (3, 2, 40, 3, [1, 63, 129]), (2, 2, 16, 4, [62, 191]),
    (2, 8, 96, 11, [64, 65]), (1, 8, 96, 66, [4099]), (4, 2, 64, 10, [127, 128, 129, 511]), (2, 2, 128, 9, [575, 2]),
    (1, 6, 112, 6, [300]), (20, 8, 96, 4, list(range(0, 240, 12))), (2, 2, 72, 4, [255, 190]), (150, 2, 48, 70, [4400 - 13 * i for i in range(150)]),
    (1, 2, 24, 400, [25000])])
def test_decode_step_against_64_bits(cuda, dtype, B, H, D, blocks, S):
    """y and g against the oracle on the held values (no rotation: the query is the input itself); the new row in the
    tail as it is, a block that becomes whole in the format's own codes, everything else untouched."""
    from mote_amd.cache8 import relation_decode8

    c, k, v, x, lam, S = _step_case(cuda, 10 + D, dtype, B, H, D, blocks, S)
    before = [t.clone() for t in c]
    xd, Sd = x.to(cuda), S.to(cuda)
    y, g = relation_decode8(xd[:, 0], xd[:, 1], xd[:, 2], Sd, c, lam.to(cuda))
    assert y.dtype == dtype and g.dtype == F32 and torch.equal(Sd.cpu(), S)
    _check_step(x[:12], k, v, lam, S, dtype, y, g)
    for b in range(B):
        s = int(S[b])
        for i, (tail, rows) in enumerate(((c.p2_tail, k), (c.info_tail, v))):
            assert torch.equal(tail[b, :, s % 64].cpu(), x[b, 1 + i])
            if s % 64 == 63:
                codes, scale = Q.block8(torch.cat([rows[b, :, s - 63: s], x[b, 1 + i][:, None]], 1))
                page = _page(c, D, b, s // 64)
                assert torch.equal(page[2 * i], codes) and torch.equal(page[2 * i + 1], scale)
                t = int(c.table[b, s // 64])
                for now, old in zip(c[2 * i: 2 * i + 2], before[2 * i: 2 * i + 2]):
                    now[t] = old[t]
            tail[b, :, s % 64] = before[4 + i][b, :, s % 64]
    for now, old in zip(c, before):
        assert torch.equal(now, old)


@pytest.mark.parametrize("layer", [0, 1])
@pytest.mark.parametrize("dtype,rope_f32", [(BF16, False), (BF16, True), (F32, False)])
def test_decode_step_with_rope_and_givens(cuda, dtype, rope_f32, layer):
    """RoPE at far positions and Givens: the step's own convention, as in the step over a bf16 cache. A table entry one
    rounding step off (the GPU's and the CPU's cos differ in the last bit of fp32) moves one query element by a step
    of its dtype; the bound is the reference's own for such steps (2e-2 in bf16, 1e-5 in fp32, relative to the
    largest value)."""
    from conftest import rel_err
    from mote_amd.cache8 import relation_decode8

    B, H, D, S = 3, 4, 96, [3967, 17, 2500]
    c, k, v, x, lam, S = _step_case(cuda, 77, dtype, B, H, D, 62, S)
    inv, theta = O.rope_inv_freq(D, 10000.0).float(), torch.rand(H // 2, generator=_gen(5)) * 0.6 - 0.3
    xd = x.to(cuda)
    y, g = relation_decode8(xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), c, lam.to(cuda), 2.0, inv.to(cuda), theta.to(cuda),
                            layer, rope_f32=rope_f32)
    q, kn, new = O.decode_rows_ref(x[:, 0], x[:, 1], x[:, 2], S.tolist(), inv, theta, layer, dtype,
                                   rope_dtype=F32 if rope_f32 else None)
    bound = 2e-2 if dtype == BF16 else 1e-5
    for b in range(B):
        s = int(S[b])
        kb = torch.cat([Q.held8(k[b, :, :s]), kn[b].double()[:, None]], 1)
        vb = torch.cat([Q.held8(v[b, :, :s]), new[b].double()[:, None]], 1)
        yr, gr = O.relation_decode_ref(q[b][None].double(), kb[None], vb[None], [s], lam.double(), 2.0, dtype=torch.float64)
        assert rel_err(y[b], yr[0]) < bound and rel_err(g[b], gr[0]) < bound
        # fp32: cos and sin of theta differ by an ulp each, 2^-23 of a value up to 1, so c x - s x' by at most
        # 2^-23 (|x| + |x'|) <= 2^-22 max|x|, below the bound; in bf16 the tables' rounding hides it
        got = c.info_tail[b, :, s % 64].cpu()
        assert torch.equal(got, new[b]) if dtype == BF16 else rel_err(got, new[b]) < bound
        assert rel_err(c.p2_tail[b, :, s % 64], kn[b]) < bound


def test_rows_that_a_sequence_does_not_hold_never_count(cuda):
    """NaN in every page behind the last block, in the tail from S on and in the pages of others changes nothing."""
    from mote_amd.cache8 import Cache8, relation_decode8

    for D, S in ((48, [70, 0]), (96, [1, 193]), (64, [128, 127]), (128, [255, 256])):
        c, k, v, x, lam, S = _step_case(cuda, 5, BF16, 2, 2, D, 6, S)
        p = Cache8(*(t.clone() for t in c))
        used = torch.cat([c.table[b, : int(S[b]) // 64] for b in range(2)]).tolist()
        dead = [i for i in range(c.p2.shape[0]) if i not in used]
        for scale in (p.p2_scale, p.info_scale):
            scale[dead] = float("nan")
        p.p2[dead], p.info[dead] = 0x7f, 0x7f
        for b in range(2):
            for tail in (p.p2_tail, p.info_tail):
                tail[b, :, int(S[b]) % 64:] = float("nan")
        p.table[:, max(int(s) // 64 + 1 for s in S):] = -1
        xd = x.to(cuda)
        a = relation_decode8(xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), c, lam.to(cuda))
        b_ = relation_decode8(xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), p, lam.to(cuda))
        assert torch.equal(a[0], b_[0]) and torch.equal(a[1], b_[1])


def test_missing_pages_and_bad_positions(cuda):
    """A block without a page, and a NaN block, show in their own sequence (and head); a position outside the table
    stores nothing."""
    from mote_amd.cache8 import relation_decode8

    c, k, v, x, lam, S = _step_case(cuda, 6, BF16, 6, 2, 64, 5, [200, 320, 7, 200, 191, 64])
    Sd = torch.tensor([200, 320, -1, 200, 191, 64], device=cuda)
    c.info_scale[int(c.table[0, 1]), 1] = float("nan")
    c.table[3, 2] = -1
    c.table[4, 2] = c.p2.shape[0]  # the block that becomes whole has no page: it is lost
    c.table[5, 1:] = -1            # not needed yet
    before = [t.clone() for t in c]
    xd = x.to(cuda)
    y, g = relation_decode8(xd[:, 0], xd[:, 1], xd[:, 2], Sd, c, lam.to(cuda))
    assert y[0, 1].isnan().all() and not y[0, 0].isnan().any() and not g[0].isnan().any()
    assert y[1:4].isnan().all() and g[1:4].isnan().all()
    assert not y[4:].isnan().any() and not g[4:].isnan().any()
    for now, old in zip(c[4:6], before[4:6]):
        assert torch.equal(now[1:3], old[1:3])
        now[0, :, 8], now[3, :, 8], now[4, :, 63], now[5, :, 0] = old[0, :, 8], old[3, :, 8], old[4, :, 63], old[5, :, 0]
        assert torch.equal(now, old)
    for now, old in zip(c[:4], before[:4]):
        assert torch.equal(now.float().nan_to_num(-1.0), old.float().nan_to_num(-1.0))


def test_advance_xm_run_and_given_outputs(cuda):
    from mote_amd.cache8 import decode8_workspace, relation_decode8

    B, H, D, blocks = 3, 4, 96, 8
    c, k, v, x, lam, S = _step_case(cuda, 8, BF16, B, H, D, blocks, [100, 0, 511])
    xd, Sd = x.to(cuda), S.to(cuda)
    ws = decode8_workspace(B, H, D, blocks * 64, cuda)
    y, g, xm = torch.full((B, H, D), 3.0, device=cuda, dtype=BF16), torch.full((B, H), 3.0, device=cuda), torch.full((B,), 3.0, device=cuda)
    before = [t.clone() for t in c]
    off = torch.zeros(1, dtype=torch.bool, device=cuda)
    args = (xd[:, 0], xd[:, 1], xd[:, 2], Sd, c, lam.to(cuda))
    kw = dict(workspace=ws, y=y, g=g, xm=xm, advance=True)
    relation_decode8(*args, run=off, **kw)
    assert (y == 3).all() and (g == 3).all() and (xm == 3).all() and torch.equal(Sd.cpu(), S)
    assert all(torch.equal(a, b) for a, b in zip(c, before))
    out = relation_decode8(*args, run=~off, **kw)
    assert out[0].data_ptr() == y.data_ptr() and torch.equal(Sd.cpu(), S + 1)
    want = torch.stack([g[:, i] for i in range(H)]).cumsum(0)[-1] / H
    assert torch.allclose(xm, want, rtol=4 * 2.0 ** -24, atol=0)  # four additions and a division
    for bad in (ws[:-1], decode8_workspace(B + 1, H, D, blocks * 64, cuda)):
        with pytest.raises(ValueError, match="workspace"):
            relation_decode8(*args, workspace=bad)


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_many_steps_equal_one_append(cuda, dtype):
    """130 steps over two block borders leave the same pages and tails as the rows appended in one call, and the same
    y as each step over a cache that was appended to."""
    from mote_amd.cache8 import cache8_write, decode8_workspace, relation_decode8

    B, H, D, blocks, n = 2, 4, 48, 5, 130
    c, k, v, _, lam, S = _step_case(cuda, 30, dtype, B, H, D, blocks, [50, 130])
    x = _rows(31, B, 3 * H, n, D, dtype).view(B, 3, H, n, D).to(cuda)
    other, _, _ = _filled(30, B, H, D, blocks, dtype, cuda, [50, 130])
    Sd, ws, lamd = S.to(cuda), decode8_workspace(B, H, D, blocks * 64, cuda), lam.to(cuda)
    for t in range(n):
        row = x[:, :, :, t].contiguous()
        if t in (0, 13, 14, 62, 63, 129):
            probe, _, _ = _filled(30, B, H, D, blocks, dtype, cuda, [50, 130])
            cache8_write(probe, x[:, 1, :, :t], x[:, 2, :, :t], S.to(cuda))
            yp, gp = relation_decode8(row[:, 0], row[:, 1], row[:, 2], (S + t).to(cuda), probe, lamd)
        y, g = relation_decode8(row[:, 0], row[:, 1], row[:, 2], Sd, c, lamd, workspace=ws, advance=True)
        if t in (0, 13, 14, 62, 63, 129):
            assert torch.equal(y, yp) and torch.equal(g, gp)
    assert torch.equal(Sd.cpu(), S + n)
    cache8_write(other, x[:, 1], x[:, 2], S.to(cuda))
    for i, (a, b) in enumerate(zip(c, other)):
        if i in (4, 5):  # a tail holds what it last held behind its rows
            for s in range(B):
                r = int(S[s] + n) % 64
                assert torch.equal(a[s, :, :r], b[s, :, :r])
        else:
            assert torch.equal(a, b)


def test_steps_in_graphs(cuda):
    """Steps captured with the device position moving over a block border, replayed between eager work, against the
    same steps one by one; two graphs and eager calls share the workspace in turn."""
    from mote_amd.cache8 import Cache8, decode8_workspace, relation_decode8

    B, H, D, blocks = 2, 4, 64, 11
    c, k, v, x, lam, S = _step_case(cuda, 9, BF16, B, H, D, blocks, [125, 3])
    inv, theta = O.rope_inv_freq(D, 10000.0).float().to(cuda), (torch.rand(H // 2, generator=_gen(5)) * 0.6 - 0.3).to(cuda)
    copy = lambda: Cache8(*(t.clone() for t in c))
    twin, warm, other, third = copy(), copy(), copy(), copy()
    xd, Sd, St, lamd = x.to(cuda), S.to(cuda), S.to(cuda), lam.to(cuda)
    ws = decode8_workspace(B, H, D, blocks * 64, cuda)
    y, g = torch.empty(B, H, D, device=cuda, dtype=BF16), torch.empty(B, H, device=cuda)
    step = lambda c_, s, **kw: relation_decode8(xd[:, 0], xd[:, 1], xd[:, 2], s, c_, lamd, 2.0, inv, theta, 1, advance=True, **kw)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        step(warm, S.to(cuda), workspace=ws, y=y, g=g)
    torch.cuda.current_stream().wait_stream(side)
    graph, second = torch.cuda.CUDAGraph(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step(c, Sd, workspace=ws, y=y, g=g)
    So, S3 = torch.tensor([62, 0], device=cuda), torch.tensor([62, 0], device=cuda)
    with torch.cuda.graph(second):
        yo, go = step(other, So, workspace=ws)
    for _ in range(5):
        graph.replay()
        yt, gt = step(twin, St)
        torch.cuda.synchronize()
        assert torch.equal(y, yt) and torch.equal(g, gt) and torch.equal(Sd, St)
        second.replay()
        y3, g3 = step(third, S3, workspace=ws)
        torch.cuda.synchronize()
        assert torch.equal(yo, y3) and torch.equal(go, g3)
    for a, b in zip((*c, *other), (*twin, *third)):
        assert torch.equal(a, b)
    assert Sd.tolist() == [130, 8]


def test_shared_pages_another_stream_and_views_of_a_store(cuda):
    """Two sequences over the same pages, on a side stream, over a layer of a larger store."""
    from mote_amd.cache8 import Cache8, relation_decode8

    B, H, D = 2, 2, 96
    c, k, v, x, lam, S = _step_case(cuda, 12, F32, B, H, D, 5, [200, 200])
    xd, lamd, Sd = x.to(cuda), lam.to(cuda), S.to(cuda)
    shared = Cache8(*(t.clone() for t in c))
    shared.table[1, :3] = shared.table[0, :3]
    for tail in shared[4:6]:
        tail[1] = tail[0]
    stores = [torch.zeros(t.shape[0], 3, *t.shape[1:], dtype=t.dtype, device=cuda) for t in c[:6]]
    for s, t in zip(stores, shared):
        s[:, 1] = t
    wide = torch.full((B, 9), 99, dtype=torch.int32, device=cuda)
    wide[:, 2:7] = shared.table
    view = Cache8(*(s[:, 1] for s in stores), wide[:, 2:7])
    both = xd.clone()
    both[1] = both[0]
    want = relation_decode8(xd[:, 0], xd[:, 1], xd[:, 2], Sd, c, lamd)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = relation_decode8(both[:, 0], both[:, 1], both[:, 2], Sd, view, lamd)
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[0])
    for s in stores:
        assert (s[:, 0] == 0).all() and (s[:, 2] == 0).all()
    four = torch.cat([xd, xd[:, :1]], 1)  # y in the rows of the projections' own buffer
    again = relation_decode8(four[:, 0], four[:, 1], four[:, 2], Sd, c, lamd)[0]
    relation_decode8(four[:, 0], four[:, 1], four[:, 2], Sd, c, lamd, y=four[:, 3])
    assert torch.equal(four[:, 3], again) and torch.equal(four[:, :3], xd)


def test_offsets_past_32_bits(cuda):
    """A pool of more than 2^32 code bytes: blocks in its last pages are written, read and swept there."""
    from mote_amd.cache8 import Cache8, cache8_read, cache8_write, relation_decode8

    B, H, D, P = 2, 4, 128, 140_000
    codes = lambda *s: torch.empty(P, H, *s, dtype=torch.uint8, device=cuda)
    scale = lambda: torch.empty(P, H, device=cuda)
    c, k, v, x, lam, S = _step_case(cuda, 40, BF16, B, H, D, 4, [200, 255])
    big = Cache8(codes(8, 64, 16), scale(), codes(128, 64), scale(), c.p2_tail.clone(), c.info_tail.clone(), P - 1 - c.table)
    assert big.p2.numel() > 1 << 32
    for t, s in zip(big[:4], c[:4]):
        t[P - s.shape[0]:] = s.flip(0)
    new = [_rows(41 + i, B, H, 60, D, BF16).to(cuda) for i in range(2)]
    start = torch.tensor([140, 190], device=cuda)  # back to the middle of a block whose tail is gone: the same in both
    xd, lamd = x.to(cuda), lam.to(cuda)
    a = relation_decode8(xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), big, lamd)
    b = relation_decode8(xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), c, lamd)
    assert torch.equal(a[0], b[0]) and torch.equal(a[1], b[1])
    for cache in (big, c):
        cache8_write(cache, *new, start)
    for g, w in zip(cache8_read(big, start + 60, 0, 256), cache8_read(c, start + 60, 0, 256)):
        assert torch.equal(g, w)
    for t, s in zip(big[:4], c[:4]):
        assert torch.equal(t[P - s.shape[0]:], s.flip(0))


def test_two_calls_at_once(cuda):
    """Steps of two caches on two streams, each with a workspace of its own, against the same steps one by one."""
    from mote_amd.cache8 import decode8_workspace, relation_decode8

    cases = [_step_case(cuda, s, BF16, 4, 8, 96, 40, [2500, 100, 1999, 64]) for s in (50, 60)]
    args = []
    for c, k, v, x, lam, S in cases:
        xd = x.to(cuda)
        args.append((xd[:, 0], xd[:, 1], xd[:, 2], S.to(cuda), c, lam.to(cuda)))
    want = [relation_decode8(*a) for a in args]
    ws = [decode8_workspace(4, 8, 96, 40 * 64, cuda) for _ in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i].append(relation_decode8(*args[i], workspace=ws[i]))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for y, gate in g:
            assert torch.equal(y, w[0]) and torch.equal(gate, w[1])
