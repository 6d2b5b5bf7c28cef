"""Products in 8-bit integers on the GPU: codes and scales bit for bit, and y within one rounding of the
exact integer sums (the sums have no order)."""

from __future__ import annotations

import pytest
import torch

from oracle import quant as Q

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


def _x(seed, M, K, dtype, scale=1.0):
    x = torch.randn(M, K, generator=torch.Generator().manual_seed(seed)) * scale
    x[:, :: max(1, K // 5)] *= 6.0
    return x.to(dtype)


def _check(y, x, w):
    """float(acc) sx sw: a rounding of acc past 2^24, of the two products, and of y's dtype."""
    ref = Q.int8_linear_ref(x.reshape(-1, x.shape[-1]), w).reshape(y.shape)
    half = torch.finfo(y.dtype).eps / 2 if y.dtype == BF16 else 0.0
    tol = ref.abs() * (half + 3 * 2.0 ** -24) * (1 + 2.0 ** -7)
    d = (y.cpu().double() - ref).abs()
    assert (d <= tol).all(), float((d - tol).max())


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K", [(1, 1), (3, 127), (5, 128), (2, 129), (4, 768), (7, 2049), (1, 5000), (9, 4095), (21, 96),
                                 (37, 200), (35, 384), (19, 385), (10, 640), (11, 1000), (6, 4097)])
def test_quantize_rows_bit_for_bit(cuda, dtype, M, K):
    from mote_amd.int8 import quantize_rows

    x = _x(K, M, K, dtype)
    q, s = quantize_rows(x.to(cuda))
    rq, rs = Q.quantize8(x)
    assert q.shape == (M, (K + 127) // 128 * 128) and (q[:, K:] == 0).all()
    assert torch.equal(q[:, :K].cpu().double(), rq) and torch.equal(s.cpu().double(), rs)


def test_quantize_rows_special_rows_and_strides(cuda):
    from mote_amd.int8 import quantize_rows

    x = _x(3, 12, 300, F32)
    for r, v in enumerate((float("inf"), float("nan"), -float("inf"), 2.0 ** -121, 1e-44, 3.3e38)):
        x[r] = 0.0 if r in (3, 4) else x[r]
        x[r, 299 - r] = v
    x[6] = 0.0
    x[7] = torch.arange(300) * 0.5  # ties: half steps of max / 127 = 149.5 / 127
    x[8, :254] = torch.arange(-127, 127) + 0.5
    x[8, 254:] = 127.0
    rq, rs = Q.quantize8(x)
    for t in (x.to(cuda), x.to(cuda).t().contiguous().t(), torch.cat([x, x], 1).to(cuda)[:, 300:],
              torch.cat([torch.zeros(12, 1), x], 1).to(cuda)[:, 1:]):
        q, s = quantize_rows(t)
        assert torch.equal(q[:, :300].cpu().double(), rq)
        assert torch.equal(s.cpu().isnan(), rs.isnan()) and torch.equal(s.cpu().double().nan_to_num(-1.0), rs.nan_to_num(-1.0))
    same = x[10:11].to(cuda).expand(5, 300)  # rows at stride zero
    q, s = quantize_rows(same)
    assert torch.equal(q[:, :300].cpu().double(), rq[10:11].expand(5, 300))


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("M,K,N", [(1, 768, 2304), (16, 768, 768), (5, 64, 1), (16, 4096, 48), (33, 4000, 300), (64, 768, 130), (50, 700, 40), (3, 1000, 17), (2, 1, 5),
                                   (9, 2050, 271), (17, 128, 16), (64, 520, 271), (130, 768, 300), (257, 129, 129),
                                   (300, 1024, 128), (1, 5000, 40), (1000, 96, 64), (128, 4224, 256), (520, 200, 1031),
                                   (12, 1500, 50), (20, 2000, 33), (700, 1200, 1700), (2000, 100, 999),
                                   (1100, 1100, 2470)])
def test_linear_is_one_rounding_from_exact(cuda, dtype, M, K, N):
    from mote_amd.int8 import int8_linear, int8_weight

    x, w = _x(M + K, M, K, dtype), _x(N, N, K, F32, 0.05)
    y = int8_linear(x.to(cuda), int8_weight(w.to(cuda)))
    assert y.shape == (M, N) and y.dtype == dtype
    _check(y, x, w)


@pytest.mark.parametrize("M,K,N", [(700, 256, 1100), (700, 1200, 1700), (2000, 256, 999), (1100, 1100, 2500), (2300, 200, 2500), (6300, 96, 2300), (16384, 64, 2304), (5000, 384, 9000)])
def test_every_tile_size_gives_a_row_its_own_result(cuda, M, K, N):
    """Sizes over the range of tiles (the rule picks by rounds of workgroups): rows, the last ones and those at
    tile borders among them, equal the few-token form's bit for bit."""
    from mote_amd.int8 import int8_linear, int8_weight

    x, w8 = _x(1, M, K, BF16).to(cuda), int8_weight(_x(2, N, K, BF16).to(cuda))
    y = int8_linear(x, w8)
    for at in (0, 120, 185, 250, 500, M // 2, M - 16):
        at = min(at, M - 16)
        assert torch.equal(y[at: at + 16], int8_linear(x[at: at + 16], w8)), at


def test_forms_agree_bit_for_bit(cuda):
    """The few-token and the many-token form give a token the same result, alone or in any batch."""
    from mote_amd.int8 import int8_linear, int8_weight

    for dtype in (BF16, F32):
        for K, N in ((768, 2304), (520, 271), (4096, 130)):
            x, w8 = _x(1, 300, K, dtype).to(cuda), int8_weight(_x(2, N, K, BF16).to(cuda))
            y = int8_linear(x, w8)
            for a, b in ((0, 1), (5, 21), (284, 300), (100, 117), (0, 64), (33, 82), (200, 265)):
                assert torch.equal(int8_linear(x[a:b], w8), y[a:b])


def test_leading_dims_strides_outputs_and_empty(cuda):
    from mote_amd.int8 import int8_linear, int8_weight

    w = _x(4, 40, 100, BF16)
    w8 = int8_weight(w.to(cuda))
    for B, T in ((2, 3), (3, 50)):
        x = _x(5, B * T, 100, BF16).view(B, T, 100)
        xd = x.to(cuda)
        y = int8_linear(xd, w8)
        assert y.shape == (B, T, 40)
        _check(y, x, w)
        wide = torch.cat([xd, xd], -1)
        assert torch.equal(int8_linear(wide[..., 100:], w8), y)
        assert torch.equal(int8_linear(xd.transpose(0, 1), w8), y.transpose(0, 1))
        odd = torch.cat([xd[..., :1], xd], -1)[..., 1:]  # rows off 16-byte boundaries
        assert torch.equal(int8_linear(odd, w8), y)
        out = torch.full((B * T, 60), 9.0, device=cuda, dtype=BF16)
        got = int8_linear(xd.reshape(-1, 100), w8, out=out[:, 7:47])
        assert got.data_ptr() == out[:, 7:].data_ptr() and torch.equal(out[:, 7:47], y.reshape(-1, 40))
        assert (out[:, :7] == 9).all() and (out[:, 47:] == 9).all()
        both = torch.cat([xd.reshape(-1, 100), out[:, :40]], 1)  # the result in other columns of x's own rows
        int8_linear(both[:, :100], w8, out=both[:, 100:])
        assert torch.equal(both[:, 100:], y.reshape(-1, 40)) and torch.equal(both[:, :100], xd.reshape(-1, 100))
    assert int8_linear(torch.empty(0, 100, device=cuda, dtype=BF16), w8).shape == (0, 40)
    assert int8_linear(xd[0, 0], w8).shape == (40,)


def test_a_row_with_a_nan_or_infinity_is_nan(cuda):
    from mote_amd.int8 import int8_linear, int8_weight

    for M in (6, 40):
        x = _x(7, M, 200, F32)
        x[1, 3], x[4, 199] = float("inf"), float("nan")
        x[2] = 0.0
        y = int8_linear(x.to(cuda), int8_weight(_x(8, 33, 200, F32).to(cuda))).cpu()
        assert y[1].isnan().all() and y[4].isnan().all() and (y[2] == 0).all()
        assert not y[[0, 2, 3, 5]].isnan().any()


def test_run_xm_and_graph(cuda):
    from mote_amd.int8 import int8_linear, int8_weight

    x, w8 = _x(9, 4, 256, BF16).to(cuda), int8_weight(_x(10, 64, 256, BF16).to(cuda))
    out, xm = torch.full((4, 64), 5.0, device=cuda, dtype=BF16), torch.full((4,), 5.0, device=cuda)
    g = torch.rand(4, 8, device=cuda)
    off = torch.zeros(1, dtype=torch.uint8, device=cuda)
    int8_linear(x, w8, out=out, run=off, g=g, xm=xm)
    assert (out == 5).all() and (xm == 5).all()
    int8_linear(x, w8, out=out, run=off + 1, g=g, xm=xm)
    assert torch.equal(out, int8_linear(x, w8))
    assert torch.allclose(xm, g.double().mean(1).float(), rtol=9 * 2.0 ** -24, atol=0)  # eight additions, a division
    many = _x(11, 200, 256, BF16).to(cuda)
    with pytest.raises(RuntimeError, match="64 rows"):
        int8_linear(many, w8, run=off)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        int8_linear(many, w8)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y_few, y_many = int8_linear(x, w8), int8_linear(many, w8)
    for i in range(3):
        x.copy_(_x(20 + i, 4, 256, BF16))
        many.copy_(_x(30 + i, 200, 256, BF16))
        graph.replay()
        a, b = int8_linear(x, w8), int8_linear(many, w8)
        torch.cuda.synchronize()
        assert torch.equal(y_few, a) and torch.equal(y_many, b)


def test_offsets_past_32_bits(cuda):
    """Outputs and inputs beyond 2^32 bytes: the last rows are those of a small call."""
    from mote_amd.int8 import int8_linear, int8_weight

    M, K, N = 1 << 20, 64, 2176
    w8 = int8_weight(_x(12, N, K, BF16).to(cuda))
    x = torch.zeros(M, K, device=cuda, dtype=BF16)
    tail = _x(13, 300, K, BF16).to(cuda)
    x[-300:] = tail
    y = int8_linear(x, w8)
    assert y.numel() * 2 > 1 << 32
    assert torch.equal(y[-300:], int8_linear(tail, w8)) and (y[:256] == 0).all() and (y[M // 2: M // 2 + 256] == 0).all()
