"""sample_tokens against the oracle in 64 bits: the same token wherever no comparison was nearer to the other answer
than fixed-point weights can tell."""

from __future__ import annotations

import math

import pytest
import torch

from oracle.sample import sample_ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32
# A weight is rounded by 2^-44 of the largest, 2^20 of them add up to 2^-24 at worst; the weights kept that u and p are
# taken of are sums themselves: twice that. Roundings are independent of the order, so sums of V stay near
# sqrt(V) 2^-44, but the bound holds for any.
def _near(V):
    return 2 * V * 2.0 ** -44 + 2.0 ** -40


def _check(x, u, got, T=1.0, k=0, p=1.0, m=0.0):
    """Every row's token; settings are numbers or a list per row. Returns how many rows were near a border."""
    B, V = x.shape
    per = lambda t: t if isinstance(t, list) else [t] * B
    near = 0
    for b in range(B):
        want, margin = sample_ref(x[b].double().numpy(), float(u[b]), per(T)[b], per(k)[b], per(p)[b], per(m)[b])
        if margin <= _near(V):
            near += 1
        else:
            assert int(got[b]) == want, (b, int(got[b]), want, margin)
    return near


def _case(seed, B, V, dtype, scale=2.5):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(B, V, generator=g) * scale).to(dtype), torch.rand(B, generator=g)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("B,V", [(1, 1), (5, 2), (64, 271), (3, 512), (3, 513), (2, 1024), (4, 1025), (8, 8192), (3, 8193), (4, 32768),
                                 (3, 32771), (2, 131072), (1, 262147)])
@pytest.mark.parametrize("T,k,p,m", [(1.0, 0, 1.0, 0.0), (0.7, 40, 0.9, 0.0), (1.3, 0, 0.95, 0.02), (0.0, 5, 0.5, 0.1)])
def test_against_the_oracle(cuda, dtype, B, V, T, k, p, m):
    from mote_amd.sample import sample_tokens

    x, u = _case(V + B, B, V, dtype)
    got = sample_tokens(x.to(cuda), u.to(cuda), temperature=T, top_k=k, top_p=p, min_p=m)
    assert got.dtype == torch.int64 and got.shape == (B,)
    assert _check(x, u, got, T, k, p, m) == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
def test_settings_of_each_row(cuda, dtype):
    """Every row its own settings, ends of their ranges among them, as device tensors and one by one."""
    from mote_amd.sample import sample_tokens

    B, V = 120, 700
    x, u = _case(1, B, V, dtype)
    T = [[0.0, 1.0, 0.3, 1e-30, 1e30, math.inf, 2.0][b % 7] for b in range(B)]
    k = [[0, 1, 5, 699, 700, 1 << 40][b % 6] for b in range(B)]
    p = [[1.0, 0.0, 0.5, 0.999, 2.0][b % 5] for b in range(B)]
    m = [[0.0, 1.0, 0.01, 5.0][b % 4] for b in range(B)]
    u[:8] = torch.tensor([0.0, 1.0 - 2.0 ** -24, 2.0 ** -40, 0.5, 0.0, 1.0 - 2.0 ** -24, 1.0, -1.0])
    xd, ud = x.to(cuda), u.to(cuda)
    f = lambda t: torch.tensor(t, dtype=F32, device=cuda)
    got = sample_tokens(xd, ud, f(T), torch.tensor(k, device=cuda), f(p), f(m))
    # a temperature that makes every weight one, and logits rounded to few values, meet borders exactly
    assert _check(x, u, got, T, k, p, m) < B // 4
    for b in range(0, B, 7):
        one = sample_tokens(xd[b: b + 1], ud[b: b + 1], T[b], k[b], p[b], m[b])
        assert int(one) == int(got[b])
    again = sample_tokens(xd.flip(0), ud.flip(0), f(T).flip(0), torch.tensor(k, device=cuda).flip(0), f(p).flip(0), f(m).flip(0))
    assert torch.equal(again.flip(0), got)


@pytest.mark.parametrize("V", [271, 3000, 20000, 70000])
def test_equal_logits(cuda, V):
    """Ties go to the lowest index first: all equal, two values, few values, and zeros of both signs. With equal weights
    and u on a power of two times whole numbers every border is exact, so nothing is near by accident."""
    from mote_amd.sample import sample_tokens

    us = [0.0, 0.25, 0.3, 0.5, 0.75, 0.999]
    x = torch.zeros(len(us), V)
    u = torch.tensor(us)
    got = sample_tokens(x.to(cuda), u.to(cuda))
    assert got.tolist() == [int(float(t) * V) for t in u]
    x[:, ::2] = -0.0
    assert sample_tokens(x.to(cuda), u.to(cuda)).tolist() == got.tolist()
    assert sample_tokens(x.to(cuda), u.to(cuda), temperature=0.0).tolist() == [0] * len(us)
    # the first 100 of the order are indices 0..99
    assert sample_tokens(x.to(cuda), u.to(cuda), top_k=100).tolist() == [int(float(t) * 100) for t in u]
    # half of the weight: the first ceil(V / 2)
    half = -(-V // 2)
    assert sample_tokens(x.to(cuda), u.to(cuda), top_p=0.5).tolist() == [int(float(t) * half) for t in u]
    g = torch.Generator().manual_seed(V)
    x = torch.randint(0, 3, (8, V), generator=g).float()
    u = torch.rand(8, generator=g)
    for kw in (dict(), dict(T=0.5, k=V // 3), dict(p=0.8), dict(m=0.2), dict(T=2.0, k=V // 2, p=0.7, m=0.3)):
        got = sample_tokens(x.to(cuda), u.to(cuda), kw.get("T", 1.0), kw.get("k", 0), kw.get("p", 1.0), kw.get("m", 0.0))
        assert _check(x, u, got, **kw) == 0


def test_flat_logits(cuda):
    """Logits that differ by little, in the last places of their type."""
    from mote_amd.sample import sample_tokens

    for dtype, scale, shift in ((F32, 1e-6, 10.0), (F32, 1e-38, 0.0), (BF16, 1e-2, 100.0), (F32, 1e30, 0.0), (F32, 3e38, 0.0)):
        x, u = _case(3, 4, 9000, F32, 1.0)
        x = (x.clamp(-1.0, 1.0) * scale + shift).to(dtype)
        assert _check(x, u, sample_tokens(x.to(cuda), u.to(cuda))) == 0
        # the first 500 of the order have the largest logit (a sixth of each row was clamped to it): their weights are
        # one in any arithmetic, the border at half of them is met exactly, and the draw is from the first 250
        assert ((x == x.amax(1, keepdim=True)).sum(1) >= 500).all()
        got = sample_tokens(x.to(cuda), u.to(cuda), 1.0, 500, 0.5)
        assert got.tolist() == [sample_ref(x[b].double().numpy(), float(u[b]), 1.0, 500, 0.5)[0] for b in range(4)]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [271, 5000, 40001])
def test_masks_infinities_and_nan(cuda, dtype, V):
    """Tokens at -inf are never drawn, nor those at the type's lowest value beside others; rows that are all -inf or hold
    a NaN anywhere give -1; logits of +inf share the draw."""
    from mote_amd.sample import sample_tokens

    inf = float("inf")
    x, u = _case(V, 12, V, dtype)
    x[0, torch.arange(V) % 7 != 3] = -inf
    x[1] = -inf
    x[1, V - 1] = -5.0
    x[2] = -inf
    x[3, V // 2] = float("nan")
    x[4, 0], x[4, 5] = float("nan"), inf
    x[5, [3, V - 2, 9]] = inf
    x[6, 10:] = torch.finfo(dtype).min
    x[7] = torch.finfo(dtype).min
    x[8] = -inf
    x[8, 7], x[8, 8] = torch.finfo(dtype).min, torch.finfo(dtype).max
    u[9] = float("nan")
    x[10] = inf
    for T, k, p, m in ((1.0, 0, 1.0, 0.0), (0.5, 3, 0.9, 0.1), (float("inf"), 0, 0.5, 0.0), (0.0, 0, 1.0, 0.0)):
        got = sample_tokens(x.to(cuda), u.to(cuda), T, k, p, m)
        for b in (2, 3, 4, 9):
            assert int(got[b]) == -1
        assert int(got[0]) % 7 == 3 and int(got[1]) == V - 1 and int(got[5]) in (3, 9, V - 2) and int(got[8]) in (7, 8)
        _check(x, u, got, T, k, p, m)


def test_strides_streams_out_and_run(cuda):
    """Rows of a wider buffer at any element, columns of one, a side stream, a given result, the predicate."""
    from mote_amd.sample import sample_tokens

    for dtype, V in ((BF16, 301), (F32, 9001), (BF16, 33333)):
        B = 5
        x, u = _case(V, B, V, dtype)
        want = sample_tokens(x.to(cuda), u.to(cuda), 0.9, 50, 0.9)
        wide = torch.full((B, V + 6), 9.0, dtype=dtype, device=cuda)
        wide[:, 3:-3] = x
        assert torch.equal(sample_tokens(wide[:, 3:-3], u.to(cuda), 0.9, 50, 0.9), want)
        assert torch.equal(sample_tokens(x.t().contiguous().t().to(cuda), u.to(cuda), 0.9, 50, 0.9), want)
        xd, ud = x.to(cuda), u.to(cuda)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = sample_tokens(xd, ud, 0.9, 50, 0.9)
        torch.cuda.current_stream().wait_stream(side)
        assert torch.equal(got, want)
        out = torch.full((B,), 77, device=cuda)
        run = torch.zeros(1, dtype=torch.uint8, device=cuda)
        sample_tokens(xd, ud, 0.9, 50, 0.9, out=out, run=run)
        assert (out == 77).all()
        run.fill_(1)
        assert sample_tokens(xd, ud, 0.9, 50, 0.9, out=out, run=run).data_ptr() == out.data_ptr()
        assert torch.equal(out, want)
        same = sample_tokens(xd[:1].expand(B, V), ud[:1].expand(B).contiguous(), 0.9, 50, 0.9)
        assert (same == want[0]).all()
    assert sample_tokens(torch.zeros(0, 9, device=cuda), torch.zeros(0, device=cuda)).shape == (0,)


def test_in_a_graph(cuda):
    """Logits, random numbers and settings change between replays."""
    from mote_amd.sample import sample_tokens

    B, V = 6, 12000
    x, u = torch.zeros(B, V, device=cuda), torch.zeros(B, device=cuda)
    T, k = torch.ones(B, device=cuda), torch.zeros(B, dtype=torch.int64, device=cuda)
    sample_tokens(x, u, T, k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = sample_tokens(x, u, T, k)
    for turn in range(4):
        xs, us = _case(turn, B, V, F32)
        x.copy_(xs), u.copy_(us), T.fill_(0.5 + turn), k.fill_(100 * turn)
        graph.replay()
        eager = sample_tokens(x, u, T, k)
        torch.cuda.synchronize()
        assert torch.equal(got, eager)
        assert _check(xs, us, got, 0.5 + turn, 100 * turn) == 0


@pytest.mark.parametrize("dtype,B,V", [(BF16, 300, 9000), (F32, 700, 8200), (F32, 1, 1 << 20), (BF16, 2, (1 << 20) - 5)])
def test_many_rows_in_pieces_and_the_longest_rows(cuda, dtype, B, V):
    """More rows than compute units, each in two pieces, and the longest rows there are; equal rows draw equal tokens."""
    from mote_amd.sample import sample_tokens

    x, u = _case(V + B, min(B, 40), V, dtype)
    x, u = x.repeat(-(-B // 40), 1)[:B], u.repeat(-(-B // 40))[:B]
    for T, k, p, m in ((1.0, 0, 0.97, 0.0), (0.8, 300, 1.0, 1e-3)):
        got = sample_tokens(x.to(cuda), u.to(cuda), T, k, p, m)
        assert torch.equal(got, got[:40].repeat(-(-B // 40))[:B])
        assert _check(x[:40], u[:40], got, T, k, p, m) == 0


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [271, 3000, 7000, 40001])
def test_top_k_beyond_the_unmasked_and_coarse_logits(cuda, dtype, V):
    """A top-k that reaches into tokens at -inf, or at the type's lowest value, keeps what there is; many tokens that share few
    values are told apart by their indices."""
    from mote_amd.sample import sample_tokens

    x, u = _case(V, 9, V, dtype)
    for low in (-float("inf"), torch.finfo(dtype).min):
        y = x.clone()
        for b, left in enumerate((1, 2, 5, 30, 49, 50, 51, 100, 200)):
            keep = torch.randperm(V, generator=torch.Generator().manual_seed(b))[:left]
            y[b] = low
            y[b, keep] = x[b, keep]
        for p, m in ((1.0, 0.0), (0.9, 0.01)):
            got = sample_tokens(y.to(cuda), u.to(cuda), 0.8, 50, p, m)
            assert _check(y, u, got, 0.8, 50, p, m) == 0
            whole = sample_tokens(y.to(cuda), u.to(cuda), 0.8, 0, p, m)
            assert got[:6].tolist() == whole[:6].tolist()
    # eighths below 1: ties of V / 8 tokens and more
    x = (x.float().abs() * 4).floor().clamp(max=7).to(dtype) / 8
    for T, k, p, m in ((1.0, 0, 1.0, 0.0), (0.7, V // 2, 0.9, 0.0), (1.5, V // 3, 1.0, 0.5)):
        got = sample_tokens(x.to(cuda), u.to(cuda), T, k, p, m)
        assert _check(x, u, got, T, k, p, m) == 0


@pytest.mark.parametrize("dtype,V", [(BF16, 131072), (F32, 60001), (F32, 6000)])
def test_a_row_alone_and_in_a_batch(cuda, dtype, V):
    """A row goes in other pieces, or by another kernel, when it is alone; its token is the same."""
    from mote_amd.sample import sample_tokens

    B = 300
    x, u = _case(V, B, V, dtype)
    xd, ud = x.to(cuda), u.to(cuda)
    kw = dict(temperature=1.2, top_k=V // 5, top_p=0.98, min_p=1e-5)
    whole = sample_tokens(xd, ud, **kw)
    part = sample_tokens(xd[:20], ud[:20], **kw)
    assert torch.equal(part, whole[:20])
    for b in (0, 7, 19, 299):
        assert int(sample_tokens(xd[b: b + 1], ud[b: b + 1], **kw)) == int(whole[b])
