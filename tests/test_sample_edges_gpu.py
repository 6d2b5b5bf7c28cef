"""sample_tokens at the ends of its settings, on rows of every kernel: in registers and in pieces."""

from __future__ import annotations

import math

import numpy as np
import pytest
import torch

from oracle.sample import sample_ref

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [3, 271, 5000, 8192, 20000, 131072])
def test_min_p_above_one_keeps_the_first_alone(cuda, dtype, V):
    """w >= min_p holds for no token, and the first of the order is always kept: of equal largest logits the first one."""
    from mote_amd.sample import sample_tokens

    B = 6
    g = torch.Generator().manual_seed(V)
    x = torch.randn(B, V, generator=g).clamp(max=2.0)
    ties = torch.rand(B, V, generator=g) < 0.3
    ties[:, -1] = True
    x = torch.where(ties, 2.5, x).to(dtype).to(cuda)
    first = ties.int().argmax(1).tolist()
    u = torch.tensor([0.0, 0.3, 0.6, 0.9, 0.999, 1.0 - 2.0 ** -24], device=cuda)
    f = lambda *t: torch.tensor(t, dtype=F32, device=cuda)
    for m in (float(np.nextafter(np.float32(1), np.float32(2))), 5.0, math.inf):
        for kw in (dict(), dict(top_k=2), dict(top_p=0.9, temperature=0.5), dict(temperature=f(*[0.7] * B))):
            assert sample_tokens(x, u, min_p=m, **kw).tolist() == first
            assert sample_tokens(x, u, min_p=f(*[m] * B), **kw).tolist() == first
    # beside rows whose setting says otherwise, and rows without a token
    mixed = sample_tokens(x, u, min_p=f(5.0, 1.0, 5.0, 0.0, 1.0, 5.0)).tolist()
    alone = sample_tokens(x, u, min_p=1.0).tolist()
    free = sample_tokens(x, u).tolist()
    assert mixed == [first[0], alone[1], first[2], free[3], alone[4], first[5]]
    places = [torch.nonzero(t).flatten().tolist() for t in ties]
    assert alone == [p[int(float(t) * len(p))] for p, t in zip(places, u.double())]
    x[0, 1], u[1] = float("nan"), float("nan")
    assert sample_tokens(x, u, min_p=2.0).tolist() == [-1, -1] + first[2:]


def _near(V):
    """Weights are rounded by 2^-44 of the largest, V of them add up to V 2^-44 at most, and the weight kept that u and p
    are taken of is such a sum itself."""
    return 2 * V * 2.0 ** -44 + 2.0 ** -40


def _check(x, u, got, T, k, p, m):
    """Every row against the oracle; returns how many rows have a comparison too near to a border to be told."""
    near = 0
    for b in range(len(x)):
        want, margin = sample_ref(x[b].double().numpy(), float(u[b]), *(t[b] if isinstance(t, list) else t for t in (T, k, p, m)))
        if margin <= _near(x.shape[1]):
            near += 1
        else:
            assert int(got[b]) == want, (b, int(got[b]), want, margin)
    return near


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [5000, 8193, 20000, 70001])
@pytest.mark.parametrize("few", [100, 3000])
def test_differences_beyond_fp32(cuda, dtype, V, few):
    """Logits whose differences overflow fp32, with temperatures at which all of them have weight, masked ones among them."""
    from mote_amd.sample import sample_tokens

    g = torch.Generator().manual_seed(V + few)
    u = torch.tensor([0.0, 0.4, 0.9, 0.9973, 0.9999, 1.0 - 2.0 ** -24])
    x = torch.full((len(u), V), 2e38)
    for row in x:
        row[torch.randperm(V, generator=g)[:few]] = -2e38
    x[1, torch.randperm(V, generator=g)[:50]] = -math.inf
    x[2, torch.randperm(V, generator=g)[: V - 40]] = -math.inf
    x[2, 1], x[2, V - 1] = 2e38, -2e38
    x[4] = -x[4]  # nearly all far below the largest
    x = x.to(dtype)
    xd, ud = x.to(cuda), u.to(cuda)
    for T in (1e38, 3e38, math.inf, 1e37):
        for k, p, m in ((0, 1.0, 0.0), (V - 30, 1.0, 0.0), (0, 0.99973, 0.0), (V - 7, 0.9997, 1e-3)):
            got = sample_tokens(xd, ud, T, k, p, m)
            assert _check(x, u, got, T, k, p, m) == 0, (T, k, p, m)


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("V", [5000, 20000])
def test_settings_of_each_row(cuda, dtype, V):
    """Greedy and drawing rows in one batch, settings at the ends of their ranges, as device tensors and one by one."""
    from mote_amd.sample import sample_tokens

    B = 120
    g = torch.Generator().manual_seed(V)
    x, u = (torch.randn(B, V, generator=g) * 2.5).to(dtype), torch.rand(B, generator=g)
    T = [[0.0, 1.0, 0.3, 1e-30, 1e30, math.inf, 2.0][b % 7] for b in range(B)]
    k = [[0, 1, 5, V - 1, V, 1 << 40][b % 6] for b in range(B)]
    p = [[1.0, 0.0, 0.5, 0.999, 2.0][b % 5] for b in range(B)]
    m = [[0.0, 1.0, 0.01, 5.0][b % 4] for b in range(B)]
    u[:8] = torch.tensor([0.0, 1.0 - 2.0 ** -24, 2.0 ** -40, 0.5, 0.0, 1.0 - 2.0 ** -24, 1.0, -1.0])
    xd, ud = x.to(cuda), u.to(cuda)
    f = lambda t: torch.tensor(t, dtype=F32, device=cuda)
    got = sample_tokens(xd, ud, f(T), torch.tensor(k, device=cuda), f(p), f(m))
    # a temperature that makes every weight one, and logits rounded to few values, meet borders exactly
    assert _check(x, u, got, T, k, p, m) < B // 4
    assert bool(((got >= 0) & (got < V)).all())
    for b in range(0, B, 7):
        assert int(sample_tokens(xd[b: b + 1], ud[b: b + 1], T[b], k[b], p[b], m[b])) == int(got[b])
    again = sample_tokens(xd.flip(0), ud.flip(0), f(T).flip(0), torch.tensor(k, device=cuda).flip(0), f(p).flip(0), f(m).flip(0))
    assert torch.equal(again.flip(0), got)
