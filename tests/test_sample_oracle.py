"""The oracle of the draw against its definition by brute force, and the frequencies that it gives."""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle.sample import sample_ref


def _brute(x, u, T, k, p, m):
    """Python loops, term by term."""
    order = sorted(range(len(x)), key=lambda i: (-x[i], i))
    if T == 0:
        return order[0]
    w = {i: math.exp((x[i] - max(x)) / T) for i in order}
    kept = order[:k] if k else order
    total, some, run = sum(w[i] for i in kept), [], 0.0
    for i in kept:
        if some and run >= p * total and p < 1:
            break
        some.append(i)
        run += w[i]
    some = [i for n, i in enumerate(some) if n == 0 or w[i] >= m]
    target, run = u * sum(w[i] for i in some), 0.0
    for i in some:
        run += w[i]
        if run > target:
            return i
    return some[-1]


@pytest.mark.parametrize("V", [1, 2, 7, 40])
@pytest.mark.parametrize("k,p,m", [(0, 1.0, 0.0), (3, 1.0, 0.0), (0, 0.5, 0.0), (0, 1.0, 0.25), (5, 0.75, 0.125), (1, 0.0, 1.0)])
def test_against_loops(V, k, p, m):
    g = np.random.default_rng(V)
    for _ in range(40):
        x, u, T = np.round(g.normal(size=V) * 4) / 2, float(np.float32(g.random())), [0.0, 0.5, 1.0, 2.0][g.integers(4)]
        token, margin = sample_ref(x, u, T, k, p, m)
        if margin > 1e-9:
            assert token == _brute(list(x), u, T, k, p, m)


def test_frequencies_and_ends():
    x = np.log(np.array([0.1, 0.4, 0.2, 0.3]))
    grid = (np.arange(1000) + 0.5) / 1000
    got = np.bincount([sample_ref(x, u)[0] for u in grid], minlength=4)
    assert np.abs(got - [100, 400, 200, 300]).max() <= 1
    assert sample_ref(x, 0.0)[0] == 1 and sample_ref(x, 1.0)[0] == 0  # the first and the last of the order
    assert [sample_ref(x, u, top_p=0.65)[0] for u in (0.0, 0.56, 0.58, 0.99)] == [1, 1, 3, 3]
    assert sample_ref(x, 0.99, top_k=1)[0] == 1 and sample_ref(x, 0.99, min_p=1.0)[0] == 1
    assert sample_ref([-math.inf] * 3, 0.5)[0] == -1 and sample_ref([0.0, math.nan], 0.5)[0] == -1
    assert sample_ref([0.0, math.inf, 1.0, math.inf], 0.6)[0] == 3 and sample_ref([0.0] * 4, 0.6)[0] == 2
