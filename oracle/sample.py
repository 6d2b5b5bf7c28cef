"""The draw of a token, on the CPU in 64 bits (numpy), from a whole sort."""

from __future__ import annotations

import numpy as np


def sample_ref(x, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(token, margin) of one row of logits [V]: the first token in the order (logit descending, index ascending) whose
    running weight exceeds u times the weight kept. margin: how far, in parts of the largest weight, any of the
    comparisons that led there was from the other answer. Settings and u are 32-bit numbers."""
    x = np.asarray(x, dtype=np.float64)
    u, T, p, m = (float(np.float32(t)) for t in (u, temperature, top_p, min_p))
    V, inf = len(x), float("inf")
    if np.isnan(x).any() or not x.max() > -inf or any(t != t for t in (u, T, p, m)):
        return -1, inf
    order = np.lexsort((np.arange(V), -x))
    if not T > 0 or m > 1:  # no weight reaches a min_p above 1: the first is all that is kept
        return int(order[0]), inf
    xs = x[order]
    w = np.ones(V, dtype=np.longdouble)
    rest = xs != xs[0]
    with np.errstate(over="ignore", invalid="ignore"):
        w[rest] = np.where(np.isinf(xs[rest]) | np.isinf(xs[0]), 0.0, np.exp((xs[rest] - xs[0]) / np.longdouble(T)))
    if 0 < top_k < V:
        w = w[:top_k]
    total, margin, kept = np.cumsum(w), inf, len(w)
    if p < 1.0:
        t = max(p, 0.0) * total[-1]
        kept = min(int(np.searchsorted(total, t, side="left")), len(w) - 1) + 1
        margin = min(margin, float(np.abs(total - t).min()))
    high = max(1, int((w >= m).sum()))
    if m > 0:
        margin = min(margin, float(np.abs(w[1:] - m).min()) if len(w) > 1 else inf)
    kept = min(kept, high)
    t = min(max(u, 0.0), 1 - 2.0 ** -24) * total[kept - 1]
    at = min(int(np.searchsorted(total[:kept], t, side="right")), kept - 1)
    if t > 0:
        margin = min(margin, float(np.abs(total[:kept] - t).min()))
    return int(order[at]), margin
