"""Derivatives that a cache in 8 bits would lose, on the CPU: refused before anything could be launched."""

from __future__ import annotations

import pytest
import torch

from mote_amd import _lib as L
from mote_amd.cache8 import cache8_read, cache8_write, cache8_zeros, relation_decode8

pytestmark = pytest.mark.skipif(not L.available(), reason="libmote_relation.so not built")

BF16 = torch.bfloat16


@pytest.mark.parametrize("name", ["p2_scale", "info_scale", "p2_tail", "info_tail"])
def test_a_cache_that_wants_a_gradient(name):
    """Tails and scales are results of a write and of a step, operands of a read: none has a derivative."""
    c = cache8_zeros(2, 4, 5, 128, 48, "cpu", BF16)
    k, x, S, lam = torch.zeros(2, 4, 8, 48, dtype=BF16), torch.zeros(2, 4, 48, dtype=BF16), torch.zeros(2, dtype=torch.int64), torch.tensor(0.5)
    calls = (lambda c: cache8_write(c, k, k), lambda c: relation_decode8(x, x, x, S, c, lam), lambda c: cache8_read(c, 10))
    leaf = c._replace(**{name: getattr(c, name).clone().requires_grad_(True)})
    for call in calls:
        with pytest.raises(RuntimeError, match="no backward"):
            call(leaf)
        with torch.no_grad(), pytest.raises(RuntimeError, match="MI355X"):
            call(leaf)
        with torch.autograd.forward_ad.dual_level(), pytest.raises(RuntimeError, match="dual"):
            call(c._replace(**{name: torch.autograd.forward_ad.make_dual(getattr(c, name), getattr(c, name).clone())}))
