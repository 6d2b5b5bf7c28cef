"""The draw's oracle at the ends of its settings, on the CPU."""

from __future__ import annotations

import math

import numpy as np
import pytest

from oracle.sample import sample_ref


@pytest.mark.parametrize("m", [float(np.nextafter(np.float32(1), np.float32(2))), 5.0, math.inf])
def test_min_p_above_one_keeps_the_first_alone(m):
    """No weight reaches it, and the first token of the order is always kept: equal logits behind it go."""
    for u in (0.0, 0.6, 0.999):
        token, margin = sample_ref([1.0, 1.0, 0.0], u, min_p=m)
        assert token == 0 and margin > 1e-7
        assert sample_ref([0.0, 3.0, 3.0, 3.0], u, 0.5, 3, 0.9, m)[0] == 1
    assert sample_ref([1.0, 1.0, 0.0], 0.6, min_p=1.0)[0] == 1
    assert sample_ref([1.0, math.nan], 0.6, min_p=m)[0] == -1 and sample_ref([1.0, 1.0], math.nan, min_p=m)[0] == -1
