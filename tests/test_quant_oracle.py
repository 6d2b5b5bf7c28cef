"""The plain forms of the 4-bit and 8-bit formats (oracle/quant.py) on the CPU: rounding at every border,
the groups and rows without a scale, and that the checks built on them would see a wrong rule."""

from __future__ import annotations

import pytest
import torch

from oracle import quant as Q


def test_e2m1_borders_round_to_the_even_code():
    mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
    assert Q.nearest_code(mids).tolist() == [0, 2, 2, 4, 4, 6, 6]
    up, down = mids * (1 + 2.0 ** -23), mids * (1 - 2.0 ** -23)
    assert Q.nearest_code(up).tolist() == [1, 2, 3, 4, 5, 6, 7]
    assert Q.nearest_code(down).tolist() == [0, 1, 2, 3, 4, 5, 6]
    assert Q.nearest_code(torch.tensor([6.0, 6.5, 1e30]).double()).tolist() == [7, 7, 7]


def test_encode4_scales_and_bounds():
    g = torch.Generator().manual_seed(0)
    x = torch.randn(50, 96, generator=g) * torch.logspace(-6, 6, 50)[:, None]
    v, s = Q.encode4(x)
    err = (Q.values4(v, s) - x.double()).abs().unflatten(-1, (3, 32)).amax(-1)
    # the widest gap is 2 codes (4 to 6): half of it, and what rounding the scale to bf16 moves at 6
    assert (err <= s.double() * (1.0 + 6 * 2.0 ** -8)).all()
    assert (s.double() - x.abs().double().unflatten(-1, (3, 32)).amax(-1) / 6).abs().le(s.double() * 2.0 ** -8).all()


def test_encode4_groups_without_a_scale():
    x = torch.zeros(5, 40)
    x[0, 3] = float("inf")
    x[1, 35] = float("nan")
    x[2, 0] = 5.9 * 2.0 ** -126  # its scale is below the smallest normal number
    x[3, 0] = 6.0 * 2.0 ** -126
    v, s = Q.encode4(x)
    assert s[0, 0].isnan() and s[0, 1] == 0 and s[1, 1].isnan() and s[1, 0] == 0
    assert s[2, 0] == 0 and (v[2] == 0).all()
    assert s[3, 0].float() == 2.0 ** -126 and v[3, 0] == 6.0
    assert (s[4] == 0).all()


def test_quantize8_reaches_the_ends_and_marks_rows_without_a_scale():
    x = torch.tensor([[1.0, -2.0, 0.5], [0.0, 0.0, 0.0], [float("inf"), 1.0, 0.0], [2.0 ** -121, 0, 0]])
    q, s = Q.quantize8(x)
    assert q[0].tolist() == [64.0, -127.0, 32.0]  # 63.5 and 31.75
    assert (q[1:] == 0).all() and s[1] == 0 and s[2].isnan() and s[3] == 0


@pytest.mark.parametrize("plant", ["ties_up", "truncate", "wide_scale"])
def test_a_wrong_rule_shows(plant):
    """A planted mistake in the oracle's rounding differs from it on ordinary bf16 rows."""
    g = torch.Generator().manual_seed(1)
    x = torch.randn(200, 32, generator=g).bfloat16().float().double()
    v, s = Q.encode4(x)
    t = (x / s.double()).abs()
    if plant == "ties_up":
        mids = torch.tensor([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0], dtype=torch.float64)
        x = torch.cat([mids, torch.tensor([6.0]).double()])[None].expand(1, 8)
        v, s = Q.encode4(x)
        t = x / s.double()
        code = (t[..., None] >= mids).sum(-1)
    elif plant == "truncate":
        code = (t[..., None] >= Q.MAGNITUDES[1:]).sum(-1)
    else:
        wide = x.abs().amax(-1, keepdim=True) / 6.0  # not rounded to bf16
        code = Q.nearest_code((x / wide).abs())
    assert not torch.equal(Q.MAGNITUDES[code], v.abs())
