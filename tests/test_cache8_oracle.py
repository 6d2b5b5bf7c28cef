"""The oracle of blocks in 8 bits: every code's value, every border between two codes, scales and the error bound."""

from __future__ import annotations

import math

import pytest
import torch

from oracle import quant as Q


def _values():
    """The 127 magnitudes of e4m3, from its definition: 4 bits of exponent (bias 7), 3 of mantissa, 0x7f is NaN."""
    out = []
    for n in range(127):
        e, f = n >> 3, n & 7
        out.append(f / 8 * 2.0 ** -6 if e == 0 else (1 + f / 8) * 2.0 ** (e - 7))
    return torch.tensor(out, dtype=torch.float64)


def test_codes_and_borders():
    v = _values()
    assert v[-1] == 448 and torch.equal(v.float(), torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).float())
    assert torch.equal(Q.nearest_e4m3(v), v) and torch.equal(Q.nearest_e4m3(-v[1:]), -v[1:])
    mid = (v[1:] + v[:-1]) / 2
    even = torch.where(torch.arange(126) % 2 == 0, v[:-1], v[1:])
    assert torch.equal(Q.nearest_e4m3(mid), even)
    assert torch.equal(Q.nearest_e4m3(torch.nextafter(mid, mid + 1)), v[1:])
    assert torch.equal(Q.nearest_e4m3(torch.nextafter(mid, mid - 1)), v[:-1])
    assert Q.nearest_e4m3(torch.tensor([448.0001, 480.0, 1e30]).double()).tolist() == [448.0] * 3
    x = torch.randn(4096, generator=torch.Generator().manual_seed(0)) * 50
    assert torch.equal(Q.nearest_e4m3(x.double()), x.to(torch.float8_e4m3fn).double())
    assert not torch.equal(even, v[1:]) and not torch.equal(even, v[:-1])  # ties always up or down would fail


@pytest.mark.parametrize("size", [1e-30, 1e-3, 1.0, 1e4, 1e30])
def test_blocks(size):
    """The scale is one rounding of max / 448; a value is off by half a step of its code: 2^-4 of it, or half of the smallest
    code; the two roundings of the scale and the product's add 3 x 2^-24 to it."""
    x = torch.randn(3, 64, 40, generator=torch.Generator().manual_seed(1)).float() * size
    x[1] = x[1].exp2() if size == 1.0 else x[1]
    codes, scale = Q.block8(x)
    top = x.double().abs().amax((1, 2))
    assert ((scale - top / 448).abs() <= 2.0 ** -24 * top / 448).all()
    assert (codes.abs().amax((1, 2)) == 448).all()  # the largest value's code
    bound = torch.maximum(x.double().abs() * 2.0 ** -4, scale[:, None, None] * 2.0 ** -10) * (1 + 2.0 ** -20) + x.double().abs() * 2.0 ** -22
    assert ((Q.values8(x) - x.double()).abs() <= bound).all()


def test_blocks_without_a_scale():
    x = torch.ones(4, 64, 8)
    x[0] = 0
    x[1] = math.ldexp(1.0, -113)
    x[2, 63, 7] = math.inf
    x[3, 0, 0] = math.nan
    codes, scale = Q.block8(x)
    assert (codes[:2] == 0).all() and scale[:2].tolist() == [0.0, 0.0] and scale[2:].isnan().all()
    assert (Q.values8(x)[:2] == 0).all() and Q.values8(x)[2:].isnan().all()
    x[1] = math.ldexp(1.0, -112)
    assert Q.block8(x)[1][1] > 0


def test_held_rows():
    x = torch.randn(2, 150, 16, generator=torch.Generator().manual_seed(2))
    h = Q.held8(x)
    assert torch.equal(h[:, 128:], x[:, 128:].double())
    assert torch.equal(h[:, 64:128], Q.values8(x[:, 64:128])) and not torch.equal(h[:, :64], x[:, :64].double())
    assert torch.equal(Q.held8(x[:, :63]), x[:, :63].double())
