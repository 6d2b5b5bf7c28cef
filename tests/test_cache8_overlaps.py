"""Tensors of a call that lie over one another, on the CPU: whatever is written has a place of its own, or the call is
refused before anything could be launched."""

from __future__ import annotations

import itertools

import pytest
import torch

from mote_amd import _lib as L
from mote_amd.cache8 import Cache8, cache8_read, cache8_write, cache8_zeros, relation_decode8

pytestmark = pytest.mark.skipif(not L.available(), reason="libmote_relation.so not built")

BF16 = torch.bfloat16
B, H, P, D = 2, 4, 5, 48
BYTES = H * 3 * 64 * 16  # of a page, P2 or I~


def _over(raw, at, like):
    """A view of `like`'s sizes, contiguous, from byte `at` of raw on."""
    n = like.numel() * like.element_size()
    return raw[at: at + n].view(like.dtype).view(like.shape)


def _calls(c):
    k = torch.zeros(B, H, 8, D, dtype=BF16)
    x = torch.zeros(B, H, D, dtype=BF16)
    return (lambda: cache8_write(c, k, k.clone()),
            lambda: relation_decode8(x, x, x, torch.zeros(B, dtype=torch.int64), c, torch.tensor(0.5)))


def _refused(c):
    for call in _calls(c):
        with pytest.raises(ValueError, match="over one another|same rows"):
            call()


def _taken(c):
    for call in _calls(c):
        with pytest.raises(RuntimeError, match="MI355X"):
            call()


def test_any_two_tensors_of_a_cache():
    """Each pair of the seven with the later one's first bytes inside the earlier one's last, and the other way round."""
    c = cache8_zeros(B, H, P, 128, D, "cpu", BF16)
    for a, b in itertools.permutations(Cache8._fields, 2):
        first, second = getattr(c, a), getattr(c, b)
        size = first.numel() * first.element_size()
        raw = torch.zeros(size + second.numel() * second.element_size() + 64, dtype=torch.uint8)
        # 16-byte boundaries, so that nothing but the overlap is wrong
        end = -(-size // 16) * 16
        _refused(c._replace(**{a: _over(raw, 0, first), b: _over(raw, end - 16, second)}))
        _taken(c._replace(**{a: _over(raw, 0, first), b: _over(raw, end, second)}))


def test_records_of_a_page():
    """Codes and scales of P2 and I~ side by side in one record per page are places of their own, whatever the order; a record
    that is too short is not."""
    c = cache8_zeros(B, H, P, 128, D, "cpu", BF16)

    def records(stride, at_info, at_s2, at_si, shift=0):
        raw = torch.zeros(shift + (P + 1) * stride, dtype=torch.uint8)[shift:].as_strided((P, stride), (stride, 1))
        part = lambda at, n: raw[:, at: at + n]
        codes = lambda at, *s: part(at, BYTES).unflatten(1, s)
        scale = lambda at: part(at, 4 * H).view(torch.float32)
        return c._replace(p2=codes(0, H, 3, 64, 16), info=codes(at_info, H, 48, 64), p2_scale=scale(at_s2), info_scale=scale(at_si))

    whole = 2 * BYTES + 32
    _taken(records(whole, BYTES, 2 * BYTES, 2 * BYTES + 16))
    _taken(records(whole, BYTES + 32, BYTES, BYTES + 16))
    _refused(records(whole, BYTES, 2 * BYTES, 2 * BYTES))          # one place for both scales
    _refused(records(whole, BYTES, 2 * BYTES - 16, 2 * BYTES))     # scales over the codes
    _refused(records(whole, BYTES - 16, 2 * BYTES, 2 * BYTES + 16))
    tails = torch.zeros(B, 2, H, 64, D, dtype=BF16)
    _taken(c._replace(p2_tail=tails[:, 0], info_tail=tails[:, 1]))
    short = torch.zeros(4 * H * 64 * D, dtype=BF16)
    step = H * 64 * D
    view = lambda at, stride: short.as_strided((B, H, 64, D), (stride, 64 * D, D, 1), at)
    _taken(c._replace(p2_tail=view(0, 2 * step), info_tail=view(step, 2 * step)))
    _refused(c._replace(p2_tail=view(0, 2 * step), info_tail=view(step - D, 2 * step)))


def test_reading_takes_shared_places():
    c = cache8_zeros(B, H, P, 128, D, "cpu", BF16)
    with pytest.raises(RuntimeError, match="MI355X"):
        cache8_read(c._replace(info_tail=c.p2_tail, info_scale=c.p2_scale), 10)


def test_a_draw_over_its_operands():
    from mote_amd.sample import sample_tokens

    n, V = 4, 64
    x, u = torch.zeros(n, V), torch.zeros(n)
    raw = torch.zeros(n * V * 4 + 64, dtype=torch.uint8)
    logits = raw[: n * V * 4].view(torch.float32).view(n, V)
    ids = lambda at: raw[at: at + 8 * n].view(torch.int64)
    for at in (0, 32, n * V * 4 - 8):
        with pytest.raises(ValueError, match="out lies over"):
            sample_tokens(logits, u, out=ids(at))
    with pytest.raises(RuntimeError, match="MI355X"):
        sample_tokens(logits, u, out=ids(n * V * 4))
    for name, dt in (("temperature", torch.float32), ("top_p", torch.float32), ("min_p", torch.float32), ("top_k", torch.int64)):
        with pytest.raises(ValueError, match="out lies over"):
            sample_tokens(x, u, out=ids(0), **{name: raw[: n * dt.itemsize].view(dt)})
    with pytest.raises(ValueError, match="out lies over"):
        sample_tokens(x, raw[16: 16 + 4 * n].view(torch.float32), out=ids(0))
    with pytest.raises(ValueError, match="out lies over"):
        sample_tokens(x, u, out=ids(0), run=raw[7:8])


def test_pages_and_lengths():
    from mote_amd.pages import pages_fork, pages_reserve

    raw = torch.zeros(64, dtype=torch.int32)
    refs, table = raw[:8], raw[8:32].view(3, 8)
    for at in (2, 6, 28):
        S = raw[at: at + 6].view(torch.int64)
        with pytest.raises(ValueError, match="lies over"):
            pages_fork(refs, table, S, 0, [1])
        with pytest.raises(ValueError, match="lies over"):
            pages_reserve(refs, table, S)
    with pytest.raises(RuntimeError, match="MI355X"):
        pages_fork(refs, table, raw[32:38].view(torch.int64), 0, [1])
