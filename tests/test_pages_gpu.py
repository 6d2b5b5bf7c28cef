"""The pages of the paged cache against plain loops on the host: every call's tables, counts and copies exactly."""

from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

BF16, F32 = torch.bfloat16, torch.float32


class Model:
    """Tables and counts as Python lists."""

    def __init__(self, B, blocks, pages):
        self.table, self.refs, self.S = [[-1] * blocks for _ in range(B)], [0] * pages, [0] * B

    def free(self, seqs):
        for s in seqs:
            for t in self.table[s]:
                if 0 <= t < len(self.refs):
                    self.refs[t] -= 1
            self.table[s] = [-1] * len(self.table[s])

    def fork(self, src, dst):
        n = min(max(self.S[src], 0) // 64, len(self.table[src]))
        for s in dst:
            self.free([s])
            self.table[s][:n] = self.table[src][:n]
            for t in self.table[s]:
                if t >= 0:
                    self.refs[t] += 1
            self.S[s] = self.S[src]

    def reserve(self, rows):
        missing = 0
        free = iter([p for p, n in enumerate(self.refs) if n == 0])
        for b, row in enumerate(self.table):
            for j in range(min(max(rows[b], 0) // 64, len(row))):
                if row[j] < 0:
                    row[j] = next(free, -1)
                    missing += row[j] < 0
        for row in self.table:
            for t in row:
                if t >= 0 and self.refs[t] == 0:
                    self.refs[t] = 1
        return missing

    def tensors(self, dev):
        return (torch.tensor(self.refs, dtype=torch.int32, device=dev), torch.tensor(self.table, dtype=torch.int32, device=dev),
                torch.tensor(self.S, device=dev))

    def same(self, refs, table, S):
        assert refs.tolist() == self.refs and table.tolist() == self.table and S.tolist() == self.S


@pytest.mark.parametrize("B,blocks,pages", [(1, 1, 1), (5, 9, 40), (16, 70, 900), (3, 2000, 7000), (300, 5, 1100), (40, 300, 12000)])
def test_a_life_of_calls(cuda, B, blocks, pages):
    """Reservations, forks and releases in turn, past the end of the pool too."""
    from mote_amd.pages import pages_fork, pages_free, pages_reserve

    g = torch.Generator().manual_seed(B)
    rand = lambda n: int(torch.randint(0, n, (1,), generator=g))
    m = Model(B, blocks, pages)
    refs, table, S = m.tensors(cuda)
    for turn in range(8):
        rows = [rand(64 * blocks + 1) for _ in range(B)]
        rows[rand(B)] = [0, 63, 64, 64 * blocks, -5, 1 << 40][turn % 6]
        missing = pages_reserve(refs, table, torch.tensor(rows, device=cuda))
        assert missing.dtype == torch.int32 and int(missing) == m.reserve(rows)
        m.same(refs, table, S)
        m.S = [min(r, 64 * sum(t >= 0 for t in row)) if r > 0 else 0 for r, row in zip(rows, m.table)]
        S.copy_(torch.tensor(m.S))
        order = torch.randperm(B, generator=g).tolist()
        src, dst = order[0], order[1: 1 + B // 3]
        pages_fork(refs, table, S, src, dst)
        m.fork(src, dst)
        m.same(refs, table, S)
        gone = order[B // 2: B // 2 + B // 4 + 1]
        pages_free(refs, table, gone)
        m.free(gone)
        m.same(refs, table, S)
    pages_free(refs, table, range(B))
    assert (refs == 0).all() and (table == -1).all()
    assert int(pages_reserve(refs, table, 64 * blocks)) == max(0, B * blocks - pages)
    m.free(range(B))
    m.reserve([64 * blocks] * B)
    m.same(refs, table, S)


def test_entries_that_name_no_page(cuda):
    """Numbers outside the pool are dropped and never counted; a position that the table does not reach shares nothing
    past its end."""
    from mote_amd.pages import pages_fork, pages_free

    refs = torch.tensor([2, 1, 0, 1], dtype=torch.int32, device=cuda)
    table = torch.tensor([[0, 9, -3], [0, 1, 3], [4, -1, 77]], dtype=torch.int32, device=cuda)
    S = torch.tensor([1 << 40, 7, 3], device=cuda)
    pages_free(refs, table, [2])
    assert refs.tolist() == [2, 1, 0, 1] and table[2].tolist() == [-1, -1, -1]
    pages_fork(refs, table, S, 0, [1])
    assert refs.tolist() == [2, 0, 0, 0] and table[1].tolist() == [0, 9, -3] and int(S[1]) == 1 << 40
    S[0] = -64
    pages_fork(refs, table, S, 0, [1, 2])
    assert refs.tolist() == [1, 0, 0, 0] and (table[1:] == -1).all() and S.tolist() == [-64, -64, -64]


@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("planes,B,H,D,rows", [(1, 2, 2, 8, 63), (4, 5, 4, 48, 64), (24, 3, 8, 96, 101), (2, 4, 2, 128, 1), (3, 3, 2, 40, 0)])
def test_fork_copies_the_newest_rows(cuda, dtype, planes, B, H, D, rows):
    """Exactly the rows of the source's open block, in every plane, over a layer range of a larger store; nothing else."""
    from mote_amd.pages import pages_fork

    g = torch.Generator().manual_seed(D)
    store = torch.randn(planes, B + 2, H, 64, D, generator=g).to(dtype).to(cuda)
    before = store.clone()
    tails = store[:, 1: B + 1]
    refs, table = torch.zeros(9, dtype=torch.int32, device=cuda), torch.full((B, 3), -1, dtype=torch.int32, device=cuda)
    S = torch.full((B,), 5, device=cuda)
    S[1] = rows
    dst = [b for b in range(B) if b != 1][: max(1, B - 2)]
    pages_fork(refs, table, S, 1, dst, tails)
    want = before.clone()
    for b in dst:
        want[:, b + 1, :, : rows % 64] = before[:, 2, :, : rows % 64]
    assert torch.equal(store, want)
    assert [int(S[b]) for b in dst] == [rows] * len(dst)


@pytest.mark.parametrize("planes,P,P2,H,size,B,blocks", [(2, 9, 9, 2, 16, 2, 4), (6, 40, 30, 3, 3 * 4096, 4, 7), (2, 1500, 1500, 2, 1040, 5, 300),
                                                          (1, 64, 500, 8, 16384 + 16, 1, 64), (4, 33, 5, 1, 20000, 3, 6),
                                                          (2, 4096, 4096, 1, 16, 2, 3000), (1, 4097, 3000, 2, 32, 2, 3000), (1, 100, 90, 1, 48, 3, 6000)])
def test_compact(cuda, planes, P, P2, H, size, B, blocks):
    """Pages in use in the order of their numbers, into a smaller, a larger or too small a pool; the old one is left as
    it was, the new one's other pages too."""
    from mote_amd.pages import PagePool, pages_compact

    g = torch.Generator().manual_seed(P)
    codes = torch.randint(0, 256, (planes, P, size), generator=g, dtype=torch.uint8).to(cuda)
    scales = torch.rand(planes, P, H, generator=g).to(cuda)
    table = torch.randint(-2, P, (B, blocks), generator=g).int()
    refs = torch.bincount(table[table >= 0].long(), minlength=P).int()
    wide = torch.zeros(B, blocks + 3, dtype=torch.int32)
    wide[:, 1:-2] = table
    into = PagePool(torch.full((planes, P2, size), 7, dtype=torch.uint8, device=cuda), torch.full((planes, P2, H), 7.0, device=cuda),
                    torch.full((P2,), 7, dtype=torch.int32, device=cuda))
    pool = PagePool(codes, scales, refs.to(cuda))
    before = [t.clone() for t in pool]
    for _ in range(2):  # the second call finds the same operands
        got, missing = pages_compact(pool, wide.to(cuda)[:, 1:-2], into)
        live = [p for p in range(P) if refs[p] > 0]
        new = {p: i for i, p in enumerate(live) if i < P2}
        n = len(new)
        want = [[new.get(int(t), -1) for t in row] for row in table]
        assert got.tolist() == want
        assert int(missing) == sum(int(t) >= 0 and int(t) not in new for row in table for t in row)
        assert torch.equal(into.codes[:, :n], codes[:, live[:n]]) and torch.equal(into.scales[:, :n], scales[:, live[:n]])
        assert (into.codes[:, n:] == 7).all() and (into.scales[:, n:] == 7).all()
        assert into.refs.tolist() == [int(refs[p]) for p in live[:n]] + [0] * (P2 - n)
    for a, b in zip(pool, before):
        assert torch.equal(a, b)


def test_calls_in_a_graph(cuda):
    """A fork and a reservation captured and replayed between eager work: each replay as the eager calls."""
    from mote_amd.pages import pages_fork, pages_free, pages_reserve

    B, blocks, P = 4, 6, 30
    m = Model(B, blocks, P)
    refs, table, S = m.tensors(cuda)
    rows = torch.tensor([200, 130, 0, 64], device=cuda)
    pages_reserve(refs, table, rows), m.reserve(rows.tolist())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        pages_free(refs, table, [3])
        pages_fork(refs, table, S, 0, [1, 2])
        missing = pages_reserve(refs, table, rows)
    for turn in range(4):
        m.S[0] = 64 * turn + 3
        S[0] = m.S[0]
        rows.copy_(torch.tensor([250 + turn, 128 * turn, 70, 384]))
        graph.replay()
        m.free([3]), m.fork(0, [1, 2])
        want = m.reserve(rows.tolist())
        torch.cuda.synchronize()
        m.same(refs, table, S)
        assert int(missing) == want
