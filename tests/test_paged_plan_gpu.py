"""ops.paged_plan against lists of pages kept in Python."""
import numpy as np
import pytest
import torch

from relax_b200 import ops

pytestmark = pytest.mark.gpu


class Pool:
    """The state on the device, and the same in Python."""

    def __init__(self, batch, width, pages, page, seed=0):
        self.rng = np.random.default_rng(seed)
        self.page, self.width, self.batch = page, width, batch
        self.free = self.rng.permutation(pages).astype(np.int32).tolist()
        self.tables, self.lengths = [[] for _ in range(batch)], [0] * batch
        i32 = dict(dtype=torch.int32, device="cuda")
        self.d_table = torch.full((batch, width + 3), -7, **i32)[:, :width]          # rows further apart than they are long
        self.d_lengths = torch.zeros(batch, **i32)
        self.d_free = torch.tensor(self.free, **i32)
        self.d_count = torch.tensor([pages], **i32)

    def want(self, counts, rows):
        back, status = [], 0
        have = [-(-n // self.page) for n in self.lengths]
        need = [-(-(n + c) // self.page) for n, c in zip(self.lengths, counts)]
        total = sum(max(c, 0) for c in counts)
        if any(not 0 <= n + c <= self.width * self.page for n, c in zip(self.lengths, counts)):
            status = -1
        elif total > rows:
            status = -2
        else:
            lacking = sum(max(w - h, 0) - max(h - w, 0) for h, w in zip(have, need)) - len(self.free)
            status = max(lacking, 0)
        positions, slots = np.full(rows, -1, np.int32), np.full(rows, -1, np.int64)
        starts = np.zeros(self.batch + 1, np.int32)
        if status == 0:
            for b in range(self.batch):
                self.free += self.tables[b][need[b]:have[b]]
                self.tables[b] = self.tables[b][:min(have[b], need[b])]
            at = 0
            for b, c in enumerate(counts):
                while len(self.tables[b]) < need[b]:
                    self.tables[b].append(self.free.pop())
                for i in range(max(c, 0)):
                    t = self.lengths[b] + i
                    positions[at], slots[at] = t, self.tables[b][t // self.page] * self.page + t % self.page
                    at += 1
                starts[b + 1] = at
                self.lengths[b] += c
        return status, starts, positions, slots

    def step(self, counts, rows, alias):
        before = self.d_table.clone(), self.d_free.clone()
        out = None
        if alias:
            out = ops.paged_plan_buffers(self.batch, rows, "cuda")._replace(lengths=self.d_lengths, free_count=self.d_count)
        got = ops.paged_plan(self.d_table, self.d_lengths, torch.tensor(counts, dtype=torch.int32, device="cuda"), self.d_free, self.d_count, self.page, rows,
                             out=out)
        had = list(self.lengths)
        status, starts, positions, slots = self.want(counts, rows)
        assert int(got.status) == status
        assert got.lengths.tolist() == self.lengths and int(got.free_count) == len(self.free)
        assert np.array_equal(got.starts.cpu().numpy(), starts)
        assert np.array_equal(got.positions.cpu().numpy(), positions) and np.array_equal(got.slots.cpu().numpy(), slots)
        assert self.d_free[: len(self.free)].tolist() == self.free
        table = self.d_table.cpu().numpy()
        for b, pages in enumerate(self.tables):
            assert table[b, : len(pages)].tolist() == pages
            kept = -(-max(had[b], self.lengths[b]) // self.page)
            assert np.array_equal(table[b, kept:], before[0][b, kept:].cpu().numpy())       # entries of no token are left alone
        if status:
            assert torch.equal(self.d_table, before[0]) and torch.equal(self.d_free, before[1])
        self.d_lengths, self.d_count = got.lengths, got.free_count
        return status


@pytest.mark.parametrize("alias", (False, True))
@pytest.mark.parametrize("page", (16, 128))
@pytest.mark.parametrize("batch,width,pages,rows", ((1, 4, 3, 40), (7, 9, 40, 300), (64, 20, 700, 4000), (700, 5, 2500, 9000)))
def test_calls_in_a_row(cuda_lib, batch, width, pages, rows, page, alias):
    p = Pool(batch, width, pages, page, seed=batch)
    seen = set()
    for i in range(12):
        most = max(1, min(width * page, 2 * rows // batch))
        counts = [int(p.rng.integers(0, most + 1)) if p.rng.random() < 0.6 else -int(p.rng.integers(0, n + 1)) for n in p.lengths]
        if i % 3 != 2:                           # (mostly calls that fit)
            counts = [min(c, width * page - n) for c, n in zip(counts, p.lengths)]
            while sum(max(c, 0) for c in counts) > rows:
                counts = [c // 2 if c > 0 else c for c in counts]
        seen.add(min(p.step(counts, rows, alias), 1))
    assert 0 in seen


def test_pages_come_back_first(cuda_lib):
    """What one sequence gives back another one gets in the same call."""
    p = Pool(3, 8, 4, 16)
    assert p.step([64, 0, 0], 64, False) == 0
    assert p.step([0, 1, 0], 64, False) == 1
    assert p.step([-40, 32, 1], 64, False) == 1
    assert p.step([-64, 33, 16], 64, False) == 0
    assert p.step([0, -33, -16], 64, True) == 0


def test_no_sequences_and_no_rows(cuda_lib):
    p = Pool(2, 2, 5, 32)
    assert p.step([0, 0], 0, False) == 0
    assert p.step([1, 0], 0, False) == -2
    empty = ops.paged_plan(p.d_table[:0], p.d_lengths[:0], p.d_lengths[:0], p.d_free, p.d_count, 32, 5)
    assert empty.starts.tolist() == [0] and empty.positions.tolist() == [-1] * 5 and int(empty.status) == 0


def test_states_that_are_none(cuda_lib):
    i32 = dict(dtype=torch.int32, device="cuda")
    p = Pool(2, 2, 5, 16)
    one = torch.tensor([1, 0], **i32)
    for lengths, counts in (([-1, 0], [1, 0]), ([33, 0], [-33, 0]), ([0, 0], [2 ** 31 - 1, 0]), ([3, 3], [-4, 0]), ([0, 0], [-2 ** 31, 0])):
        got = ops.paged_plan(p.d_table, torch.tensor(lengths, **i32), torch.tensor(counts, **i32), p.d_free, p.d_count, 16, 40)
        assert int(got.status) == -1 and got.lengths.tolist() == lengths and got.starts.tolist() == [0, 0, 0] and (got.slots == -1).all()
    assert int(ops.paged_plan(p.d_table, p.d_lengths, one, p.d_free, p.d_count, 16, 40, max_tokens=20).status) == 0
    assert int(ops.paged_plan(p.d_table, p.d_lengths, 21 * one, p.d_free, p.d_count, 16, 40, max_tokens=20).status) == -1
    for count in (-1, 6):
        assert int(ops.paged_plan(p.d_table, p.d_lengths, one, p.d_free, torch.tensor([count], **i32), 16, 40).status) == -3


def test_many_sequences_many_rows(cuda_lib):
    p = Pool(8192, 2, 16384, 16, seed=4)
    counts = p.rng.integers(0, 33, 8192).tolist()
    assert p.step(counts, 8192 * 32, False) == 0
    assert p.step((-np.array(counts) // 2).tolist(), 8192, True) == 0


def test_a_captured_call(cuda_lib):
    p = Pool(5, 6, 30, 16, seed=5)
    counts = torch.tensor([1, 1, 0, 17, 3], dtype=torch.int32, device="cuda")
    out = ops.paged_plan_buffers(5, 64, "cuda")._replace(lengths=p.d_lengths, free_count=p.d_count)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.paged_plan(p.d_table, p.d_lengths, counts, p.d_free, p.d_count, 16, 64, out=out)
    for _ in range(4):
        graph.replay()
        status, starts, positions, slots = p.want(counts.tolist(), 64)
        assert int(out.status) == status == 0 and out.lengths.tolist() == p.lengths and int(out.free_count) == len(p.free)
        assert np.array_equal(out.slots.cpu().numpy(), slots) and np.array_equal(out.positions.cpu().numpy(), positions)


def test_refusals(cuda_lib):
    p = Pool(3, 4, 9, 16)
    n = torch.zeros(3, dtype=torch.int32, device="cuda")
    good = dict(page_table=p.d_table, lengths=p.d_lengths, counts=n, free_pages=p.d_free, free_count=p.d_count, page_size=16, rows=4)
    ops.paged_plan(**good)
    for bad in (dict(page_table=p.d_table.long()), dict(lengths=n[:2]), dict(counts=n.float()), dict(free_count=n), dict(free_pages=p.d_free.long()),
                dict(free_pages=p.d_table), dict(rows=-1), dict(counts=n.cpu()), dict(page_table=p.d_table.t()),
                dict(out=ops.paged_plan_buffers(3, 5, "cuda")), dict(out=ops.paged_plan_buffers(2, 4, "cuda"))):
        with pytest.raises(ValueError):
            ops.paged_plan(**{**good, **bad})
    for bad in (dict(page_size=17), dict(page_table=torch.zeros((8193, 4), dtype=torch.int32, device="cuda"), lengths=torch.zeros(8193, dtype=torch.int32, device="cuda"),
                                         counts=torch.zeros(8193, dtype=torch.int32, device="cuda")), dict(max_tokens=-1)):
        with pytest.raises(ops.B200Error):
            ops.paged_plan(**{**good, **bad})
