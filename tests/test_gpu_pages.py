"""The page table on the device (lmx_kv8_extend, lmx_kv8_trim) against a plain
restatement in Python: whole numbers, all equal."""
import random

import numpy as np
import pytest
import torch

from lutmac_amd import kv8

pytestmark = pytest.mark.gpu
PAGE = 64


class Plain:
    def __init__(self, pages, lengths, free, n_free):
        self.pages, self.lengths, self.free, self.n_free = pages.copy(), lengths.copy(), free.copy(), int(n_free)

    def extend(self, new, positions, slots):
        offsets, granted, asked, needed, taken = [0], [], 0, 0, 0
        for s, n in enumerate(new):
            n, old = max(int(n), 0), int(self.lengths[s])
            if n == 0 or old + n > min(self.pages.shape[1] * PAGE, 2 ** 31 - 1):
                granted.append(0)
                offsets.append(offsets[-1])
                continue
            need = -(-(old + n) // PAGE) - -(-old // PAGE)
            asked, needed = asked + n, needed + need
            if asked > len(positions) or (need and needed > self.n_free):
                n = 0
            else:
                for j in range(need):
                    self.pages[s, -(-old // PAGE) + j] = self.free[self.n_free - 1 - taken]
                    taken += 1
                for j in range(n):
                    r, p = offsets[-1] + j, old + j
                    positions[r] = p
                    if slots is not None:
                        page = int(self.pages[s, p // PAGE])
                        slots[r] = -1 if page < 0 else page * PAGE + p % PAGE
                self.lengths[s] += n
            granted.append(n)
            offsets.append(offsets[-1] + n)
        self.n_free -= taken
        return offsets, granted

    def trim(self, drop):
        gone = []
        for s, d in enumerate(drop):
            old = int(self.lengths[s])
            keep = old - min(max(int(d), 0), old)
            a, b = (min(-(-n // PAGE), self.pages.shape[1]) for n in (keep, old))
            gone += [int(p) for p in self.pages[s, a:b]]
            self.pages[s, a:b] = -1
            self.lengths[s] = keep
        for j, p in enumerate(gone):
            at = self.n_free + len(gone) - 1 - j
            if at < len(self.free):
                self.free[at] = p
        self.n_free = min(self.n_free + len(gone), len(self.free))


class Both:
    def __init__(self, n_seqs, max_pages, n_pages, rows, seed=0):
        self.held = kv8.KvPages.empty(n_seqs, max_pages, n_pages)
        if n_pages:
            self.held.free.copy_(torch.randperm(n_pages, generator=torch.Generator().manual_seed(seed)))
        self.plain = Plain(self.held.pages.cpu().numpy(), self.held.lengths.cpu().numpy(), self.held.free.cpu().numpy(), n_pages)
        self.rows = rows

    def same(self):
        assert int(self.held.n_free) == self.plain.n_free
        assert np.array_equal(self.held.lengths.cpu().numpy(), self.plain.lengths)
        assert np.array_equal(self.held.pages.cpu().numpy(), self.plain.pages)
        n = self.plain.n_free
        assert np.array_equal(self.held.free.cpu().numpy()[:n], self.plain.free[:n])

    def extend(self, new, with_slots=True):
        positions = torch.full((self.rows,), -7, dtype=torch.int32, device="cuda")
        slots = torch.full((self.rows,), -7, dtype=torch.int64, device="cuda") if with_slots else None
        want_p, want_s = np.full(self.rows, -7, np.int32), np.full(self.rows, -7, np.int64)
        got = self.held.extend(torch.tensor(new, dtype=torch.int32, device="cuda"), positions, slots)
        offsets, granted = self.plain.extend(new, want_p, want_s if with_slots else None)
        assert got[0].tolist() == offsets and got[1].tolist() == granted
        assert np.array_equal(positions.cpu().numpy(), want_p)
        if with_slots:
            assert np.array_equal(slots.cpu().numpy(), want_s)
        self.same()
        return granted

    def trim(self, drop):
        self.held.trim(torch.tensor(drop, dtype=torch.int32, device="cuda"))
        self.plain.trim(drop)
        self.same()


@pytest.mark.parametrize("n,most,rows", [(1, 1, 8), (1, 700, 4096), (3, 200, 600), (64, 5, 320), (1000, 3, 2500), (1024, 2, 3000), (1025, 70, 30000),
                                         (2500, 9, 20000), (40, 9000, 200000), (5000, 1, 5000), (9000, 9, 30000)])
def test_steps(cuda, n, most, rows):
    """Some steps of growing and shrinking; tight rows and pages leave some out."""
    rng = random.Random(n + most)
    b = Both(n, 2 * (most // PAGE) + 3, max(2, n * most // PAGE + n // 2), rows, seed=n)
    for step in range(4):
        granted = b.extend([rng.choice([0, 1, rng.randint(0, most), rng.randint(0, most), -3]) for _ in range(n)], step % 2 == 0)
        before = [t.clone() for t in (b.held.pages, b.held.lengths, b.held.free, b.held.n_free)]
        again = b.extend([rng.randint(0, most) for _ in range(n)])
        b.trim(again)   # all of it back: as it was
        for t, was in zip((b.held.pages, b.held.lengths), before):
            assert torch.equal(t, was)
        k = int(before[3])
        assert int(b.held.n_free) == k and torch.equal(b.held.free[:k], before[2][:k])
        b.trim([rng.choice([0, rng.randint(0, g + 1), g, 10 ** 9 if rng.random() < 0.2 else 0, -5]) for g in granted])
    b.trim(b.held.lengths.tolist())
    assert int(b.held.n_free) == b.held.free.numel() and (b.held.pages == -1).all()


def test_borders(cuda):
    """Lengths at the ends of pages, of the table and of the rows."""
    b = Both(6, 3, 20, 400)
    b.extend([64, 63, 65, 128, 1, 0])
    b.extend([1, 1, 63, 64, 191, 192])      # (the last two: just the whole table row)
    b.extend([0, 128, 64, 1, 0, 1])         # just full; past the end of the table
    b.trim([1, 0, 1, 64, 128, 192])
    b.extend([1, 1, 1, 1, 1, 1])
    # rows: just enough, one too many
    b = Both(3, 10, 40, 100)
    assert b.extend([50, 50, 1]) == [50, 50, 0]
    assert b.extend([50, 51, 20]) == [50, 0, 0]
    # pages: those that need none go on
    b = Both(4, 10, 2, 500)
    assert b.extend([10, 10, 10, 10]) == [10, 10, 0, 0]
    assert b.extend([20, 60, 5, 20]) == [20, 0, 0, 0]
    assert b.extend([20, 54, 5, 0]) == [20, 54, 0, 0]


def test_odd_states(cuda):
    """Counts that no sequence can have: nothing outside the arrays is touched."""
    big = 2 ** 31 - 1
    b = Both(5, 4, 6, 64)
    b.extend([big, -big, 3, big, 1])
    b.trim([-1, big, -big, 0, big])
    held = b.held
    held.n_free.fill_(10 ** 9)      # more than there are: taken as all
    b.plain.n_free = 6
    b.extend([1, 1, 1, 1, 1])
    held.n_free.fill_(-4)
    b.plain.n_free = 0
    b.extend([1, 1, 1, 1, 64])
    held.lengths.copy_(torch.tensor([-5, big, 500, 0, 64]))   # longer than the table
    b.plain.lengths[:] = [0, big, 500, 0, 64]
    granted = held.extend(torch.tensor([0, 1, 1, 0, 0], dtype=torch.int32, device="cuda"),
                          torch.zeros(64, dtype=torch.int32, device="cuda"))[1]
    assert granted.tolist() == [0] * 5
    held.trim(torch.tensor([0, big, big, big, big], dtype=torch.int32, device="cuda"))
    b.plain.trim([0, big, big, big, big])
    assert np.array_equal(held.pages.cpu().numpy(), b.plain.pages) and int(held.n_free) == b.plain.n_free


@pytest.mark.parametrize("n,max_pages,pages,rows", [(0, 4, 5, 10), (3, 0, 5, 10), (3, 4, 0, 10), (3, 4, 5, 0)])
def test_nothing_to_give(cuda, n, max_pages, pages, rows):
    b = Both(n, max_pages, pages, rows)
    assert sum(b.extend([1] * n)) == (3 if n and max_pages and pages and rows else 0)
    b.trim([1] * n)


def test_arguments_that_are_one(cuda):
    """Sequences that end drop their own lengths; counts asked and granted in one tensor."""
    for n in (5, 3000):
        b = Both(n, 4, 2 * n, 2 * n)
        new = torch.full((n,), 3, dtype=torch.int32, device="cuda")
        positions = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
        _, granted, _, _ = b.held.extend(new, positions, granted=new)
        assert granted is new and new.tolist() == [3 if 3 * (s + 1) <= 2 * n else 0 for s in range(n)]
        b.held.trim(b.held.lengths)
        assert not b.held.lengths.any() and int(b.held.n_free) == 2 * n and (b.held.pages == -1).all()
        assert torch.equal(b.held.free.sort()[0].cpu(), torch.arange(2 * n, dtype=torch.int32))


def test_one_long_sequence(cuda):
    """A prompt of many pages beside single tokens; slots past 2^31."""
    b = Both(3, 6000, 7000, 300000)
    b.extend([5, 299990, 1])
    b.trim([1, 200000, 0])
    held = b.held
    held.pages[:1, 0] = 2 ** 31 - 2   # (a table that the caller fills may say anything)
    positions, slots = torch.zeros(300000, dtype=torch.int32, device="cuda"), torch.zeros(300000, dtype=torch.int64, device="cuda")
    held.extend(torch.tensor([2, 0, 0], dtype=torch.int32, device="cuda"), positions, slots)
    assert slots[:2].tolist() == [(2 ** 31 - 2) * 64 + 4, (2 ** 31 - 2) * 64 + 5]


def test_captured(cuda):
    """A captured step replayed: every replay goes on from the state that it finds."""
    b = Both(70, 50, 400, 300)
    new = torch.zeros(70, dtype=torch.int32, device="cuda")
    drop, offsets, granted = torch.zeros_like(new), torch.zeros(71, dtype=torch.int32, device="cuda"), torch.zeros_like(new)
    positions, slots = torch.full((300,), -7, dtype=torch.int32, device="cuda"), torch.full((300,), -7, dtype=torch.int64, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        b.held.extend(new, positions, slots, offsets=offsets, granted=granted)
        b.held.trim(drop)
    want_p, want_s = np.full(300, -7, np.int32), np.full(300, -7, np.int64)
    rng = random.Random(5)
    for _ in range(5):
        n, d = [rng.randint(0, 5) for _ in range(70)], [rng.randint(0, 3) for _ in range(70)]
        new.copy_(torch.tensor(n)), drop.copy_(torch.tensor(d))
        graph.replay()
        torch.cuda.synchronize()
        o, g = b.plain.extend(n, want_p, want_s)
        b.plain.trim(d)
        assert offsets.tolist() == o and granted.tolist() == g
        assert np.array_equal(positions.cpu().numpy(), want_p) and np.array_equal(slots.cpu().numpy(), want_s)
        b.same()
