"""Page tables with entries that are no pages (negative: the caller took some out: a window that
moved on, a prefix put elsewhere): lmx_kv8_trim gives back the others alone, so that no
later sequence is granted a page that is none."""
import random

import pytest
import torch

from lutmac_amd import kv8

pytestmark = pytest.mark.gpu
PAGE = 64


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


@pytest.mark.parametrize("n,most,share", [(1, 1, 1.0), (3, 2, 0.5), (5, 2, 0.3), (40, 20, 0.4), (70, 20, 0.05), (3, 700, 0.5), (2, 300, 1.0), (1100, 1, 0.5),
                                          (1300, 9, 0.3), (2500, 3, 0.01), (9, 200, 0.0)])
def test_holes(cuda, n, most, share):
    rng = random.Random(n + most)
    pages = n * most + 5
    held = kv8.KvPages.empty(n, most + 2, pages)
    held.free.copy_(torch.randperm(pages, generator=torch.Generator().manual_seed(n)))
    lengths = [rng.randint(0, most * PAGE) for _ in range(n)]
    held.extend(i32(lengths), torch.zeros(n * most * PAGE, dtype=torch.int32, device="cuda"))
    assert held.lengths.tolist() == lengths
    table, free = held.pages.tolist(), held.free.tolist()[: int(held.n_free)]
    for s in range(n):
        for j in range(-(-lengths[s] // PAGE)):
            if rng.random() < share:
                table[s][j] = rng.choice([-1, -1, -5, -2 ** 31])
    held.pages.copy_(i32(table))
    drop = [rng.choice([0, lengths[s], rng.randint(0, lengths[s])]) for s in range(n)]
    gone = []
    for s in range(n):
        a, b = -(-(lengths[s] - drop[s]) // PAGE), -(-lengths[s] // PAGE)
        gone += [p for p in table[s][a:b] if p >= 0]
        table[s][a:b] = [-1] * (b - a)
    held.trim(i32(drop))
    free += gone[::-1]
    assert int(held.n_free) == len(free) and held.free[: len(free)].tolist() == free
    assert held.pages.tolist() == table and held.lengths.tolist() == [a - b for a, b in zip(lengths, drop)]
    # whoever is granted pages gets real ones, each once
    before = held.n_free.clone()
    new = [rng.randint(1, most * PAGE) for _ in range(n)]
    rows = sum(new)
    slots = torch.full((rows,), -7, dtype=torch.int64, device="cuda")
    held.trim(held.lengths)
    assert int(held.n_free) >= int(before)
    offsets, granted, _, _ = held.extend(i32(new), torch.zeros(rows, dtype=torch.int32, device="cuda"), slots)
    assert (slots[: int(offsets[-1])] >= 0).all()
    mine = held.pages[held.pages >= 0]
    assert mine.unique().numel() == mine.numel() == sum(-(-g // PAGE) for g in granted.tolist())


@pytest.mark.parametrize("first", [1, 1000, 2 ** 31 - 41])
def test_pages_of_other_numbers(cuda, first):
    """A stack of pages that do not begin at 0 (a part of a cache, one without its page 0)."""
    held = kv8.KvPages.empty(5, 4, 40)
    held.free.add_(first)
    was = held.free.clone()
    lengths = [200, 1, 64, 0, 256]
    held.extend(i32(lengths), torch.zeros(1000, dtype=torch.int32, device="cuda"))
    assert held.pages[0].tolist() == list(range(first, first + 4))
    held.trim(i32(lengths))
    assert int(held.n_free) == 40 and torch.equal(held.free, was)
    held.extend(i32(lengths), torch.zeros(1000, dtype=torch.int32, device="cuda"))
    held.pages[0, 1] = -1
    held.trim(i32(lengths))
    assert int(held.n_free) == 39 and held.free[:39].tolist() == [p for p in was.tolist() if p != first + 1]


def test_replays(cuda):
    """A captured call, with holes in some replays and none in others."""
    n, most = 30, 4
    held = kv8.KvPages.empty(n, most, n * most)
    new, drop, positions = i32([0] * n), i32([0] * n), torch.zeros(n * most * PAGE, dtype=torch.int32, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held.trim(drop)
    lost = 0
    for i in range(4):
        held.extend(i32([PAGE * 3 - 5] * n), positions)
        if i % 2:
            held.pages[i, 1] = -1
            lost += 1
        drop.fill_(PAGE * 3 - 5)
        graph.replay()
        torch.cuda.synchronize()
        free = held.free[: int(held.n_free)]
        assert free.numel() == n * most - lost and free.unique().numel() == free.numel() and (held.pages == -1).all()
