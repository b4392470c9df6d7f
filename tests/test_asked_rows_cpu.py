"""Rows of a step among those laid out by what was asked for (kv8.asked_rows)."""
import random

import pytest
import torch

from lutmac_amd import kv8


@pytest.mark.parametrize("n", [0, 1, 2, 9, 200])
def test_asked_rows(n):
    rng = random.Random(n)
    for _ in range(20):
        new = [rng.choice([0, 0, 1, 3, 7]) for _ in range(n)]
        granted = [m if rng.random() < 0.6 else 0 for m in new]
        asked, offsets, want = [3], [0], []   # (the layout may begin anywhere)
        for m, g in zip(new, granted):
            want += range(asked[-1], asked[-1] + g)
            asked.append(asked[-1] + m)
            offsets.append(offsets[-1] + g)
        rows = len(want) + rng.choice([0, 1, 10])
        got = kv8.asked_rows(torch.tensor(asked[:-1], dtype=torch.int32), torch.tensor(offsets, dtype=torch.int32), rows)
        assert got.dtype == torch.int64 and got.tolist() == want + [0] * (rows - len(want))
