"""Rotation of as many rows as a call takes."""
import pytest
import torch

from lutmac_amd import kv8
from test_gpu_rotary import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("hd,rows", [(386, 1 << 24), (386, (1 << 24) - 5), (64, (1 << 20) + 3), (2, 3 * (1 << 20))])
def test_most_rows(cuda, hd, rows):
    """2^24 rows of 193 pairs are 2^32 threads and more: some rows near the ends and near
    every 2^20th against 64 bits, in place; the others are zeros and stay."""
    rope = kv8.rope_table(1000, hd)
    x = torch.zeros(rows, 1, hd, dtype=torch.float16, device="cuda")
    at = torch.randint(0, 1000, (rows,), dtype=torch.int32, device="cuda")
    some = torch.tensor(sorted({r for m in range(0, rows + 1, 1 << 20) for r in range(m - 3, m + 3) if 0 <= r < rows} | {rows - 1}), device="cuda")
    q = torch.randn(len(some), 1, hd, device="cuda").half()
    x[some] = q
    missed = some[1]
    at[missed] = -1
    kv8.rotate(x, None, at, rope, q_out=x)
    keep = some != missed
    check(q[keep], x[some[keep]], rope, at[some[keep]], False, False)
    assert torch.equal(x[missed], q[1])
    x[some] = 0
    assert not x.any()
