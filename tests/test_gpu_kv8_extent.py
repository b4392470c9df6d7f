"""Lengths at the end of their type, and tables without pages: rows without a place
in the cache."""
import pytest
import torch

from kv8_reference import PAGE
from lutmac_amd.kv8 import KvCache8, rope_table

pytestmark = pytest.mark.gpu
LAST = 2 ** 31 - 1


def setup(length, rows, width, dtype=torch.float32, heads=12, hd=64):
    cache = KvCache8.empty(2, 2, hd)
    g = torch.Generator().manual_seed(rows)
    k, v = (torch.randn(rows, 2, hd, generator=g).to(dtype).cuda() for _ in range(2))
    q = torch.randn(rows, heads, hd, generator=g).to(dtype).cuda()
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    return cache, k, v, q, (i32([0, rows]), i32([length]), torch.zeros(1, width, dtype=torch.int32, device="cuda"))


@pytest.mark.parametrize("length", [LAST, LAST - 63, LAST - 64, LAST - 130])
@pytest.mark.parametrize("rows", [1, 3, 70, 140])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_positions_up_to_the_last(cuda, length, rows, dtype):
    """Without a rotation table queries are copied whatever their position; keys and
    values past the page table are not written."""
    cache, k, v, q, where = setup(length, rows, 2, dtype)
    out = torch.full_like(q, 7.0)
    cache.append(k, v, *where, q=q, q_out=out)
    assert torch.equal(out, q)
    assert not cache.k.any() and not cache.v.any() and not cache.k_scale.any()
    cache.k_scale.fill_(1.0), cache.v_scale.fill_(1.0), cache.v.fill_(3)
    # every row sees all 2 pages: 3, up to fp32's roundings of the weights and two sums
    assert ((cache.attend(q, *where).float() - 3.0).abs() <= 3.0 * 2.0 ** -20).all()


@pytest.mark.parametrize("length", [LAST, LAST - 63, LAST - 130, 200])
@pytest.mark.parametrize("rows", [1, 3, 70])
def test_positions_past_the_rotation_table(cuda, length, rows):
    """Rows past the rotation table are left out whole, however far."""
    cache, k, v, q, where = setup(length, rows, 2)
    out = torch.full_like(q, 7.0)
    cache.append(k, v, *where, rope=rope_table(length - rows if length == 200 else 100, 64), q=q, q_out=out)
    assert (out == 7.0).all() and not cache.k.any() and not cache.v.any() and not cache.k_scale.any()


@pytest.mark.parametrize("rows", [1, 40])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
def test_table_without_pages(cuda, rows, dtype):
    cache, k, v, q, where = setup(rows, rows, 0, dtype)
    assert torch.equal(cache.append(k, v, *where, q=q), q)
    assert not cache.k.any() and not cache.k_scale.any()
    out = torch.full_like(q, 7.0)
    assert (cache.attend(q, *where, out=out) == 0).all()


def test_page_before_the_last_position(cuda):
    """The page that ends at the last position of a long table's reach."""
    cache, k, v, q, where = setup(2 * PAGE, 5, 2)
    where[2].copy_(torch.tensor([[0, 1]]))
    cache.append(k, v, *where, q=q)
    assert cache.k[1, :, PAGE - 5:].any() and not cache.k[1, :, :PAGE - 5].any() and not cache.k[0].any()
