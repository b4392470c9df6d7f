"""Attention over the paged 8-bit cache (lutmac_kv8.h) where the bound of
kv8_bounds.py says more than that of kv8_reference.py: rows whose weight lies in a
few tokens, queries with far channels, and values that are not finite beside finite
ones."""
import numpy as np
import pytest
import torch

import kv8_bounds
from test_gpu_kv8 import TYPES, Setup, f64

pytestmark = pytest.mark.gpu


def check(s, q=None, ref=None):
    """The attention of a Setup's rows, held to the bound."""
    q = s.q if q is None else q
    out = s.cache.attend(q, *s.where)
    want, most = kv8_bounds.attend(ref or s.reference(), f64(q), s.offsets, s.lengths, s.pages, s.hd ** -0.5, s.dtype)
    n = int(s.offsets[-1])
    got, want, most = f64(out)[:n], want[:n], most[:n]
    nan = np.isnan(want)
    np.testing.assert_array_equal(np.isnan(got), nan)
    over = (np.abs(got - want) / np.maximum(most, 1e-300))[~nan]   # (rows that see nothing: 0 of 0)
    assert over.size == 0 or over.max() <= 1, f"{over.max():.3g} times the bound, off by {np.abs(got - want)[~nan].max():.3g}"
    return got, nan


def peaked(dtype, hd, group, n, share, others, zeros, new=2, kv=2, seed=40):
    """Sequence 0: a first token with about `share` of each row's weight before n others
    of scores of spread 0.5 and values around 1, its page's values zero or not; beside
    it sequences of `others` tokens each, none before."""
    s = Setup(dtype, hd, kv, group, [new] + others, [n] + [0] * len(others), seed=seed, behind=0)
    g = torch.Generator().manual_seed(seed)
    q = torch.randint(-2, 3, s.q.shape, generator=g).float()   # (whole numbers: exact in any fixed point)
    q[..., 5] = 4
    s.q.copy_(q)
    c, first = s.cache, int(s.pages[0, 0])
    c.k[..., 5] = 0
    c.k_scale.fill_(0.5 / (2 ** 0.5 * 40))   # spread of scores: codes of 40, queries of sqrt 2, hd ** 0.5 cancels
    c.v.copy_((torch.randn(c.v.shape, generator=g) * 30 + 40).round().clamp(-127, 127))
    c.v_scale.fill_(0.025)
    c.k[first, :, :16] = 0
    c.k[first, :, 0, 5] = 127
    c.k_scale[first, :, 0] = (np.log(share / (1 - share) * n) + 0.125) / (4 * 127 * hd ** -0.5)
    if zeros:
        c.v[first] = 0
    return s


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("hd,group", [(64, 4), (128, 2)])
@pytest.mark.parametrize("n,share", [(300, 0.9), (4000, 0.5), (4000, 0.9), (30000, 0.5), (30000, 0.8), (30000, 0.9)])
@pytest.mark.parametrize("one_part", [True, False])
@pytest.mark.parametrize("zeros", [True, False])
def test_tail_behind_a_heavy_first_token(cuda, dtype, hd, group, n, share, one_part, zeros):
    """(Beside 199 sequences of one token a row's pages are not split.)"""
    check(peaked(dtype, hd, group, n, share, [1] * 199 if one_part else [], zeros))


PROMPTS = [64] * 15   # sequences beside the first that bring a call to the kernel of prompts


@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("n,share", [(300, 0.9), (3000, 0.5), (3000, 0.9)])
@pytest.mark.parametrize("zeros", [True, False])
def test_tail_behind_a_heavy_first_token_in_prompts(cuda, dtype, hd, n, share, zeros):
    """Rows enough for the kernel of prompts, in one part and several (of long tables)."""
    s = peaked(dtype, hd, 2, n, share, PROMPTS, zeros, new=70, kv=8)
    assert kv8_bounds.tiled(dtype, len(s.q), 16, 2, 8)
    check(s)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("hd,group", [(64, 3), (128, 1)])
@pytest.mark.parametrize("loud", [60, 700])
def test_queries_with_a_far_channel(cuda, dtype, hd, group, loud):
    """One channel far louder than the others, which decide where the weight goes (its
    keys are zero): they keep the bits that their type holds, in steps and in prompts."""
    for new, old, kv in (([1, 2], [40, 300], 2), ([70, 66], [0, 200], 2), ([100] * 19, [0, 200] + [5] * 17, 8)):
        s = Setup(dtype, hd, kv, group, new, old, seed=50 + loud, behind=0)
        s.q[..., 17] = loud
        s.cache.k[..., 17] = 0
        check(s)


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("hd,group", [(64, 2), (128, 4), (128, 1)])
@pytest.mark.parametrize("new,old,bad", [(8, 12, 5), (3, 14, 2), (1, 63, 0), (10, 60, 4), (100, 30, 50)])
def test_value_not_finite_beside_rows_before_it(cuda, dtype, hd, group, new, old, bad):
    """A tile whose later rows see a block with a value that is not finite, its earlier
    ones not; the places behind the last row hold the codes of whoever had the page
    before."""
    for value in (float("nan"), float("inf")):
        others = [1] if new < 100 or value == value else [101] * 19   # (once with the kernel of prompts)
        s = Setup(dtype, hd, 2 if len(others) == 1 else 8, group, [new] + others, [old] + [5] * len(others), seed=20 + bad, behind=0)
        s.v[bad, 0, 7] = value
        ref, q = s.check_append()
        _, nan = check(s, q, ref)
        sees = old + np.arange(new) >= (old + bad) // 16 * 16   # (rows from the block's first token on)
        assert (nan[:new, :group] == sees[:, None, None]).all() and not nan[:, group:].any() and not nan[new:].any()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128])
def test_value_not_finite_of_little_weight(cuda, dtype, hd):
    """A block that is not finite gives NaN to the rows that see it though their weights
    of it are zero."""
    s = Setup(dtype, hd, 1, 2, [1, 4], [200, 70], seed=31, behind=0)
    s.q.copy_(torch.ones_like(s.q))
    page = int(s.pages[0, 1])
    s.cache.k_scale[page, 0, 2] = 1.0
    s.cache.k[page, 0, 32:48] = -127   # scores some 1000 below the others
    s.cache.v_scale[page, 0, 2] = float("nan")
    _, nan = check(s)
    assert nan[0].all() and not nan[1:].any()
