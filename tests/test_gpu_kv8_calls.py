"""Calls of the paged 8-bit cache that its documents allow: rows before the first
sequence, the widest groups, shared pages, steps of several streams at once."""
import numpy as np
import pytest
import torch

from test_gpu_kv8 import TYPES, Setup, f64
from test_gpu_kv8_peaked import check

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("kv,group", [(1, 64), (3, 7), (5, 1), (1, 33)])
@pytest.mark.parametrize("new,old", [([1, 1], [0, 130]), ([5, 0, 66], [70, 3, 15])])
def test_groups(cuda, dtype, kv, group, new, old):
    s = Setup(dtype, 64, kv, group, new, old, seed=80 + group)
    ref, q = s.check_append()
    check(s, q, ref)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("new,old", [([3, 1], [20, 64]), ([200, 100, 17], [0, 300, 63])])
def test_rows_before_the_first_sequence(cuda, dtype, new, old):
    """Rows below offsets[0] belong to no sequence, as those behind the last do."""
    for first in (1, 65, 300):
        s = Setup(dtype, 128, 2, 4, [first] + new, [0] + old, seed=81)
        # the first sequence is left out: its rows stay, its page table row goes
        s.offsets, s.lengths, s.pages = s.offsets[1:].copy(), s.lengths[1:].copy(), s.pages[1:].copy()
        s.where = tuple(torch.from_numpy(a).cuda() for a in (s.offsets, s.lengths, s.pages))
        ref, q = s.check_append()
        out = torch.full_like(q, 7.0)
        s.cache.attend(q, *s.where, out=out)
        assert (out[:first] == 7.0).all() and (out[int(s.offsets[-1]):] == 7.0).all()
        got = out.clone()
        want = ref.attend(f64(q), s.offsets, s.lengths, s.pages, 128 ** -0.5, dtype)
        n = int(s.offsets[-1])
        assert (np.abs(f64(got)[first:n] - want[0][first:n]) <= want[1][first:n]).all()


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_shared_pages(cuda, dtype):
    """Sequences that share their first pages, and a page that one has twice."""
    s = Setup(dtype, 64, 2, 2, [1, 4, 1], [300, 250, 200], seed=82, behind=0)
    s.pages[1, :3] = s.pages[0, :3]
    s.pages[2, :2] = s.pages[0, 1]
    s.where[2].copy_(torch.from_numpy(s.pages))
    check(s)
    ref, q = s.check_append()   # (new tokens go to pages of one sequence each)
    check(s, q, ref)


def test_calls_at_once(cuda):
    """Calls on several streams at a time, with outputs and workspaces of their own, on
    one cache that none writes."""
    s = [Setup("bfloat16", 128, 4, 4, new, old, seed=83, width=40) for new, old in
         (([1] * 9, [2000] * 9), ([300, 5], [0, 900]), ([1], [2500]), ([7] * 4, [50] * 4))]
    alone = [x.cache.attend(x.q, *x.where) for x in s]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in s]
    outs = []
    for _ in range(20):
        outs.append([x.cache.attend(x.q, *x.where, stream=t) for x, t in zip(s, streams)])
    torch.cuda.synchronize()
    for row in outs:
        for x, o, want in zip(s, row, alone):
            n = int(x.offsets[-1])
            assert torch.equal(o[:n], want[:n])
