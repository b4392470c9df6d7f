"""The kernel of prompts (lmx_kv8_prompt.hip): calls large enough for it, with whole
and part tiles, prefixes, absent pages, sequences without rows, rows before position
0 and scales that are not seen, within the bound of kv8_bounds.py."""
import numpy as np
import pytest
import torch

import kv8_bounds
from test_gpu_kv8 import Setup, f64
from test_gpu_kv8_peaked import check

pytestmark = pytest.mark.gpu
TYPES = ["float16", "bfloat16"]
RAGGED = ([97, 0, 260, 33, 1, 16, 64, 129], [64, 10, 31, 700, 0, 63, 1000, 1])


def prompts(dtype, hd, group, new=RAGGED[0], old=RAGGED[1], kv=8, **kw):
    s = Setup(dtype, hd, kv, group, new, old, **kw)
    assert kv8_bounds.tiled(dtype, len(s.q), len(new), group, kv)
    return s


def upload(s):
    s.where = tuple(torch.from_numpy(a).cuda() for a in (s.offsets, s.lengths, s.pages))


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd,group", [(64, 4), (128, 5), (128, 4)])
@pytest.mark.parametrize("width", [None, 40])
def test_ragged(cuda, dtype, hd, group, width):
    """Tables to spare split a tile's pages over workgroups; some rows lie behind the
    last sequence; then some pages are absent and a block's values are zero."""
    s = prompts(dtype, hd, group, seed=60 + hd + group, width=width, behind=3)
    check(s)
    s.cache.k_scale.mul_(4)   # scores that outgrow their first reference
    s.pages[0, 1] = -1
    s.pages[3, 0] = s.cache.n_pages
    s.pages[6, 3:5] = -9
    s.cache.v_scale[int(s.pages[0, 0]), 0, 2] = 0.0
    upload(s)
    check(s)


@pytest.mark.parametrize("dtype", TYPES)
def test_rows_behind_the_last_sequence_stay(cuda, dtype):
    s = prompts(dtype, 64, 4, seed=70, behind=5)
    out = torch.full_like(s.q, 7.0)
    s.cache.attend(s.q, *s.where, out=out)
    n = int(s.offsets[-1])
    assert (out[n:] == 7.0).all() and not (out[:n] == 7.0).all()
    q = s.q.clone()   # (out may be q)
    s.cache.attend(q, *s.where, out=q)
    assert torch.equal(q[:n], out[:n])


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("hd", [64, 128])
def test_places_outside(cuda, dtype, hd):
    """Positions before the first token, and past the table of pages."""
    s = prompts(dtype, hd, 4, [200] * 6, [0, 0, 100, 300, 64, 0], seed=71, behind=0, width=4)
    s.lengths[0], s.lengths[5] = 90, 0   # (110 and all of the 200 rows before position 0)
    upload(s)
    got, nan = check(s)
    assert (got[:110] == 0).all() and (got[1000:] == 0).all() and not nan.any()


@pytest.mark.parametrize("dtype", TYPES)
def test_unseen_scales(cuda, dtype):
    """Scales behind a sequence's end may hold anything; a query that is not finite
    gives NaN, its neighbours not."""
    s = prompts(dtype, 128, 4, [200] * 6, [0, 30, 100, 300, 64, 1], seed=72, behind=0)
    for i, n in enumerate(s.lengths):
        page, block = int(s.pages[i, (n - 1) // 64]), (int(n) - 1) % 64 // 16
        s.cache.v_scale[page, :, block + 1:] = float("nan") if i % 2 else float("inf")
        s.cache.k_scale[page, :, block + 1:] = float("inf") if i % 2 else float("nan")
    s.q[3, 5, 100], s.q[777, 31, 0] = float("inf"), float("nan")
    _, nan = check(s)
    assert nan[3, 5].all() and nan[777, 31].all() and nan.sum() == 2 * 128


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rising", [True, False])
def test_reference_rises_and_falls(cuda, dtype, rising):
    """Scores that grow page by page by more than a weight's range, or fall."""
    s = prompts(dtype, 128, 2, [180] * 6, [500] * 6, seed=73, behind=0)
    rise = torch.linspace(0.001, 0.4, s.pages.shape[1] * 4).view(-1, 1, 4).cuda()
    for i in range(6):
        s.cache.k_scale[torch.from_numpy(s.pages[i]).long().cuda()] = rise if rising else rise.flip(0, 2)
    check(s)


@pytest.mark.parametrize("dtype", TYPES)
def test_value_scales_far_apart(cuda, dtype):
    s = prompts(dtype, 64, 4, [130] * 8, [200] * 8, seed=74, behind=0)
    n = s.cache.v_scale.numel()
    for lo, hi in ((-30, 4), (-99, -60)):   # (outputs stay in the types' range)
        at = torch.randperm(n, generator=torch.Generator().manual_seed(hi))
        s.cache.v_scale.view(-1).copy_(2.0 ** torch.linspace(lo, hi, n)[at].cuda())
        if dtype == "bfloat16" or hi > 0:
            check(s)


@pytest.mark.parametrize("dtype", TYPES)
def test_each_kernel_and_repeats(cuda, dtype):
    """A sequence in a call of its own goes to the other kernel: both within their
    bounds of the same values; the same call again gives the same bits."""
    s = prompts(dtype, 128, 4, seed=75, behind=0)
    out = s.cache.attend(s.q, *s.where)
    for _ in range(5):
        assert torch.equal(s.cache.attend(s.q, *s.where), out)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device="cuda")
    for i in (0, 3):
        a, b = int(s.offsets[i]), int(s.offsets[i + 1])
        assert not kv8_bounds.tiled(dtype, b - a, 1, 4, 8)
        q, where = s.q[a:b], ([0, b - a], [int(s.lengths[i])], s.pages[i:i + 1])
        alone = s.cache.attend(q, i32(where[0]), i32(where[1]), s.where[2][i:i + 1].contiguous())
        want, most = kv8_bounds.attend(s.reference(), f64(q), *where, 128 ** -0.5, dtype)
        assert (np.abs(f64(alone) - want) <= most).all()


def test_graph_follows_lengths(cuda):
    """A captured call of prompts replays with the lengths that the tensors hold then."""
    s = prompts("bfloat16", 128, 4, [150] * 8, [100] * 8, seed=76, behind=0, width=8)
    work = torch.empty(max(1, s.cache.attend_workspace(torch.bfloat16, len(s.q), s.heads, 8, 8)), dtype=torch.uint8, device="cuda")
    out = torch.empty_like(s.q)
    s.cache.attend(s.q, *s.where, out=out, workspace=work)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        s.cache.attend(s.q, *s.where, out=out, workspace=work)
    for step in range(4):
        s.where[1].sub_(20 * (step > 0))
        s.lengths -= 20 * (step > 0)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, s.cache.attend(s.q, *s.where))
    check(s)
