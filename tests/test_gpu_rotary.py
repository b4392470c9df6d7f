"""Rotation of queries and keys (lmx_rotary) against 64 bits: a product and a fused
sum round twice, 2^-24 of |a c| + |b s| each, then the result to its type."""
import math

import pytest
import torch

from lutmac_amd import kv8

pytestmark = pytest.mark.gpu
HALF_STEP = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TYPES = sorted(HALF_STEP, key=str)


def pairs(x, rd, interleaved):
    y = x[..., :rd]
    return (y[..., 0::2], y[..., 1::2]) if interleaved else y.chunk(2, -1)


def joined(a, b, interleaved):
    return torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)


def check(x, y, rope, positions, interleaved, inverse):
    rd = 2 * rope.shape[1]
    c, s = rope[positions.long()].double()[:, None].unbind(-1)
    s = -s if inverse else s
    a, b = pairs(x.double(), rd, interleaved)
    want = joined(a * c - b * s, a * s + b * c, interleaved)
    size = joined((a * c).abs() + (b * s).abs(), (a * s).abs() + (b * c).abs(), interleaved)
    most = 2 * 2.0 ** -24 * size + want.abs() * HALF_STEP[x.dtype] + (2.0 ** -25 if x.dtype == torch.float16 else 1e-44)
    assert ((y[..., :rd].double() - want).abs() <= most).all()
    assert torch.equal(y[..., rd:], x[..., rd:])


def make(dtype, rows, heads, kv, hd, rd, positions, seed=1):
    g = torch.Generator().manual_seed(seed)
    q, k = torch.randn(rows, heads, hd, generator=g).to(dtype).cuda(), torch.randn(rows, kv, hd, generator=g).to(dtype).cuda()
    at = torch.randint(0, positions, (rows,), generator=g, dtype=torch.int32).cuda()
    return q, k, at, kv8.rope_table(positions, rd)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("rows,heads,kv,hd,rd", [(1, 1, 1, 2, 2), (1, 32, 8, 64, 64), (7, 12, 2, 128, 128), (300, 5, 5, 80, 32),
                                                 (33, 3, 1, 96, 96), (5, 2, 1, 7, 6), (64, 4, 2, 256, 64), (9, 1, 1, 1024, 1022),
                                                 (2, 128, 128, 256, 256), (1000, 2, 1, 66, 34)])
def test_rotate(cuda, dtype, interleaved, rows, heads, kv, hd, rd):
    q, k, at, rope = make(dtype, rows, heads, kv, hd, rd, 5000)
    for inverse in (False, True):
        a, b = kv8.rotate(q, k, at, rope, interleaved=interleaved, inverse=inverse)
        check(q, a, rope, at, interleaved, inverse)
        check(k, b, rope, at, interleaved, inverse)
    a, b = kv8.rotate(q, None, at, rope, interleaved=interleaved)
    assert b is None
    check(q, a, rope, at, interleaved, False)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_in_place_strides_and_alignment(cuda, dtype, interleaved):
    """Rows inside a wider array (q | k | v), in place; arrays that start at an odd
    element; what lies between is left alone."""
    q, k, at, rope = make(dtype, 50, 6, 2, 64, 48, 700)
    want = kv8.rotate(q, k, at, rope, interleaved=interleaved)
    for lead in (0, 1):
        for gap in (0, 3, 128):
            width = 8 * 64 + gap
            flat = torch.full((50 * width + lead,), 7.0, dtype=dtype, device="cuda")
            rows = flat[lead:].view(50, width)
            qs, ks = rows[:, :384].unflatten(1, (6, 64)), rows[:, 384:512].unflatten(1, (2, 64))
            qs.copy_(q), ks.copy_(k)
            a, b = kv8.rotate(qs, ks, at, rope, interleaved=interleaved, q_out=qs, k_out=ks)
            assert a is qs and b is ks and torch.equal(a, want[0]) and torch.equal(b, want[1])
            assert (rows[:, 512:] == 7.0).all() and (flat[:lead] == 7.0).all()
            qs.copy_(q)
            out = torch.empty_like(q)
            kv8.rotate(qs, None, at, rope, interleaved=interleaved, q_out=out)
            assert torch.equal(out, want[0]) and torch.equal(qs, q)


def test_rows_without_a_place(cuda):
    """Rows whose position the table lacks are not written."""
    q, k, at, rope = make(torch.float32, 40, 4, 2, 64, 64, 100)
    at[3], at[7], at[8], at[39] = -1, 100, 2 ** 31 - 1, -2 ** 31
    a, b = torch.full_like(q, 7.0), torch.full_like(k, 7.0)
    kv8.rotate(q, k, at, rope, q_out=a, k_out=b)
    out = torch.zeros(40, dtype=torch.bool)
    out[[3, 7, 8, 39]] = True
    assert (a[out] == 7.0).all() and (b[out] == 7.0).all()
    check(q[~out], a[~out], rope, at[~out.cuda()], False, False)
    check(k[~out], b[~out], rope, at[~out.cuda()], False, False)


def test_inverse_is_the_gradient(cuda):
    """<g, R x> = <R^-1 g, x>, against differences too; there and back again."""
    q, k, at, rope = make(torch.float32, 20, 3, 1, 64, 32, 5000)
    for interleaved in (False, True):
        g = torch.randn_like(q)
        grad = kv8.rotate(g, None, at, rope, interleaved=interleaved, inverse=True)[0].double()
        y = kv8.rotate(q, None, at, rope, interleaved=interleaved)[0]
        assert abs(((g * y).double().sum() - (grad * q).sum()) / grad.norm() / q.norm()) < 1e-6
        d = torch.zeros_like(q)
        d[4, 1, 5] = 0.5
        z = kv8.rotate(q + d, None, at, rope, interleaved=interleaved)[0]
        # (two results each off by 2^-22 of at most 8)
        assert abs(((z - y).double() * g).sum() / 0.5 - grad[4, 1, 5]) < 2 * 64 * 8 * 2.0 ** -22 / 0.5
        back = kv8.rotate(y, None, at, rope, interleaved=interleaved, inverse=True)[0]
        assert (back - q).abs().max() < 8 * 8 * 2.0 ** -24


def test_as_append_rotates(cuda):
    """Whole heads in halves: what the cache's append does to queries, to its rounding."""
    q, k, at, rope = make(torch.float32, 30, 4, 2, 64, 64, 100)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    at = torch.arange(30, dtype=torch.int32, device="cuda") + 7
    cache = kv8.KvCache8.empty(1, 2, 64)
    mine = kv8.rotate(q, k, at, rope)[0]
    theirs = cache.append(k, k, i32([0, 30]), i32([37]), i32([[0]]), rope=rope, q=q)
    assert (mine - theirs).abs().max() <= 3 * 2.0 ** -24 * 2 * q.abs().max()


@pytest.mark.parametrize("interleaved", [False, True])
def test_far_positions_and_replays(cuda, interleaved):
    """Positions near 2^20 in a table whose offsets pass 2^31 bytes' half; a captured
    call follows its positions."""
    q, k, at, _ = make(torch.bfloat16, 64, 4, 2, 128, 128, 10)
    rope = torch.randn(1 << 22, 64, 2, device="cuda")
    at.copy_(torch.randint((1 << 22) - 1000, 1 << 22, (64,), dtype=torch.int32))
    a, b = torch.empty_like(q), torch.empty_like(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv8.rotate(q, k, at, rope, interleaved=interleaved, q_out=a, k_out=b)
    for _ in range(3):
        at.copy_(torch.randint(0, 1 << 22, (64,), dtype=torch.int32))
        graph.replay()
        torch.cuda.synchronize()
        check(q, a, rope, at, interleaved, False)
        check(k, b, rope, at, interleaved, False)
    stream = torch.cuda.Stream()
    c, _ = kv8.rotate(q, k, at, rope, interleaved=interleaved, stream=stream)
    stream.synchronize()
    assert torch.equal(c, a)
    assert kv8.rotate(q[:0], k[:0], at[:0], rope)[0].shape == (0, 4, 128) and math.isfinite(float(a.float().sum()))
