"""Rotation by tables whose pairs are not of length one, and positions far into a table."""
import pytest
import torch

from lutmac_amd import kv8
from test_gpu_rotary import TYPES, check, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("interleaved", [False, True])
def test_scaled_table(cuda, dtype, interleaved):
    """inverse is the transpose: <g, R x> = <R^T g, x>; there and back is the square of the
    table's factor."""
    q, k, at, _ = make(dtype, 30, 4, 2, 64, 48, 5000)
    rope = kv8.rope_table(5000, 48, scaling={"type": "yarn", "factor": 16.0, "original": 512})
    times = float(rope[0, 0, 0])
    assert times > 1.2
    y, _ = kv8.rotate(q, k, at, rope, interleaved=interleaved)
    check(q, y, rope, at, interleaved, False)
    g = torch.randn_like(q)
    grad, _ = kv8.rotate(g, None, at, rope, interleaved=interleaved, inverse=True)
    check(g, grad, rope, at, interleaved, True)
    if dtype == torch.float32:
        # (both sides off by at most 2^-22 of their factors' sizes)
        assert abs((g.double() * y.double()).sum() - (grad.double() * q.double()).sum()) < 2.0 ** -21 * times * g.double().norm() * q.double().norm()
        back, _ = kv8.rotate(y, None, at, rope, interleaved=interleaved, inverse=True)
        # (|x| below 6, pairs below 8.5; each way off by 2^-22 of that times the factor)
        assert (back[..., :48].double() - times ** 2 * q[..., :48].double()).abs().max() < 2 * 2.0 ** -22 * 8.5 * times ** 2
        assert torch.equal(back[..., 48:], q[..., 48:])


@pytest.mark.parametrize("interleaved", [False, True])
def test_captured_at_far_positions(cuda, interleaved):
    """Positions near 2^22 in a table of 2 GiB, in the first replay and in the last."""
    n = 1 << 22
    q, k, at, _ = make(torch.bfloat16, 64, 4, 2, 128, 128, 10)
    rope = torch.randn(n, 64, 2, device="cuda")
    a, b = torch.empty_like(q), torch.empty_like(k)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kv8.rotate(q, k, at, rope, interleaved=interleaved, q_out=a, k_out=b)
    for low in (n - 1000, 0, n - 64):
        at.copy_(torch.randint(low, n, (64,), dtype=torch.int32))
        at[5] = n - 1
        graph.replay()
        torch.cuda.synchronize()
        check(q, a, rope, at, interleaved, False)
        check(k, b, rope, at, interleaved, False)
