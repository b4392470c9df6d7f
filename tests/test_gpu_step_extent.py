"""The operators of a drafted step past 32 bits of offsets, and several calls at once."""
import pytest
import torch

import lutmac_amd as L
from lutmac_amd import kv8
from test_gpu_f8 import make as make_linear
from test_gpu_rotary import check as check_rotated
from test_gpu_verify import make as make_drafts

pytestmark = pytest.mark.gpu


def test_linear_output_past_32_bits(cuda):
    """2.3e9 outputs; the products of a single block are exact, so that other calls of the
    same rows give the same bits."""
    x, w, scale, bias = make_linear(70000, 100, 32768, torch.bfloat16, 1, narrow=True)
    y = L.linear_f8(x, w, scale, bias=bias)
    for rows in (slice(0, 300), slice(30600, 30900), slice(32500, 32768)):
        assert torch.equal(y[rows], L.linear_f8(x[rows].contiguous(), w, scale, bias=bias))


def test_logits_past_32_bits(cuda):
    rows, vocab = 15000, 151936
    logits = torch.zeros(rows, vocab, dtype=torch.bfloat16, device="cuda")
    best = (torch.arange(rows, device="cuda") * 7919) % vocab
    logits[torch.arange(rows, device="cuda"), best] = 50.0
    offsets = torch.arange(0, rows + 1, 3, dtype=torch.int32, device="cuda")
    drafts = best.to(torch.int32)
    drafts[1::6] += 1 - 2 * (drafts[1::6] == vocab - 1).int()
    accepted, tokens = L.verify_drafts(logits, drafts, offsets, torch.rand(rows, 2, device="cuda"))
    want = torch.full((rows // 3, 3), -1, dtype=torch.int64, device="cuda")
    wrong = torch.arange(rows // 3, device="cuda") % 2 == 0   # their second token
    want[:, :2] = best.view(-1, 3)[:, :2]
    want[~wrong, 2] = best.view(-1, 3)[~wrong, 2]
    assert torch.equal(accepted.long(), torch.where(wrong, 1, 2)) and torch.equal(tokens.long().view(-1, 3), want)


def test_rotation_past_32_bits(cuda):
    rows = (1 << 18) + 100
    rope = kv8.rope_table(1000, 128)
    q = torch.randn(100, 64, 128, device="cuda").to(torch.bfloat16)
    at = torch.randint(0, 1000, (rows,), dtype=torch.int32, device="cuda")
    x = torch.zeros(rows, 64, 128, dtype=torch.bfloat16, device="cuda")
    x[-100:] = q
    kv8.rotate(x, None, at, rope, interleaved=True, q_out=x)
    check_rotated(q, x[-100:], rope, at[-100:], True, False)
    assert not x[:-100].any()


def test_calls_at_once(cuda):
    """Calls on several streams at a time, each with outputs and workspaces of its own."""
    linears = [make_linear(1500, 9000, n, dtype, 40 + n) for n, dtype in ((48, torch.float16), (3, torch.float32), (20, torch.bfloat16), (300, torch.bfloat16))]
    drafts = [make_drafts(counts, 40000, torch.bfloat16, 50 + i) for i, counts in enumerate(([3] * 20, [1, 5], [2] * 60, [8]))]
    want = [(L.linear_f8(*a[:3], bias=a[3]), *L.verify_drafts(**d)) for a, d in zip(linears, drafts)]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in want]
    for _ in range(5):
        got = [[L.linear_f8(*a[:3], bias=a[3], stream=s), *L.verify_drafts(**d, stream=s)] for a, d, s in zip(linears, drafts, streams)]
        torch.cuda.synchronize()
        assert all(torch.equal(g, w) for some, all_ in zip(got, want) for g, w in zip(some, all_))
