"""Steps in which sequences are refused: those behind them move up, and get their own
tokens all the same (kv8.asked_rows), eagerly and captured."""
import pytest
import torch

import lutmac_amd as L
from lutmac_amd import kv8
from test_gpu_draft_step import HD, HEADS, KV, VOCAB, WIDTH, Toy

pytestmark = pytest.mark.gpu
START = [10, 63, 20, 64, 5, 61]


class Waiting(Toy):
    """A toy whose sequences have START tokens and, all together, one page more than those
    need; the rows' tokens are laid out by what is asked for, at `asked`."""

    def __init__(self, rows):
        super().__init__(len(START), rows, 0.0)
        g = torch.Generator(device="cuda").manual_seed(5)
        self.held = kv8.KvPages.empty(len(START), 6, len(START) + 1)
        self.asked = torch.zeros(len(START), dtype=torch.int32, device="cuda")
        n = sum(START)
        i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
        offsets, _, _, _ = self.held.extend(i32(START), torch.zeros(n, dtype=torch.int32, device="cuda"))
        some = [torch.randn(n, KV, HD, generator=g, device="cuda").to(self.dtype) for _ in range(2)]
        self.cache.append(*some, offsets, self.held.lengths, self.held.pages)

    def step(self):
        self.held.extend(self.new, self.positions, offsets=self.offsets, granted=self.granted)
        at = kv8.asked_rows(self.asked, self.offsets, self.rows)
        x = self.embed[self.given[at].long()]
        q, k, v = L.linear_f8(x, *self.qkv).view(self.rows, -1, HD).split([HEADS, KV, KV], 1)
        kv8.rotate(q, k, self.positions, self.rope, interleaved=True, q_out=self.q, k_out=self.k)
        where = self.offsets, self.held.lengths, self.held.pages
        self.cache.append(self.k, v, *where)
        mixed = self.cache.attend(self.q, *where).view(self.rows, WIDTH)
        logits = L.linear_f8(x + 0.01 * mixed.nan_to_num(0.0), *self.head) * 4
        L.verify_drafts(logits, self.drafts[at], self.offsets, self.uniforms, temperature=self.temperature, accepted=self.accepted,
                        tokens=self.tokens)
        self.held.trim(torch.where(self.granted > 0, self.granted - 1 - self.accepted, 0).to(torch.int32))


@pytest.mark.parametrize("captured", [False, True])
def test_refused_in_the_middle(cuda, captured):
    toy = Waiting(30)
    run = toy.step
    if captured:
        toy.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            toy.step()
        run = graph.replay
    rng = torch.Generator().manual_seed(6)
    n = len(START)
    after = toy.next.tolist()
    last = [int(t) for t in torch.randint(0, VOCAB, (n,), generator=rng)]
    got, lengths, between = [[t] for t in last], list(START), 0
    for step in range(24):
        if step in (8, 16):   # a sequence ends: its page goes to one that waits
            drop = torch.zeros(n, dtype=torch.int32, device="cuda")
            drop[step // 8 * 2 - 2] = 10 ** 6
            toy.held.trim(drop)
            lengths[step // 8 * 2 - 2] = 0
        given, drafts, new, right, asked = [], [], [], [], []
        for s in range(n):
            count, tokens = int(torch.randint(0, 4, (), generator=rng)), [last[s]]
            good = int(torch.randint(0, count + 1, (), generator=rng))
            for j in range(count):
                t = after[tokens[-1]]
                tokens.append(t if j < good else (t + 1 + j) % VOCAB)
            asked.append(len(given))
            given += tokens
            drafts += tokens[1:] + [-1]
            new.append(count + 1)
            right.append(good)
        pad = toy.rows - len(given)
        for t, v in ((toy.given, given + [0] * pad), (toy.drafts, drafts + [0] * pad), (toy.new, new), (toy.asked, asked)):
            t.copy_(torch.tensor(v, dtype=torch.int32))
        run()
        torch.cuda.synchronize()
        granted, accepted, row = toy.granted.tolist(), toy.accepted.tolist(), 0
        assert all(g in (0, m) for g, m in zip(granted, new))
        between += any(granted[s] == 0 and any(granted[s + 1:]) for s in range(n))
        for s, g in enumerate(granted):
            if not g:
                assert accepted[s] == 0
                continue
            out = [t for t in toy.tokens[row:row + g].tolist() if t >= 0]
            assert accepted[s] == right[s] and len(out) == right[s] + 1
            assert toy.positions[row:row + g].tolist() == list(range(lengths[s], lengths[s] + g))
            got[s] += out
            last[s] = out[-1]
            lengths[s] += len(out)
            row += g
        assert toy.offsets.tolist()[-1] == row and toy.held.lengths.tolist() == lengths
    assert between > 5   # (some wait while others behind them go on)
    for tokens in got:
        assert all(b == after[a] for a, b in zip(tokens, tokens[1:]))
