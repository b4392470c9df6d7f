"""Steps that check drafted tokens, all on the device: pages granted, rows rotated,
appended to and attended over the 8-bit cache, logits by the 8-bit float linear
layer, drafts verified, rejected tokens taken back.

The model is a toy whose greedy tokens are known: a token's embedding leads to the
logit of the next of a fixed cycle by a wide margin, attention adds a little.  Each
operator's results are also held against a plain form on the way."""
import pytest
import torch

import lutmac_amd as L
from lutmac_amd import kv8
from test_gpu_rotary import check as check_rotated
from test_gpu_verify import plain as plain_verify

pytestmark = pytest.mark.gpu
VOCAB, HEADS, KV, HD = 300, 4, 2, 64
WIDTH = HEADS * HD


class Toy:
    def __init__(self, seqs, rows, temperature, dtype=torch.bfloat16):
        g = torch.Generator(device="cuda").manual_seed(3)
        normal = lambda *s: torch.randn(*s, generator=g, device="cuda")   # noqa: E731
        self.seqs, self.rows, self.dtype = seqs, rows, dtype
        self.next = torch.randperm(VOCAB, generator=g, device="cuda").roll(1)
        embed = torch.nn.functional.normalize(normal(VOCAB, WIDTH), dim=1)
        self.embed = (embed * 16).to(dtype)
        head = torch.empty_like(embed)
        head[self.next] = embed
        self.qkv = L.blocks_f8(normal((HEADS + 2 * KV) * HD, WIDTH) / 16)
        self.head = L.blocks_f8(head)
        self.rope = kv8.rope_table(4096, 48, scaling={"type": "yarn", "factor": 4.0, "original": 1024})
        self.cache = kv8.KvCache8.empty(seqs * 6 + 4, KV, HD)
        self.held = kv8.KvPages.empty(seqs, 6, seqs * 6 + 4)
        i32 = lambda *s: torch.zeros(*s, dtype=torch.int32, device="cuda")   # noqa: E731
        self.new, self.given, self.drafts = i32(seqs), i32(rows), i32(rows)
        self.offsets, self.granted, self.positions = i32(seqs + 1), i32(seqs), i32(rows)
        self.uniforms = torch.rand(rows, 2, generator=g, device="cuda")
        self.temperature = torch.full((seqs,), temperature, device="cuda")
        self.accepted, self.tokens = i32(seqs), i32(rows)
        # (rows behind the last sequence are computed on, but reach nothing)
        self.q = torch.zeros(rows, HEADS, HD, dtype=dtype, device="cuda")
        self.k = torch.zeros(rows, KV, HD, dtype=dtype, device="cuda")

    def step(self):
        """The rows' tokens in `given`, `drafts` those that the next rows are: all on the
        device, so that it can be captured."""
        self.held.extend(self.new, self.positions, offsets=self.offsets, granted=self.granted)
        x = self.embed[self.given.long()]
        self.plain_q, self.plain_k, v = L.linear_f8(x, *self.qkv).view(self.rows, -1, HD).split([HEADS, KV, KV], 1)
        kv8.rotate(self.plain_q, self.plain_k, self.positions, self.rope, interleaved=True, q_out=self.q, k_out=self.k)
        where = self.offsets, self.held.lengths, self.held.pages
        self.cache.append(self.k, v, *where)
        self.mixed = self.cache.attend(self.q, *where)
        self.logits = L.linear_f8(x + 0.01 * self.mixed.view(self.rows, WIDTH).nan_to_num(0.0), *self.head) * 4
        L.verify_drafts(self.logits, self.drafts, self.offsets, self.uniforms, temperature=self.temperature,
                        accepted=self.accepted, tokens=self.tokens)
        self.held.trim(torch.where(self.granted > 0, self.granted - 1 - self.accepted, 0).to(torch.int32))


def drive(toy, run, steps, rng):
    """`steps` steps with drafts that are right up to a random place; returns what
    each sequence got."""
    last = [int(t) for t in torch.randint(0, VOCAB, (toy.seqs,), generator=rng)]
    after = toy.next.tolist()
    got = [[t] for t in last]
    lengths = [0] * toy.seqs
    for _ in range(steps):
        given, drafts, new, right = [], [], [], []
        for s in range(toy.seqs):
            n = int(torch.randint(0, 4, (), generator=rng))   # drafted tokens; now and then none takes part
            if n == 0 and int(torch.randint(0, 3, (), generator=rng)) == 0:
                new.append(0)
                right.append(None)
                continue
            tokens, good = [last[s]], int(torch.randint(0, n + 1, (), generator=rng))
            for j in range(n):
                t = after[tokens[-1]]
                tokens.append(t if j < good else (t + 1 + j) % VOCAB)
            given += tokens
            drafts += tokens[1:] + [-1]
            new.append(n + 1)
            right.append(good)
        pad = toy.rows - len(given)
        for t, v in ((toy.given, given + [0] * pad), (toy.drafts, drafts + [0] * pad), (toy.new, new)):
            t.copy_(torch.tensor(v, dtype=torch.int32))
        run()
        torch.cuda.synchronize()
        assert toy.granted.tolist() == new
        accepted, tokens = plain_verify(toy.logits, toy.drafts, toy.offsets, toy.uniforms, temperature=toy.temperature)
        assert toy.accepted.tolist() == accepted and all(toy.tokens[r] == t for r, t in tokens.items())
        check_rotated(toy.plain_q[:len(given)], toy.q[:len(given)], toy.rope, toy.positions[:len(given)], True, False)
        row = 0
        for s, n in enumerate(new):
            if n:
                out = [t for t in toy.tokens[row:row + n].tolist() if t >= 0]
                assert len(out) == accepted[s] + 1
                assert toy.positions[row:row + n].tolist() == list(range(lengths[s], lengths[s] + n))
                lengths[s] += accepted[s] + 1
                got[s] += out
                last[s] = out[-1]
                if not float(toy.temperature[0]):
                    assert accepted[s] == right[s]
            row += n
        assert toy.held.lengths.tolist() == lengths
        used = sum(-(-n // 64) for n in lengths)
        assert int(toy.held.n_free) == toy.held.free.numel() - used
        pages = torch.cat([toy.held.pages[toy.held.pages >= 0], toy.held.free[: int(toy.held.n_free)]])
        assert torch.equal(pages.sort()[0].cpu(), torch.arange(toy.held.free.numel(), dtype=torch.int32))
    return got


@pytest.mark.parametrize("captured", [False, True])
def test_greedy_steps_follow_the_model(cuda, captured):
    toy = Toy(5, 24, 0.0)
    run = toy.step
    if captured:
        toy.step()   # (no sequence takes part yet)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            toy.step()
        run = graph.replay
    after = toy.next.tolist()
    for tokens in drive(toy, run, 40, torch.Generator().manual_seed(1)):
        assert len(tokens) > 40
        assert all(b == after[a] for a, b in zip(tokens, tokens[1:]))


def test_sampled_steps(cuda):
    toy = Toy(4, 16, 1.5, torch.float32)
    drive(toy, toy.step, 12, torch.Generator().manual_seed(2))


def test_attention_of_the_steps_is_that_of_the_cache(cuda):
    """What the planned rows attend to is what a table built by hand gives."""
    toy = Toy(3, 12, 0.0)
    drive(toy, toy.step, 5, torch.Generator().manual_seed(4))
    toy.new.copy_(torch.tensor([2, 0, 3], dtype=torch.int32))
    toy.given.fill_(7)
    lengths = [n + m for n, m in zip(toy.held.lengths.tolist(), [2, 0, 3])]
    toy.step()
    i32 = lambda v: torch.tensor(v, dtype=torch.int32, device="cuda")   # noqa: E731
    # what was taken back comes again, in the same places
    toy.held.extend(i32([a - b for a, b in zip(lengths, toy.held.lengths.tolist())]), toy.positions)
    again = toy.cache.attend(toy.q, i32([0, 2, 2, 5]), i32(lengths), toy.held.pages)
    assert torch.equal(again[:5], toy.mixed[:5])
