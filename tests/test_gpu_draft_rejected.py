"""What rejected tokens leave in the 8-bit cache, and how a program takes that back too."""
import pytest
import torch

from lutmac_amd import kv8

pytestmark = pytest.mark.gpu
KV, HD, PAGE, BLOCK = 2, 64, 64, 16


def i32(v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


class Run:
    """Sequences of `lengths` tokens and `drafted` new ones each, of which `kept` stay;
    the dropped ones are `times` as large."""

    def __init__(self, lengths, drafted, kept, times, dtype=torch.float32, seed=1):
        g = torch.Generator(device="cuda").manual_seed(seed)
        self.n, self.lengths, self.drafted, self.kept = len(lengths), lengths, drafted, kept
        some = lambda n: torch.randn(n, KV, HD, generator=g, device="cuda")   # noqa: E731
        self.held = kv8.KvPages.empty(self.n, 8, 8 * self.n)
        self.cache = kv8.KvCache8.empty(8 * self.n, KV, HD)
        self.old = [(some(n).to(dtype), some(n).to(dtype)) for n in lengths]
        self.new = [(some(n), some(n)) for n in drafted]
        for (k, v), m in zip(self.new, kept):
            k[m:] *= times
            v[m:] *= times
        self.new = [(k.to(dtype), v.to(dtype)) for k, v in self.new]
        self.append(self.old)

    def append(self, rows, extend=True):
        counts = [len(k) for k, _ in rows]
        offsets = i32([sum(counts[:s]) for s in range(self.n + 1)])
        if extend:
            got = self.held.extend(i32(counts), torch.zeros(max(1, sum(counts)), dtype=torch.int32, device="cuda"))
            assert got[1].tolist() == counts
        self.cache.append(torch.cat([k for k, _ in rows]), torch.cat([v for _, v in rows]), offsets, self.held.lengths, self.held.pages)

    def tensors(self):
        return self.cache.k, self.cache.v, self.cache.k_scale, self.cache.v_scale

    def blocks(self):
        """Indices into the cache's tensors of the blocks that next tokens fall into."""
        out = []
        for s, n in enumerate(self.held.lengths.tolist()):
            if n % BLOCK:
                page, b = int(self.held.pages[s, n // PAGE]), n % PAGE // BLOCK
                at = slice(b * BLOCK, (b + 1) * BLOCK)
                out.append(((page, slice(None), at), (page, slice(None), slice(None), at), (page, slice(None), b), (page, slice(None), b)))
        return out

    def drop(self):
        self.held.trim(i32([a - b for a, b in zip(self.drafted, self.kept)]))

    def values(self, s):
        """(keys, values) [tokens, KV, HD] as the cache holds them, and their scales."""
        out = [[], [], [], []]
        for j in range(int(self.held.lengths[s])):
            page, t = int(self.held.pages[s, j // PAGE]), j % PAGE
            ks, vs = self.cache.k_scale[page, :, t // BLOCK].double(), self.cache.v_scale[page, :, t // BLOCK].double()
            out[0].append(self.cache.k[page, :, t].double() * ks[:, None])
            out[1].append(self.cache.v[page, :, :, t].double() * vs[:, None])
            out[2].append(ks)
            out[3].append(vs)
        return [torch.stack(x) for x in out]


CASES = [([20, 16, 5, 63, 64, 0, 100], [4, 4, 1, 5, 3, 6, 40], [2, 1, 0, 3, 1, 4, 20])]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("lengths,drafted,kept", CASES)
def test_kept_tokens_are_rounded_to_the_grown_scale(cuda, lengths, drafted, kept, dtype):
    r = Run(lengths, drafted, kept, 30.0, dtype)
    r.append(r.new)
    r.drop()
    for s in range(r.n):
        got = r.values(s)
        for i in (0, 1):
            true = torch.cat([r.old[s][i], r.new[s][i][:kept[s]]]).double()
            # half a step of the scale that the token was rounded to first (at most that of
            # its block now) and half of the grown one; scales are rounded to fp32
            off = ((got[i] - true).abs() / got[2 + i][..., None]).amax((1, 2))
            assert off.max() <= 1.0 + 2.0 ** -15
            first = lengths[s] // BLOCK * BLOCK
            if first:   # (blocks before the one that was growing are as they were)
                assert off[:first].max() <= 0.5 + 2.0 ** -15


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("times", [30.0, float("inf"), float("nan")])
@pytest.mark.parametrize("lengths,drafted,kept", CASES)
def test_as_if_never_drafted(cuda, lengths, drafted, kept, times, dtype):
    """The block put back and the kept rows appended again: the same bits as a cache that
    saw the kept tokens alone."""
    r = Run(lengths, drafted, kept, times, dtype)
    there = r.blocks()
    was = [[t[at].clone() for t, at in zip(r.tensors(), block)] for block in there]
    r.append(r.new)
    r.drop()
    if times != times or times > 1e9:   # what is left otherwise
        assert any(not r.values(s)[2 + i].isfinite().all() for s in range(r.n) for i in (0, 1))
    for block, old in zip(there, was):
        for t, at, o in zip(r.tensors(), block, old):
            t[at] = o
    r.append([(k[:m], v[:m]) for (k, v), m in zip(r.new, kept)], extend=False)
    w = Run(lengths, kept, kept, 1.0, dtype)
    w.new = [(k[:m], v[:m]) for (k, v), m in zip(r.new, kept)]
    w.append(w.new)
    for s in range(r.n):
        for a, b in zip(r.values(s), w.values(s)):
            assert torch.equal(a, b)
