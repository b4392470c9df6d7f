"""The paged 8-bit KV cache on the GPU (lutmac_kv8.h) against its plain 64-bit
restatement (kv8_reference.py): codes, scales and rotated queries equal to the
last bit, attention within the bound derived there."""
import numpy as np
import pytest
import torch

import lutmac_amd as L
from kv8_reference import PAGE, Cache, check_rotated
from lutmac_amd.kv8 import KvCache8, rope_table

pytestmark = pytest.mark.gpu
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def f64(t):
    return t.detach().double().cpu().numpy()


class Setup:
    """Sequences with `old` tokens before the call and `new` in it on a shuffled
    page table, q|k|v rows in one tensor, rows behind the last sequence, and a
    cache of random codes everywhere (stale ones among them)."""

    def __init__(self, dtype, hd, kv, group, new, old, seed=0, spare=3, behind=2, width=None):
        g = torch.Generator().manual_seed(seed)
        rng = np.random.default_rng(seed)
        self.dtype, self.hd, self.kv, self.heads = dtype, hd, kv, kv * group
        self.lengths = np.array([o + n for o, n in zip(old, new)], np.int32)
        self.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        need = [-(-int(n) // PAGE) for n in self.lengths]
        width = max(1, max(need)) if width is None else width
        pool = sum(need) + spare
        order = rng.permutation(pool).astype(np.int32)
        self.pages = np.full((len(new), width), -1, np.int32)
        at = 0
        for s, n in enumerate(need):
            n = min(n, width)
            self.pages[s, :n] = order[at:at + n]
            at += n
        rows = int(self.offsets[-1]) + behind
        qkv = torch.randn(rows, self.heads + 2 * kv, hd, generator=g)
        qkv[:, :, 3] *= 9
        self.qkv = qkv.to(TYPES[dtype]).cuda()
        self.q, self.k, self.v = self.qkv.split([self.heads, kv, kv], 1)
        self.rope = rope_table(max(1, int(self.lengths.max())), hd, 10000.0)
        self.cache = KvCache8((torch.randn(pool, kv, PAGE, hd, generator=g) * 40).round().clamp(-127, 127).to(torch.int8).cuda(),
                              (torch.randn(pool, kv, hd, PAGE, generator=g) * 40).round().clamp(-127, 127).to(torch.int8).cuda(),
                              (0.01 + 0.05 * torch.rand(pool, kv, 4, generator=g)).cuda(),
                              (0.01 + 0.05 * torch.rand(pool, kv, 4, generator=g)).cuda())
        self.where = tuple(torch.from_numpy(a).cuda() for a in (self.offsets, self.lengths, self.pages))

    def reference(self):
        c = self.cache
        return Cache(c.k.cpu().numpy(), c.v.cpu().numpy(), c.k_scale.cpu().numpy(), c.v_scale.cpu().numpy())

    def same_cache(self, ref):
        c = self.cache
        for name in ("k", "v", "k_scale", "v_scale"):
            np.testing.assert_array_equal(getattr(c, name).cpu().numpy(), getattr(ref, name), err_msg=name)

    def check_append(self):
        ref = self.reference()
        want = ref.append(f64(self.k), f64(self.v), f64(self.q), self.offsets, self.lengths, self.pages, self.rope.cpu().numpy())
        out = torch.full((self.q.shape[0], self.heads, self.hd), 7.0, dtype=TYPES[self.dtype], device="cuda")
        self.cache.append(self.k, self.v, *self.where, rope=self.rope, q=self.q, q_out=out)
        self.same_cache(ref)
        placed = ~np.isnan(want).all((1, 2))
        check_rotated(f64(out)[placed], want[placed], f64(self.q)[placed], self.dtype)
        assert (f64(out)[~placed] == 7.0).all()
        return ref, out

    def check_attend(self, ref=None, q=None, scale=None, **kw):
        ref = ref or self.reference()
        q = self.q if q is None else q
        out = torch.full((q.shape[0], self.heads, self.hd), 7.0, dtype=TYPES[self.dtype], device="cuda")
        self.cache.attend(q, *self.where, scale=scale, out=out, **kw)
        want, most = ref.attend(f64(q), self.offsets, self.lengths, self.pages, scale or self.hd ** -0.5, self.dtype)
        got, n = f64(out), int(self.offsets[-1])
        assert (got[n:] == 7.0).all()
        nan = np.isnan(want[:n])
        np.testing.assert_array_equal(np.isnan(got[:n]), nan)
        over = np.abs(got[:n] - want[:n])[~nan] - most[:n][~nan]
        assert over.size == 0 or over.max() <= 0, f"off by {over.max()} more than the bound"
        return out


RAGGED = [([1], [0]), ([1], [64]), ([3, 0, 1, 17], [0, 5, 15, 100]), ([16, 130, 2, 65], [16, 0, 63, 1]),
          ([0, 0, 40], [0, 70, 9])]


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("new,old", RAGGED)
def test_append(cuda, dtype, hd, new, old):
    Setup(dtype, hd, 2, 3, new, old, seed=len(new) + hd).check_append()


@pytest.mark.parametrize("dtype", sorted(TYPES))
@pytest.mark.parametrize("hd", [64, 128])
@pytest.mark.parametrize("group", [1, 4, 5])
@pytest.mark.parametrize("new,old", RAGGED)
def test_attend(cuda, dtype, hd, group, new, old):
    Setup(dtype, hd, 2, group, new, old, seed=len(new) + hd + group).check_attend()


@pytest.mark.parametrize("dtype,hd", [("float32", 64), ("bfloat16", 128)])
@pytest.mark.parametrize("new,old", [([1, 1, 2], [1300, 1, 2047]), ([90, 1], [900, 700]), ([200], [0])])
def test_attend_long(cuda, dtype, hd, new, old):
    """Contexts that are split over workgroups, and prompts of many row tiles."""
    Setup(dtype, hd, 1, 4, new, old, seed=3, width=64).check_attend()


def test_many_sequences(cuda):
    """More sequences than one look of the search holds (64), than two (4096)."""
    rng = np.random.default_rng(5)
    s = Setup("float32", 64, 1, 2, [int(n) for n in rng.integers(0, 3, 150)], [int(n) for n in rng.integers(0, 40, 150)], seed=5)
    ref, q = s.check_append()
    s.check_attend(ref, q)
    s = Setup("float32", 64, 1, 1, [int(n) for n in rng.integers(0, 2, 4500)], [0] * 4500, seed=6)
    ref, q = s.check_append()
    s.check_attend(ref, q)


@pytest.mark.parametrize("dtype", sorted(TYPES))
def test_steps_together(cuda, dtype):
    """Append and attend, step after step: prompts, then one token each, one
    sequence finishing earlier; q rotated in place."""
    s = Setup(dtype, 64, 2, 2, [5, 33, 1], [0, 0, 0], seed=9, spare=9, width=3)
    s.pages[:] = np.arange(9, dtype=np.int32).reshape(3, 3)[::-1]
    ref = s.reference()
    for step in range(36):
        new = [5, 33, 1] if step == 0 else [1, 1, 1 if step < 20 else 0]
        g = torch.Generator().manual_seed(step)
        s.offsets = np.concatenate([[0], np.cumsum(new)]).astype(np.int32)
        s.lengths = np.array(new, np.int32) if step == 0 else s.lengths + np.array(new, np.int32)
        s.rope = rope_table(80, 64)
        s.where = tuple(torch.from_numpy(a).cuda() for a in (s.offsets, s.lengths, s.pages))
        # growing values, so that scales grow within their blocks
        s.qkv = ((1 + 0.1 * step) * torch.randn(int(s.offsets[-1]), 8, 64, generator=g)).to(TYPES[dtype]).cuda()
        s.q, s.k, s.v = s.qkv.split([4, 2, 2], 1)
        before = f64(s.q)
        want = ref.append(f64(s.k), f64(s.v), before, s.offsets, s.lengths, s.pages, s.rope.cpu().numpy())
        q = s.cache.append(s.k, s.v, *s.where, rope=s.rope, q=s.q, q_out=s.q)
        assert q.data_ptr() == s.q.data_ptr()
        check_rotated(f64(q), want, before, dtype)
        s.same_cache(ref)
        s.check_attend(ref, q)


def test_append_exact_borders(cuda):
    """Quotients that lie exactly between two codes go to the even one: kept codes
    when the scale doubles or grows sixfold, new ones at multiples of half a step."""
    for factor in (2.0, 6.0):
        s = Setup("float32", 64, 1, 1, [1], [1], seed=1)
        s.cache.k_scale.fill_(0.75)
        s.cache.v_scale.fill_(0.75)
        for t in (s.k, s.v):
            t.copy_((torch.arange(64.0) + 0.5).cuda() * 0.75 * factor)
            t[..., 63] = 127 * 0.75 * factor
        ref = s.reference()
        ref.append(f64(s.k), f64(s.v), None, s.offsets, s.lengths, s.pages, None)
        assert s.cache.append(s.k, s.v, *s.where) is None
        s.same_cache(ref)


def test_append_special_values(cuda):
    """Zeros, tiny values, infinities and NaN: the block's own scale only; a NaN
    scale stays until the block starts anew; rows that see it become NaN."""
    for value in (0.0, 1e-38, float("inf"), float("nan"), -float("inf"), 3e38):
        s = Setup("float32", 64, 2, 2, [20, 3], [40, 10], seed=2)
        s.k[4, 1], s.v[7, 0] = 0.0, 0.0
        s.k[4, 1, 5] = value
        s.v[7, 0, 60] = value
        s.k[20, 0], s.v[20:23] = value if value == value else 1.0, 0.0
        ref, _ = s.check_append()
        if value != 3e38:
            s.check_attend(ref)
        # the sequences go on: one row more each
        s.offsets, s.lengths = np.array([0, 1, 2], np.int32), s.lengths + 1
        s.rope = rope_table(100, 64)
        s.where = tuple(torch.from_numpy(a).cuda() for a in (s.offsets, s.lengths, s.pages))
        s.check_append()


def test_places_outside(cuda):
    """Pages outside the pool, positions before the first token, past the table of
    pages and past the rotation table: no place, nothing seen, nothing written."""
    s = Setup("bfloat16", 64, 1, 2, [70, 5, 9], [10, 3, 130], seed=4, width=2)
    s.pages[0, 1] = 99
    s.pages[1, 0] = -7
    s.lengths[2] = 4   # five of the nine rows lie before position 0
    s.where = tuple(torch.from_numpy(a).cuda() for a in (s.offsets, s.lengths, s.pages))
    s.check_append()
    s.check_attend()
    s = Setup("bfloat16", 64, 1, 2, [70, 30], [100, 0], seed=4, width=2)   # 170 tokens, 128 places
    s.check_append()
    s.check_attend()
    s = Setup("float32", 128, 1, 2, [70, 30], [10, 0], seed=4)
    s.rope = rope_table(25, 128)
    s.check_append()


def test_unseen_scales(cuda):
    """Scales of blocks behind a sequence's end are not looked at; rows without any
    token give zeros; a query that is not finite gives NaN, its neighbours not."""
    s = Setup("float16", 128, 1, 4, [2, 1, 4], [30, 64, 0], seed=8)
    s.lengths[2] = 0
    s.where = tuple(torch.from_numpy(a).cuda() for a in (s.offsets, s.lengths, s.pages))
    for t in (s.cache.k_scale, s.cache.v_scale):
        t[int(s.pages[0, 0]), :, 2:] = float("nan")
        t[int(s.pages[1, 1]), :, 1:] = float("inf")
    s.q[1, 2, 100] = float("inf")
    s.q[2, 0, 0] = float("nan")
    s.q[0, 3] = 0.0
    out = s.check_attend()
    assert (out[3:7] == 0).all()


@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
@pytest.mark.parametrize("hd,group", [(64, 3), (128, 8)])
@pytest.mark.parametrize("new,old,width", [([300], [0], 5), ([97, 0, 260, 33], [64, 10, 31, 700], 12), ([150], [2000], 40)])
def test_attend_prompts(cuda, dtype, hd, group, new, old, width):
    """Prompts of 16-bit types take 256 rows a workgroup: whole and part tiles,
    prefixes, tables with pages to spare (some outside the pool) and parts."""
    s = Setup(dtype, hd, 2, group, new, old, seed=15, width=width)
    s.cache.k_scale.mul_(4)   # scores that outgrow their first reference
    s.check_attend()
    s.pages[0, 1] = -1
    s.where[2].copy_(torch.from_numpy(s.pages))
    s.cache.v_scale[int(s.pages[0, 0]), 0, 2] = 0.0
    s.check_attend()


def test_prompt_reference_rises(cuda):
    """Scores that grow page by page by more than a weight's range, and fall."""
    for sign in (1.0, -1.0):
        s = Setup("bfloat16", 128, 1, 2, [200], [400], seed=16)
        rise = torch.linspace(0.001, 0.4, s.cache.n_pages * 4)
        s.cache.k_scale.view(-1, 4)[torch.from_numpy(s.pages[0]).long().cuda()] = \
            (rise if sign > 0 else rise.flip(0))[:s.pages.shape[1] * 4].view(-1, 4).cuda()
        s.check_attend()


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_value_scales_far_apart(cuda, dtype):
    """V scales of 2^-99 to 2^100 in neighbouring blocks, K scales that leave scores
    of hundreds, and blocks of zeros."""
    s = Setup(dtype, 64, 1, 2, [3, 40], [200, 0], seed=11)
    n = s.cache.v_scale.numel()
    for seed in range(10 if dtype == "float32" else 0):
        at = torch.randperm(n, generator=torch.Generator().manual_seed(seed))
        s.cache.v_scale.view(-1).copy_(2.0 ** torch.linspace(-99, 100, n)[at].cuda())
        s.check_attend()
    s.cache.v_scale.fill_(2.0 ** -99)
    s.check_attend()
    s.cache.v_scale.fill_(0.02)
    s.cache.v_scale[:, :, 1] = 0.0
    s.cache.k_scale.mul_(30)
    s.check_attend()


def test_far_pages(cuda):
    """A pool whose codes pass 4 GiB: pages at its far end."""
    pool, kv, hd = 70000, 8, 128
    if torch.cuda.mem_get_info()[0] < 12 << 30:
        pytest.skip("needs 12 GiB of device memory")
    s = Setup("bfloat16", hd, kv, 2, [20, 1], [50, 130], seed=12)
    big = KvCache8(torch.empty(pool, kv, PAGE, hd, dtype=torch.int8, device="cuda"),
                   torch.empty(pool, kv, hd, PAGE, dtype=torch.int8, device="cuda"),
                   torch.empty(pool, kv, 4, device="cuda"), torch.empty(pool, kv, 4, device="cuda"))
    small, n = s.cache, s.cache.n_pages
    for name in ("k", "v", "k_scale", "v_scale"):
        getattr(big, name)[pool - n:].copy_(getattr(small, name))
    q0 = small.append(s.k, s.v, *s.where, rope=s.rope, q=s.q)
    out0 = small.attend(q0, *s.where)
    far = s.where[2] + (pool - n)
    q1 = big.append(s.k, s.v, s.where[0], s.where[1], far, rope=s.rope, q=s.q)
    rows = int(s.offsets[-1])
    for name in ("k", "v", "k_scale", "v_scale"):
        assert torch.equal(getattr(big, name)[pool - n:], getattr(small, name))
    assert torch.equal(q1[:rows], q0[:rows])
    assert torch.equal(big.attend(q1, s.where[0], s.where[1], far)[:rows], out0[:rows])


def test_graph_follows_lengths(cuda):
    """A captured step replays with the lengths and pages that the tensors hold
    then, among eager work, and equals the eager call."""
    s = Setup("float32", 64, 2, 4, [1] * 6, [200, 3, 64, 63, 0, 15], seed=13, spare=40, width=8)
    free = [p for p in range(s.cache.n_pages) if p not in set(s.pages[s.pages >= 0].tolist())]
    for i in range(6):
        for j in range(8):
            if s.pages[i, j] < 0 and free:
                s.pages[i, j] = free.pop()
    s.where[2].copy_(torch.from_numpy(s.pages))
    s.rope = rope_table(512, 64)
    work = torch.empty(max(1, s.cache.attend_workspace(torch.float32, 8, s.heads, 6, 8)), dtype=torch.uint8, device="cuda")
    q_out, out = torch.empty_like(s.q), torch.empty(8, s.heads, 64, device="cuda")
    ref = s.reference()
    graph = torch.cuda.CUDAGraph()
    torch.cuda.synchronize()
    with torch.cuda.graph(graph):
        s.cache.append(s.k, s.v, *s.where, rope=s.rope, q=s.q, q_out=q_out)
        s.cache.attend(q_out, *s.where, out=out, workspace=work)
    for step in range(5):
        s.qkv.copy_(torch.randn(s.qkv.shape, generator=torch.Generator().manual_seed(100 + step)).cuda())
        graph.replay()
        torch.cuda.synchronize()
        want = ref.append(f64(s.k), f64(s.v), f64(s.q), s.offsets, s.lengths, s.pages, s.rope.cpu().numpy())
        s.same_cache(ref)
        n = int(s.offsets[-1])
        check_rotated(f64(q_out[:n]), want[:n], f64(s.q[:n]), "float32")
        assert torch.equal(out[:n], s.cache.attend(q_out, *s.where)[:n])
        s.check_attend(ref, q_out)
        s.lengths += 1
        s.where[1].add_(1)


def test_streams_and_repeats(cuda):
    """The same call on another stream and many times over gives the same bits."""
    s = Setup("bfloat16", 128, 2, 4, [1, 1, 30], [1000, 3, 200], seed=14, width=40)
    first = s.cache.attend(s.q, *s.where).clone()
    other = torch.cuda.Stream()
    other.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(other):
        outs = [s.cache.attend(s.q, *s.where) for _ in range(20)]
    explicit = s.cache.attend(s.q, *s.where, stream=other)
    other.synchronize()
    n = int(s.offsets[-1])
    for o in outs + [explicit]:
        assert torch.equal(o[:n], first[:n])


def test_given_stream_owns_what_it_writes(cuda):
    """A call on a given stream takes its output and workspace from that stream's
    memory: what is freed on another stream while its work is under way is not
    written over."""
    s = Setup("bfloat16", 128, 2, 4, [1, 1, 30], [1000, 3, 200], seed=15, width=40)
    first, n = s.cache.attend(s.q, *s.where).clone(), int(s.offsets[-1])
    other = torch.cuda.Stream()
    torch.cuda.synchronize()
    marks, outs = [], []
    for i in range(10):
        x = torch.full(first.shape, float(i), dtype=first.dtype, device="cuda")
        marks.append((x * 2).sum(dtype=torch.float64))   # (frees x * 2 on the current stream)
        outs.append(s.cache.attend(s.q, *s.where, stream=other))
        del x
    torch.cuda.synchronize()
    for i, (m, o) in enumerate(zip(marks, outs)):
        assert m.item() == 2.0 * i * first.numel() and torch.equal(o[:n], first[:n])
