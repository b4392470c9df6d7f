"""Verification of drafted tokens (lmx_verify_drafts) against a plain restatement in
64 bits: whole numbers, all equal (a token differs only where a number lies within
rounding of 64 bits of a border)."""
import numpy as np
import pytest
import torch

import lutmac_amd as L

pytestmark = pytest.mark.gpu
TYPES = [torch.float32, torch.float16, torch.bfloat16]


def weights(x, t):
    """Weights of a row's logits (64 bits), None if they are no distribution."""
    top = x.max()
    if np.isnan(x).any() or top in (np.inf, -np.inf):
        return None
    if not t > 0:
        w = np.zeros(len(x))
        w[int(np.argmax(x))] = 1.0
        return w
    with np.errstate(invalid="ignore"):
        w = np.exp((x - top) / t)
    return np.where(x == -np.inf, 0.0, w)


def sampled(w, u):
    upto = np.cumsum(w)
    past = np.nonzero(upto > u * upto[-1])[0]
    return int(past[0]) if len(past) else int(np.nonzero(w)[0][-1])


def plain(logits, drafts, offsets, uniforms, probs=None, temperature=None):
    x, u = logits.double().cpu().numpy(), uniforms.double().cpu().numpy()
    q = None if probs is None else probs.double().cpu().numpy()
    d, off = drafts.tolist(), offsets.tolist()
    t = [1.0] * (len(off) - 1) if temperature is None else temperature.tolist()
    accepted, out = [], {}
    for s in range(len(off) - 1):
        a, b = off[s], off[s + 1]
        if a == b:
            accepted.append(0)
            continue
        out.update({r: -1 for r in range(a, b)})
        for r in range(a, b):
            w = weights(x[r], t[s])
            if w is None:
                break
            if r < b - 1:
                ok = 0 <= d[r] < len(w)
                share = 1.0 if q is None else q[r, d[r]] if ok else 0.0
                if ok and u[r, 0] * share * w.sum() < w[d[r]]:
                    out[r] = d[r]
                    continue
                if q is not None:
                    rest = np.maximum(w - q[r] * w.sum(), 0.0)
                else:
                    rest = w.copy()
                    if ok:
                        rest[d[r]] = 0.0
                w = rest if rest.sum() > 0 else w
            out[r] = sampled(w, u[r, 1])
            break
        accepted.append(r - a)
    return accepted, out


def make(counts, vocab, dtype, seed, probs=True, spread=2.5, first=0, behind=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    off = [first]
    for c in counts:
        off.append(off[-1] + c)
    rows = off[-1] + behind
    logits = (torch.randn(rows, vocab, generator=g, device="cuda") * spread).to(dtype)
    near = logits.float() + 0.6 * torch.randn(rows, vocab, generator=g, device="cuda")
    p = torch.softmax(near, -1)
    race = -torch.log(torch.rand(rows, vocab, generator=g, device="cuda").clamp_min(1e-30))
    drafts = (p / race).argmax(-1).to(torch.int32) if rows else torch.zeros(0, dtype=torch.int32, device="cuda")
    return dict(logits=logits, drafts=drafts, offsets=torch.tensor(off, dtype=torch.int32, device="cuda"),
                uniforms=torch.rand(rows, 2, generator=g, device="cuda"), probs=p if probs else None)


def check(a, **kw):
    rows = a["logits"].shape[0]
    accepted = torch.full((len(a["offsets"]) - 1,), -7, dtype=torch.int32, device="cuda")
    tokens = torch.full((rows,), -7, dtype=torch.int32, device="cuda")
    got = L.verify_drafts(**a, accepted=accepted, tokens=tokens, **kw)
    assert got[0] is accepted and got[1] is tokens
    want, out = plain(**a)
    assert accepted.tolist() == want
    full = [-7] * rows
    for r, t in out.items():
        full[r] = t
    assert tokens.tolist() == full
    return want, full


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("probs", [True, False])
@pytest.mark.parametrize("vocab", [1, 2, 31, 1000, 8192, 8193, 32003, 128256])
def test_verify(cuda, dtype, probs, vocab):
    accepted = []
    for seed, spread in ((1, 2.5), (2, 0.3), (3, 8.0)):
        a = make([1, 5, 0, 3, 9, 2, 1], vocab, dtype, seed, probs, spread, first=seed % 3, behind=seed % 2)
        accepted += check(a)[0]
        a["temperature"] = torch.tensor([0.7, 1.0, 1.0, 0.0, 0.0, 2.5, float("nan")], device="cuda")
        accepted += check(a)[0]
    if vocab > 1000:
        assert 0 in accepted and max(accepted) > 0   # (both come up)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_many_sequences(cuda, dtype):
    rng = np.random.default_rng(4)
    for probs in (True, False):
        a = make(rng.integers(0, 8, 300).tolist(), 997, dtype, 5, probs)
        a["temperature"] = torch.tensor(rng.choice([0.0, 0.5, 1.0], 300), dtype=torch.float32, device="cuda")
        check(a)
    check(make([300, 1, 40], 503, dtype, 6, True, 0.01))   # many accepted in a row


@pytest.mark.parametrize("vocab", [7, 9000])
def test_masks(cuda, vocab):
    """Tokens of -inf are never drawn, the type's lowest value is a number; rows with
    no distribution stop their sequence with -1."""
    for dtype in TYPES:
        low = torch.finfo(dtype).min
        a = make([4] * 12, vocab, dtype, 8)
        x, inf = a["logits"], float("inf")
        x[0] = -inf                       # nothing allowed
        x[5, :] = -inf
        x[5, vocab - 1] = low             # one allowed
        x[8] = low                        # all equal
        x[13, 3] = float("nan")
        x[17, 5] = inf
        x[20:24] = -inf
        x[24:28, : vocab - 2] = -inf
        x[28:32, 2:] = low
        x[32:36] = 0.0
        x[36] = -inf
        x[36, int(a["drafts"][36])] = 1.0
        a["probs"][40:44] = 0.0           # a draft that nothing is known of
        a["probs"][44:48] = 1.0           # nothing left of p - q
        check(a)
        a["temperature"] = torch.tensor([0.0, 1.0] * 6, device="cuda")
        check(a)
        a["temperature"] = torch.tensor([1e-30, 1e30, float("inf")] * 4, device="cuda")
        check(a)
        a["probs"] = None
        check(a)


def test_extreme_uniforms(cuda):
    """u of 0, just below 1 and (not allowed, but no harm) 1; tokens outside the
    vocabulary."""
    a = make([3] * 40, 2000, torch.float32, 9)
    n = a["uniforms"].shape[0]
    a["uniforms"][:, 0] = torch.tensor([0.0, 1 - 2.0 ** -24, 0.5], device="cuda").repeat(n)[:n]
    a["uniforms"][:, 1] = torch.tensor([1 - 2.0 ** -24, 0.0], device="cuda").repeat(n)[:n]
    check(a)
    a["drafts"][::7] = -1
    a["drafts"][3::11] = 2000
    a["drafts"][5::13] = 2 ** 31 - 1
    check(a)
    a["probs"] = None
    check(a)
    a["uniforms"][:, 1] = 1.0
    check(a)


def test_greedy_ties(cuda):
    """Of equal largest logits the first, wherever its part of the row."""
    x = torch.zeros(6, 40000, device="cuda")
    for r, at in enumerate(([39999], [8191, 8192], [20000, 30000, 39999], [0, 39999], [12345], [])):
        x[r, at] = 3.0
    firsts = [39999, 8191, 20000, 0, 12345, 0]
    a = dict(logits=x, offsets=torch.arange(7, dtype=torch.int32, device="cuda"), drafts=torch.zeros(6, dtype=torch.int32, device="cuda"),
             uniforms=torch.rand(6, 2, device="cuda"), temperature=torch.zeros(6, device="cuda"))
    assert check(a)[1] == firsts
    a["offsets"] = torch.tensor([0, 6], dtype=torch.int32, device="cuda")
    a["temperature"] = torch.zeros(1, device="cuda")
    a["drafts"].copy_(torch.tensor(firsts))
    assert check(a)[0] == [5]
    a["drafts"][2] = 30000   # as large, but not the first
    assert check(a)[0] == [2]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_strides_and_alignment(cuda, dtype):
    """Rows of a wider array that start at any element."""
    a = make([3, 2, 4], 9001, dtype, 10)
    want = check(a)
    for lead, gap in ((1, 0), (0, 5), (3, 1023)):
        for name in ("logits", "probs"):
            t = a[name]
            flat = torch.full((t.shape[0] * (9001 + gap) + lead,), 50.0, dtype=t.dtype, device="cuda")
            view = flat[lead:].view(t.shape[0], 9001 + gap)[:, :9001]
            view.copy_(t)
            assert check({**a, name: view}) == want
    work = torch.full((L.verify_drafts_workspace(3, 9, 9001, dtype) + 16,), 0xFF, dtype=torch.uint8, device="cuda")
    assert check(a, workspace=work[:-16]) == want
    assert (work[-16:] == 0xFF).all()
    with pytest.raises(L.LmxError):
        L.verify_drafts(**a, workspace=work[:-17])


def test_frequencies(cuda):
    """What comes out is distributed as p: 40000 sequences with one drafted token each.
    (A share p of n draws is off by more than 6 sqrt(p / n) once in 10^8.)"""
    n, vocab = 40000, 8
    g = torch.Generator(device="cuda").manual_seed(11)
    x = torch.randn(vocab, generator=g, device="cuda")
    q = torch.softmax(torch.randn(vocab, generator=g, device="cuda"), -1)
    drafts = torch.zeros(2 * n, dtype=torch.int32, device="cuda")
    drafts[::2] = torch.multinomial(q, n, replacement=True, generator=g).to(torch.int32)
    accepted, tokens = L.verify_drafts(x.expand(2 * n, vocab).contiguous(), drafts, torch.arange(0, 2 * n + 1, 2, dtype=torch.int32, device="cuda"),
                                       torch.rand(2 * n, 2, generator=g, device="cuda"), probs=q.expand(2 * n, vocab).contiguous())
    p = torch.softmax(x.double(), -1)
    for rows in (tokens[::2], tokens[1::2][accepted == 1]):
        share = torch.bincount(rows.long(), minlength=vocab).double() / len(rows)
        assert ((share - p).abs() < 6 * (p / len(rows)).sqrt()).all()
    assert abs(float((accepted == 1).double().mean()) - float(torch.minimum(p, q.double()).sum())) < 6 / n ** 0.5


def test_replays_and_streams(cuda):
    a = make([4, 1, 6], 20000, torch.bfloat16, 12)
    a["temperature"] = torch.ones(3, device="cuda")
    accepted, tokens = torch.empty(3, dtype=torch.int32, device="cuda"), torch.empty(11, dtype=torch.int32, device="cuda")
    work = torch.empty(L.verify_drafts_workspace(3, 11, 20000, torch.bfloat16), dtype=torch.uint8, device="cuda")
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        L.verify_drafts(**a, accepted=accepted, tokens=tokens, workspace=work)
    for i in range(4):
        b = make([2 + i, 0, 9 - i], 20000, torch.bfloat16, 20 + i)
        for name in ("logits", "drafts", "offsets", "uniforms", "probs"):
            a[name].copy_(b[name])
        a["temperature"].fill_((1.0, 0.0, 0.5, 2.0)[i])
        work.fill_(0xFF)
        graph.replay()
        torch.cuda.synchronize()
        got = accepted.tolist(), tokens.tolist()
        assert got == tuple(check(a))
    stream = torch.cuda.Stream()
    other = L.verify_drafts(**a, stream=stream)
    stream.synchronize()
    assert (other[0].tolist(), other[1].tolist()) == got
    empty = make([], 100, torch.float32, 1)
    assert L.verify_drafts(**empty)[0].shape == (0,)
    assert L.verify_drafts(**make([0, 0], 100, torch.float32, 1))[0].tolist() == [0, 0]
