"""The decoder on an 8-bit KV cache (lmx_decoder_create_kv, LMX_KV_INT8).

Logits are held against a forward pass in 64 bits over the plain cache of
kv8_reference.  A value within DECIDED of the border between two codes may
take either code on the device (its keys and values come out of fp32 linears);
what each of these choices does to the logits is computed by the pass run again
with that one code changed, and allowed.
"""
import ctypes

import numpy as np
import pytest
import torch

import kv8_reference as R
import lutmac_amd as L
import oracle
from lutmac_amd import decode as D

gpu = pytest.mark.gpu
# relative to the logits' norm: fp32 sums in another order, over the layers
TOL = 1e-5
# of a code: fp32 linears, off by some 2^-22 of the largest key, times 127
DECIDED = 2.0 ** -13


class Cache(R.Cache):
    """Counts the values near a border between two codes and turns the one numbered `turn`."""

    def start(self, turn):
        self.near, self.turn = 0, turn
        return self

    def round(self, x):
        c = np.round(x)
        for i in np.argwhere(np.abs(np.abs(x - c) - 0.5) < DECIDED):
            if self.near == self.turn:
                c[tuple(i)] += 1 if x[tuple(i)] > c[tuple(i)] else -1
            self.near += 1
        return c.astype(np.int8)


def dense(entry, rows, cols, group):
    """The matrix behind 4-bit planes: its products with the unit vectors."""
    w = np.empty((rows, cols))
    for j in range(cols):
        x = np.zeros(cols, np.float32)
        x[j] = 1.0
        w[:, j] = oracle.planes_gemv(L.FMT_INT4, entry[0], entry[1], rows, cols, group, x)
    return w


class Plain:
    """The decoder's forward pass in 64 bits over the plain 8-bit cache."""

    def __init__(self, model):
        self.m, self.c = model, model.cfg
        shapes = model.shapes()
        self.w = [{n: dense(y[n], *shapes[n], model.group) for n in shapes} for y in model.layers]
        self.head = dense(model.head, self.c.vocab, self.c.hidden, model.group)
        hd = self.c.head_dim
        angle = np.arange(self.c.max_seq)[:, None] * self.c.rope_theta ** (-np.arange(0, hd, 2) / hd)
        self.rope = np.stack([np.cos(angle), np.sin(angle)], -1)

    def norm(self, x, w):
        return x / np.sqrt((x * x).mean(-1, keepdims=True) + self.c.rms_eps) * w

    def run(self, tokens, passes, turn=-1):
        """Logits of every position of `tokens`, appended in runs of `passes` positions;
        how many codes lay near a border."""
        c, hd = self.c, self.c.head_dim
        n_pages = (c.max_seq + R.PAGE - 1) // R.PAGE
        pages = np.arange(n_pages)[None]
        at, out, near = 0, [], 0
        caches = [Cache(np.zeros((n_pages, c.n_kv_heads, R.PAGE, hd), np.int8),
                        np.zeros((n_pages, c.n_kv_heads, hd, R.PAGE), np.int8),
                        np.zeros((n_pages, c.n_kv_heads, 4), np.float32),
                        np.zeros((n_pages, c.n_kv_heads, 4), np.float32)) for _ in self.w]
        for n in passes:
            x = self.head[tokens[at:at + n]]
            for y, w, cache in zip(self.m.layers, self.w, caches):
                qkv = self.norm(x, y["in_norm"]) @ w["qkv"].T
                if y["qkv_bias"] is not None:
                    qkv = qkv + y["qkv_bias"]
                q, k, v = np.split(qkv, [c.q_dim, c.q_dim + c.kv_dim], -1)
                cache.start(turn - near)
                where = ([0, n], [at + n], pages)
                q = cache.append(k.reshape(n, -1, hd), v.reshape(n, -1, hd), q.reshape(n, -1, hd), *where, self.rope)
                near += cache.near
                o, _ = cache.attend(q, *where, hd ** -0.5, "float32")
                x = x + o.reshape(n, -1) @ w["o"].T
                gate, up = np.split(self.norm(x, y["post_norm"]) @ w["gate_up"].T, 2, -1)
                x = x + (gate / (1 + np.exp(-gate)) * up) @ w["down"].T
            out.append(self.norm(x, self.m.final_norm) @ self.head.T)
            at += n
        return np.concatenate(out), near

    def bounded(self, tokens, passes):
        """Logits, and how far the device's may be from them."""
        want, near = self.run(tokens, passes)
        most = np.linalg.norm(want, axis=-1, keepdims=True) * TOL * np.ones_like(want)
        for i in range(near):
            # twice: what two choices do together is their sum to first order
            most += 2 * np.abs(self.run(tokens, passes, i)[0] - want)
        return want, most


def small(max_seq, n_layers=2, head_dim=64, heads=4, kv=2, bias=False, seed=3):
    cfg = D.small_config(hidden=256, n_layers=n_layers, n_heads=heads, n_kv_heads=kv, head_dim=head_dim, ffn=512, vocab=300,
                         max_seq=max_seq, rope_mode=D.ROPE_REFERENCE, rope_factor=1.0, rope_theta=1e4, qkv_bias=bias)
    return D.SyntheticModel(cfg, seed=seed, group=128, random_norms=True)


def step_logits(dec, tokens):
    """[positions, batch, vocab] of single steps; tokens [batch, positions]."""
    dec.reset(tokens)
    lg = torch.empty(dec.batch * dec.cfg.vocab, dtype=torch.float32, device="cuda")
    return np.stack([dec.step(lg).cpu().numpy().reshape(dec.batch, -1).copy() for _ in range(tokens.shape[1])])


@pytest.mark.parametrize("bad", [-1, 2])
def test_unknown_format_is_refused(bad):
    h = ctypes.c_void_p()
    cs = D.small_config().c_struct()
    assert L.lib().lmx_decoder_create_kv(ctypes.byref(cs), 1, bad, ctypes.byref(h)) == L.ERR_INVALID_ARGUMENT
    assert L.lib().lmx_decoder_create_kv(ctypes.byref(cs), 0, 1, ctypes.byref(h)) == L.ERR_INVALID_ARGUMENT
    assert L.lib().lmx_decoder_create_kv(None, 1, 1, ctypes.byref(h)) == L.ERR_INVALID_ARGUMENT
    assert h.value is None


@gpu
@pytest.mark.parametrize("n,kw", [(20, {}), (12, dict(head_dim=128, heads=6, bias=True, seed=4)), (70, dict(n_layers=1, kv=1, heads=2))],
                         ids=["two layers", "bias and 128", "two pages"])
def test_steps(cuda, n, kw):
    m = small(max_seq=n + 3, **kw)
    tokens = np.random.default_rng(n).integers(0, m.cfg.vocab, n)
    got = step_logits(D.Decoder(m, kv="int8"), tokens[None])[:, 0]
    want, most = Plain(m).bounded(tokens, [1] * n)
    assert (np.abs(got - want) <= most).all(), (np.abs(got - want) / most).max()


@gpu
@pytest.mark.parametrize("batch", [2, 5])
def test_batched_steps(cuda, batch):
    m, n = small(max_seq=20), 10
    tokens = np.random.default_rng(batch).integers(0, m.cfg.vocab, (batch, n))
    got = step_logits(D.Decoder(m, batch=batch, kv="int8"), tokens)
    plain = Plain(m)
    for b in range(batch):
        want, most = plain.bounded(tokens[b], [1] * n)
        assert (np.abs(got[:, b] - want) <= most).all(), (b, (np.abs(got[:, b] - want) / most).max())


def check_picks(plain, out, n_prompt, passes):
    """Every generated token's logit is the largest one, up to the bound."""
    n = len(out)
    want, most = plain.bounded(out[:-1], passes)
    for t in range(n_prompt - 1, n - 1):
        pick = out[t + 1]
        assert want[t, pick] + most[t, pick] >= (want[t] - most[t]).max(), t


@gpu
@pytest.mark.parametrize("batch,n_prompt,n_new", [(1, 2, 12), (1, 30, 6), (3, 17, 5)])
def test_generate(cuda, batch, n_prompt, n_new):
    # more than 4 prompt tokens: all but the last in one pass (batch 1: the
    # steps of more than 3 new tokens are a replayed graph, twice over)
    m = small(max_seq=64)
    prompt = np.random.default_rng(n_prompt).integers(0, m.cfg.vocab, (batch, n_prompt))
    dec = D.Decoder(m, batch=batch, kv="int8")
    out = np.atleast_2d(dec.generate(prompt, n_new)[0])
    again = np.atleast_2d(dec.generate(prompt, n_new)[0])
    np.testing.assert_array_equal(out, again)
    np.testing.assert_array_equal(out[:, :n_prompt], prompt)
    plain = Plain(m)
    first = [n_prompt - 1] if n_prompt > 4 else [1] * (n_prompt - 1)
    for b in range(batch):
        check_picks(plain, out[b], n_prompt, first + [1] * n_new)
    if n_prompt <= 4:   # the same steps one by one
        dec.reset(prompt)
        for _ in range(n_prompt + n_new - 1):
            dec.step()
        np.testing.assert_array_equal(np.atleast_2d(dec.tokens(n_prompt + n_new)), out)


@gpu
def test_fp32_decoder_is_untouched_beside_it(cuda):
    # an 8-bit and an fp32 decoder of one model, steps in turn: the fp32 one's
    # logits are those of a decoder made without a choice, bit by bit
    m = small(max_seq=32)
    tokens = np.random.default_rng(9).integers(0, m.cfg.vocab, (1, 16))
    want = step_logits(D.Decoder(m), tokens)
    a, b = D.Decoder(m, kv="f32"), D.Decoder(m, kv="int8")
    a.reset(tokens)
    b.reset(tokens)
    la, lb = (torch.empty(m.cfg.vocab, dtype=torch.float32, device="cuda") for _ in range(2))
    for t in range(16):
        b.step(lb)
        np.testing.assert_array_equal(a.step(la).cpu().numpy(), want[t, 0])


@gpu
def test_sequences_start_over(cuda):
    # nothing of a longer sequence before is left in the next one's logits
    m = small(max_seq=70)
    rng = np.random.default_rng(10)
    tokens = rng.integers(0, m.cfg.vocab, (1, 9))
    fresh = step_logits(D.Decoder(m, kv="int8"), tokens)
    dec = D.Decoder(m, kv="int8")
    dec.generate(rng.integers(0, m.cfg.vocab, 60), 10)
    np.testing.assert_array_equal(step_logits(dec, tokens), fresh)


@gpu
def test_file_on_int8_cache(cuda, tmp_path):
    formats = {n: (L.FMT_INT4, 128, 0) for n in (*D.QuantizedModel.NAMES, "embed")}
    cfg = D.small_config(rope_mode=D.ROPE_REFERENCE, rope_factor=1.0, rope_theta=1e4, vocab=300, hidden=256, ffn=512)
    m = D.QuantizedModel(cfg, formats, seed=5)
    m.save_v2(tmp_path / "m.lutmac")
    f = D.LutmacModel(tmp_path / "m.lutmac", max_seq=cfg.max_seq, kv="int8")
    prompt = np.random.default_rng(6).integers(0, cfg.vocab, 20)
    got = f.generate(prompt, 8)[0]
    np.testing.assert_array_equal(got, D.Decoder(m, kv="int8").generate(prompt, 8)[0])
    f.close()
