"""Refusals of the 8-bit serving operators, before any GPU work: the C entry
points' checks of sizes and pointers, and the Python layer's of tensors."""
import ctypes

import numpy as np
import pytest
import torch

import lutmac_amd as L
from lutmac_amd.kv8 import KvCache8, rope_table

A = 1 << 20   # an aligned address that no refused call reads


def cache(**kw):
    d = dict(k=A, v=A, k_scale=A, v_scale=A, n_pages=4, n_kv_heads=2, head_dim=64)
    d.update(kw)
    return L.Kv8CacheC(*[d[n] for n, _ in L.Kv8CacheC._fields_])


def batch(**kw):
    d = dict(offsets=A, lengths=A, pages=A, n_seqs=3, max_pages=5, n_rows=7)
    d.update(kw)
    return L.Kv8BatchC(*[d[n] for n, _ in L.Kv8BatchC._fields_])


def append(c=None, b=None, kind=L.F32, k=A, ks=128, v=A, vs=128, q=A, qs=256, o=A, os=256, heads=4, rope=A, n=10):
    c, b = c or cache(), b or batch()
    return L.lib().lmx_kv8_append(ctypes.addressof(c), ctypes.addressof(b), kind, k, ks, v, vs, q, qs, o, os, heads, rope, n, None)


def attend(c=None, b=None, kind=L.F32, q=A, qs=256, heads=4, scale=0.1, out=A, os=256, work=A, size=1 << 40):
    c, b = c or cache(), b or batch()
    return L.lib().lmx_kv8_attention(ctypes.addressof(c), ctypes.addressof(b), kind, q, qs, heads, scale, out, os, work, size, None)


BAD_CACHE = [dict(head_dim=96), dict(head_dim=256), dict(n_kv_heads=0), dict(n_pages=0), dict(n_pages=1 << 31), dict(k=None),
             dict(v_scale=None), dict(k=A + 8), dict(v=A + 4)]
BAD_BATCH = [dict(offsets=None), dict(lengths=None), dict(pages=None), dict(n_rows=1 << 25), dict(n_seqs=1 << 21),
             dict(max_pages=1 << 25)]


@pytest.mark.parametrize("bad", BAD_CACHE, ids=str)
def test_bad_cache(bad):
    assert append(c=cache(**bad)) == L.ERR_INVALID_ARGUMENT
    assert attend(c=cache(**bad)) == L.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("bad", BAD_BATCH, ids=str)
def test_bad_batch(bad):
    assert append(b=batch(**bad)) == L.ERR_INVALID_ARGUMENT
    assert attend(b=batch(**bad)) == L.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("bad", [dict(k=None), dict(v=None), dict(k=A + 8), dict(ks=100), dict(ks=129), dict(vs=64), dict(o=None),
                                 dict(qs=128), dict(os=252), dict(heads=3), dict(heads=0), dict(heads=130), dict(n=0),
                                 dict(rope=A + 4), dict(kind=L.BF16, ks=132)], ids=str)
def test_bad_append(bad):
    assert append(**bad) == L.ERR_INVALID_ARGUMENT
    assert L.lib().lmx_last_error()


@pytest.mark.parametrize("bad", [dict(q=None), dict(out=None), dict(q=A + 8), dict(qs=255), dict(os=128), dict(heads=5),
                                 dict(heads=0), dict(scale=0.0), dict(scale=-1.0), dict(scale=float("nan")),
                                 dict(scale=float("inf"))], ids=str)
def test_bad_attention(bad):
    assert attend(**bad) == L.ERR_INVALID_ARGUMENT


def test_unknown_types_and_nothing_to_do():
    assert append(kind=3) == attend(kind=-1) == L.ERR_UNSUPPORTED_FORMAT
    for b in (batch(n_seqs=0), batch(n_rows=0)):
        assert append(b=b) == attend(b=b) == L.OK
    assert L.lib().lmx_kv8_append(None, None, 0, *[None, 0] * 4, 1, None, 0, None) == L.ERR_INVALID_ARGUMENT
    assert L.lib().lmx_kv8_attention(None, None, 0, None, 0, 1, 1.0, None, 0, None, 0, None) == L.ERR_INVALID_ARGUMENT


def test_attention_workspace():
    """A long table splits: the call refuses a workspace that is short, missing or
    unaligned; a table of one page needs none."""
    n = ctypes.c_size_t()
    size = lambda c, b, h: L.lib().lmx_kv8_attention_workspace(ctypes.addressof(c), ctypes.addressof(b), L.F32, h, ctypes.byref(n))
    assert size(cache(), batch(max_pages=1), 4) == L.OK and n.value == 0
    b = batch(max_pages=1024)
    assert size(cache(), b, 4) == L.OK and n.value > 0
    for kw in (dict(work=None), dict(size=n.value - 1), dict(work=A + 4)):
        assert attend(b=b, **kw) == L.ERR_INVALID_ARGUMENT
    assert size(cache(), b, 3) == L.ERR_INVALID_ARGUMENT
    assert L.lib().lmx_kv8_attention_workspace(ctypes.addressof(cache()), ctypes.addressof(b), L.F32, 4, None) == L.ERR_INVALID_ARGUMENT


def linear(w=A, ws=128, sc=A, bias=None, x=A, y=A, kind=L.F32, rows=10, cols=100, n=3, work=A, size=1 << 30):
    return L.lib().lmx_linear_i8(w, ws, sc, bias, x, y, kind, rows, cols, n, work, size, None)


@pytest.mark.parametrize("bad", [dict(w=None), dict(sc=None), dict(x=None), dict(y=None), dict(w=A + 8), dict(ws=120), dict(ws=96),
                                 dict(ws=1 << 19), dict(rows=0), dict(cols=0), dict(cols=131073, ws=131088), dict(rows=1 << 25),
                                 dict(n=1 << 23), dict(x=A + 2), dict(y=A + 1), dict(bias=A + 2), dict(sc=A + 2), dict(work=None),
                                 dict(work=A + 8), dict(size=100)], ids=str)
def test_bad_linear(bad):
    assert linear(**bad) == L.ERR_INVALID_ARGUMENT


def test_linear_of_nothing():
    assert linear(n=0) == L.OK
    assert linear(kind=7) == L.ERR_UNSUPPORTED_FORMAT
    assert L.lib().lmx_weight_codes_i8(None, A, 16, A, None) == L.ERR_INVALID_ARGUMENT
    assert L.linear_i8_workspace(10, 100, 3) >= 3 * 100


def test_python_checks():
    def z(*s, dtype=torch.int8):
        return torch.zeros(*s, dtype=dtype)
    f = torch.float32
    good = (z(2, 1, 64, 64), z(2, 1, 64, 64), z(2, 1, 4, dtype=f), z(2, 1, 4, dtype=f))
    c = KvCache8(*good)
    for i, bad in [(0, z(2, 1, 32, 64)), (0, z(2, 1, 64, 96)), (1, z(2, 1, 64, 128)), (1, z(2, 1, 64, 64, dtype=torch.uint8)),
                   (2, z(2, 1, 5, dtype=f)), (3, z(2, 1, 4, dtype=torch.float64)), (0, z(2, 1, 64, 64).transpose(2, 3))]:
        with pytest.raises(ValueError):
            KvCache8(*[bad if i == j else t for j, t in enumerate(good)])
    k = z(3, 1, 64, dtype=f)
    i32 = lambda *s: z(*s, dtype=torch.int32)
    ok = dict(offsets=i32(2), lengths=i32(1), pages=i32(1, 2))
    for bad in [dict(offsets=i32(3)), dict(lengths=z(1, dtype=torch.int64)), dict(pages=i32(2, 2)), dict(pages=i32(1, 4)[:, ::2]),
                dict(offsets=i32(4)[::2])]:
        with pytest.raises(ValueError, match="offsets:|lengths:|pages:"):
            c.append(k, k, **{**ok, **bad})
        with pytest.raises(ValueError, match="offsets:|lengths:|pages:"):
            c.attend(k, **{**ok, **bad})
    for bad in [dict(v=z(2, 1, 64, dtype=f)), dict(v=k.half()), dict(k=z(3, 2, 64, dtype=f)), dict(q=z(3, 2, 32, dtype=f)),
                dict(q_out=k), dict(rope=z(5, 32, dtype=f)), dict(q=z(3, 64, 2, dtype=f).transpose(1, 2))]:
        with pytest.raises(ValueError, match="^(k|v|q|rope): |^q_out without q"):
            c.append(**{**dict(k=k, v=k), **bad}, **ok)
    with pytest.raises(ValueError, match="^q_out: "):
        c.append(k, k, q=k, q_out=k[:2], **ok)
    with pytest.raises(ValueError, match="^out: "):
        c.attend(k, out=k.half(), **ok)
    for bad in [lambda: c.append(k, k, **ok), lambda: c.append(k, k, q=k, rope=z(5, 32, 2, dtype=f), **ok), lambda: c.attend(k, **ok)]:
        with pytest.raises(ValueError, match="current device"):   # (all is well but for the device)
            bad()
    with pytest.raises(TypeError, match="expected a tensor"):
        c.attend(k.numpy(), **ok)
    with pytest.raises(L.LmxError):
        c.append(k.double(), k.double(), **ok)
    with pytest.raises(L.LmxError):
        c.attend(k.double(), **ok)
    x, w, s = z(2, 20, dtype=f), z(5, 32)[:, :20], z(5, dtype=f)
    for bad in [dict(x=x[:, :19]), dict(x=x.t()), dict(w=w.float()), dict(w=z(20, 5).t()), dict(w_scale=s[:4]), dict(bias=s.half()),
                dict(y=z(2, 4, dtype=f))]:
        with pytest.raises(ValueError, match=f"^{next(iter(bad))}: "):
            L.linear_i8(**{**dict(x=x, w=w, w_scale=s), **bad})
    with pytest.raises(ValueError, match="current device"):
        L.linear_i8(x, w, s)
    with pytest.raises(L.LmxError):
        L.linear_i8(x.double(), w, s)


def test_rope_table():
    t = rope_table(5, 64, theta=10000.0, factor=2.0, device="cpu").numpy().astype(np.float64)
    for p in range(5):
        for d in (0, 1, 31):
            a = p / 2.0 * 10000.0 ** (-2.0 * d / 64)
            assert abs(t[p, d, 0] - np.cos(a)) < 1e-7 and abs(t[p, d, 1] - np.sin(a)) < 1e-7
