"""Refusals of the operators of a drafted step, before any GPU work: the C entry
points' checks of sizes and pointers, and the Python layer's of tensors; rotation
tables against their formulas."""
import ctypes
import math

import pytest
import torch

import lutmac_amd as L
from lutmac_amd import kv8

A = 1 << 20   # an aligned address that no refused call reads


def linear(w=A, ws=128, sc=A, bias=None, x=A, y=A, kind=L.F32, rows=10, cols=100, n=3, work=A, size=1 << 30):
    return L.lib().lmx_linear_f8(w, ws, sc, bias, x, y, kind, rows, cols, n, work, size, None)


@pytest.mark.parametrize("bad", [dict(w=None), dict(sc=None), dict(x=None), dict(y=None), dict(w=A + 8), dict(ws=120), dict(ws=96),
                                 dict(ws=1 << 19), dict(rows=0), dict(cols=0), dict(cols=131073, ws=131088), dict(rows=1 << 25),
                                 dict(n=1 << 23), dict(x=A + 2), dict(y=A + 1), dict(bias=A + 2), dict(sc=A + 2), dict(work=None),
                                 dict(work=A + 8), dict(size=100)], ids=str)
def test_bad_linear(bad):
    assert linear(**bad) == L.ERR_INVALID_ARGUMENT
    assert L.lib().lmx_last_error()


def test_linear_of_nothing():
    assert linear(n=0) == L.OK
    assert linear(kind=3) == L.ERR_UNSUPPORTED_FORMAT
    assert L.lib().lmx_linear_f8_workspace(10, 10, 1, 0, None) == L.ERR_INVALID_ARGUMENT
    assert L.linear_f8_workspace(10, 100, 3, torch.bfloat16) >= 3 * 100


def pages(**kw):
    d = dict(pages=A, lengths=A, free_pages=A, n_free=A, n_seqs=3, max_pages=5, n_pages=7)
    d.update(kw)
    return L.Kv8PagesC(*[d[n] for n, _ in L.Kv8PagesC._fields_])


def extend(p=None, new=A, rows=10, offsets=A, granted=A, positions=A, slots=A):
    p = p or pages()
    return L.lib().lmx_kv8_extend(ctypes.addressof(p), new, rows, offsets, granted, positions, slots, None)


def trim(p=None, drop=A):
    p = p or pages()
    return L.lib().lmx_kv8_trim(ctypes.addressof(p), drop, None)


@pytest.mark.parametrize("bad", [dict(pages=None), dict(lengths=None), dict(free_pages=None), dict(n_free=None), dict(pages=A + 2),
                                 dict(lengths=A + 1), dict(free_pages=A + 2), dict(n_free=A + 2), dict(n_seqs=1 << 21),
                                 dict(max_pages=1 << 25), dict(n_pages=1 << 31)], ids=str)
def test_bad_pages(bad):
    assert extend(pages(**bad)) == L.ERR_INVALID_ARGUMENT
    assert trim(pages(**bad)) == L.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("bad", [dict(new=None), dict(new=A + 2), dict(rows=1 << 25), dict(offsets=None), dict(offsets=A + 2),
                                 dict(granted=None), dict(positions=None), dict(positions=A + 1), dict(slots=A + 4)], ids=str)
def test_bad_extend(bad):
    assert extend(**bad) == L.ERR_INVALID_ARGUMENT


def test_bad_trim():
    assert trim(drop=None) == trim(drop=A + 2) == L.ERR_INVALID_ARGUMENT
    assert L.lib().lmx_kv8_trim(None, A, None) == L.lib().lmx_kv8_extend(None, A, 1, A, A, A, A, None) == L.ERR_INVALID_ARGUMENT
    assert trim(pages(n_seqs=0), drop=None) == L.OK


def rotary(kind=L.F32, q=A, qs=256, qo=A, qos=256, heads=4, k=A, ks=128, ko=A, kos=128, kv=2, hd=64, rd=64, inter=0, inv=0, at=A, rows=3,
           rope=A, n=10):
    return L.lib().lmx_rotary(kind, q, qs, qo, qos, heads, k, ks, ko, kos, kv, hd, rd, inter, inv, at, rows, rope, n, None)


@pytest.mark.parametrize("bad", [dict(q=None), dict(qo=None), dict(ko=None), dict(at=None), dict(rope=None), dict(rope=A + 4),
                                 dict(at=A + 2), dict(n=0), dict(n=1 << 31), dict(hd=0), dict(hd=1025), dict(rd=0), dict(rd=63),
                                 dict(rd=66), dict(heads=0), dict(heads=1025), dict(kv=0), dict(kv=1025), dict(rows=1 << 25),
                                 dict(qs=255), dict(kos=127), dict(qs=1 << 41), dict(q=A + 2), dict(ko=A + 1), dict(inter=2), dict(inv=-1),
                                 dict(qos=300), dict(kind=L.F16, q=A + 1)], ids=str)
def test_bad_rotary(bad):
    assert rotary(**bad) == L.ERR_INVALID_ARGUMENT


def test_rotary_of_nothing():
    assert rotary(rows=0) == L.OK
    assert rotary(kind=5) == L.ERR_UNSUPPORTED_FORMAT


def drafts(**kw):
    d = dict(offsets=A, drafts=A, uniforms=A, temperature=A, n_seqs=3, n_rows=7, vocab=1000)
    d.update(kw)
    return L.DraftsC(*[d[n] for n, _ in L.DraftsC._fields_])


def verify(d=None, kind=L.F32, x=A, xs=1000, q=A, qs=1000, accepted=A, tokens=2 * A, work=A, size=1 << 30):
    d = d or drafts()
    return L.lib().lmx_verify_drafts(ctypes.addressof(d), kind, x, xs, q, qs, accepted, tokens, work, size, None)


@pytest.mark.parametrize("bad", [dict(offsets=None), dict(drafts=None), dict(uniforms=None), dict(offsets=A + 2), dict(drafts=A + 1),
                                 dict(uniforms=A + 4), dict(temperature=A + 2), dict(n_seqs=1 << 21), dict(n_rows=1 << 21), dict(vocab=0),
                                 dict(vocab=1 << 25)], ids=str)
def test_bad_drafts(bad):
    assert verify(drafts(**bad)) == L.ERR_INVALID_ARGUMENT


@pytest.mark.parametrize("bad", [dict(x=None), dict(x=A + 2), dict(xs=999), dict(xs=1 << 41), dict(q=A + 2), dict(qs=999), dict(accepted=None),
                                 dict(accepted=A + 2), dict(tokens=None), dict(tokens=A + 1), dict(tokens=A), dict(work=None), dict(work=A + 8),
                                 dict(size=16)], ids=str)
def test_bad_verify(bad):
    assert verify(**bad) == L.ERR_INVALID_ARGUMENT


def test_verify_of_nothing():
    assert verify(drafts(n_seqs=0), x=None) == L.OK
    assert verify(kind=9) == L.ERR_UNSUPPORTED_FORMAT
    assert L.lib().lmx_verify_drafts_workspace(ctypes.addressof(drafts()), 0, None) == L.ERR_INVALID_ARGUMENT
    assert L.lib().lmx_verify_drafts(None, 0, A, 1, A, 1, A, A, A, 1, None) == L.ERR_INVALID_ARGUMENT
    assert L.verify_drafts_workspace(3, 7, 1000, torch.float16) > 0


def z(*s, dtype=torch.float32):
    return torch.zeros(*s, dtype=dtype)


I32, I64, F8 = torch.int32, torch.int64, torch.float8_e4m3fn


@pytest.mark.parametrize("bad", [dict(x=z(2, 199)), dict(x=z(200, 2).t()), dict(w=z(130, 208)[:, :200]), dict(w=z(200, 130).to(F8).t()),
                                 dict(w_scale=z(1, 2)), dict(w_scale=z(2, 1)), dict(w_scale=z(2, 2).double()), dict(bias=z(129)),
                                 dict(bias=z(130).half()), dict(y=z(2, 129))], ids=str)
def test_python_linear(bad):
    good = dict(x=z(2, 200), w=z(130, 208).to(F8)[:, :200], w_scale=z(2, 2))
    with pytest.raises(ValueError, match=f"^{next(iter(bad))}: "):
        L.linear_f8(**{**good, **bad})
    with pytest.raises(ValueError, match="current device"):
        L.linear_f8(**good)
    with pytest.raises(L.LmxError):
        L.linear_f8(**{**good, "x": z(2, 200).double()})
    with pytest.raises(TypeError, match="expected a tensor"):
        L.linear_f8(**{**good, "w": None})


def test_python_pages():
    good = dict(pages=z(3, 4, dtype=I32), lengths=z(3, dtype=I32), free=z(9, dtype=I32), n_free=z(1, dtype=I32))
    held = kv8.KvPages(**good)
    for bad in [dict(pages=z(3, 4)), dict(pages=z(4, 3, dtype=I32).t()), dict(lengths=z(4, dtype=I32)), dict(lengths=z(3, dtype=I64)),
                dict(free=z(3, 3, dtype=I32)), dict(free=z(18, dtype=I32)[::2]), dict(n_free=z(2, dtype=I32))]:
        with pytest.raises(ValueError, match=f"^{next(iter(bad))}: "):
            kv8.KvPages(**{**good, **bad})
    ok = dict(new=z(3, dtype=I32), positions=z(8, dtype=I32), slots=z(8, dtype=I64))
    for bad in [dict(new=z(2, dtype=I32)), dict(new=z(3, dtype=I64)), dict(positions=z(8, dtype=I64)), dict(positions=z(2, 4, dtype=I32)),
                dict(slots=z(7, dtype=I64)), dict(slots=z(8, dtype=I32)), dict(offsets=z(3, dtype=I32)), dict(granted=z(4, dtype=I32))]:
        with pytest.raises(ValueError, match=f"^{next(iter(bad))}: "):
            held.extend(**{**ok, **bad})
    with pytest.raises(ValueError, match="current device"):
        held.extend(**ok)
    with pytest.raises(ValueError, match="^drop: "):
        held.trim(z(2, dtype=I32))
    with pytest.raises(ValueError, match="current device"):
        held.trim(z(3, dtype=I32))
    with pytest.raises(TypeError, match="expected a tensor"):
        held.trim([1, 2, 3])


def test_python_rotate():
    good = dict(q=z(5, 4, 64), k=z(5, 2, 64), positions=z(5, dtype=I32), rope=z(9, 32, 2))
    for bad in [dict(q=z(5, 256)), dict(q=z(5, 64, 4).transpose(1, 2)), dict(k=z(5, 2, 32)), dict(k=z(4, 2, 64)), dict(k=z(5, 2, 64).half()),
                dict(positions=z(4, dtype=I32)), dict(positions=z(5, dtype=I64)), dict(rope=z(9, 33, 2)), dict(rope=z(9, 32, 3)),
                dict(rope=z(9, 64)), dict(rope=z(9, 0, 2)), dict(rope=z(9, 32, 2).double()), dict(q_out=z(5, 4, 32)), dict(k_out=z(5, 2, 64).half())]:
        with pytest.raises(ValueError, match=f"^{next(iter(bad))}: "):
            kv8.rotate(**{**good, **bad})
    with pytest.raises(ValueError, match="k_out without k"):
        kv8.rotate(**{**good, "k": None, "k_out": z(5, 2, 64)})
    with pytest.raises(ValueError, match="current device"):
        kv8.rotate(**good)
    with pytest.raises(L.LmxError):
        kv8.rotate(**{**good, "q": z(5, 4, 64).double()})


def test_python_verify():
    good = dict(logits=z(6, 50), drafts=z(6, dtype=I32), offsets=z(3, dtype=I32), uniforms=z(6, 2), probs=z(6, 50), temperature=z(2))
    for bad in [dict(logits=z(50)), dict(logits=z(50, 6).t()), dict(drafts=z(5, dtype=I32)), dict(drafts=z(6, dtype=I64)),
                dict(offsets=z(0, dtype=I32)), dict(offsets=z(3)), dict(uniforms=z(6)), dict(uniforms=z(6, 2).double()),
                dict(probs=z(6, 49)), dict(probs=z(6, 50).half()), dict(temperature=z(3)), dict(accepted=z(3, dtype=I32)),
                dict(tokens=z(6, dtype=I64))]:
        with pytest.raises(ValueError, match=f"^{next(iter(bad))}: "):
            L.verify_drafts(**{**good, **bad})
    with pytest.raises(ValueError, match="current device"):
        L.verify_drafts(**good)
    with pytest.raises(L.LmxError):
        L.verify_drafts(**{**good, "logits": z(6, 50).double()})


def angles(table):
    """Frequencies of a table from its second position, and the factor of its values."""
    t = table.double()
    return torch.atan2(t[1, :, 1], t[1, :, 0]), t[0, :, 0]


def test_scaled_tables():
    """Angles of position 1 to 2^-23 of pi, against the published rules pair by pair."""
    def same(table, want, times=1.0):
        got, factor = angles(table)
        for d, w in enumerate(want):
            assert abs(float(got[d]) - w) < 4e-7, d
            assert abs(float(factor[d]) - times) < 1e-6
    plain = [10000.0 ** (-2 * d / 64) for d in range(32)]
    same(kv8.rope_table(2, 64, device="cpu"), plain)
    same(kv8.rope_table(2, 64, device="cpu", scaling={"type": "linear", "factor": 8}), [f / 8 for f in plain])
    ntk = kv8.rope_table(2, 64, device="cpu", scaling={"type": "ntk", "factor": 8})
    assert abs(float(angles(ntk)[0][0]) - 1) < 4e-7 and abs(float(angles(ntk)[0][31]) / (plain[31] / 8) - 1) < 1e-4
    # the published rule of the Llama-3 scaling, in wavelengths
    factor, low, high, original = 32.0, 1.0, 4.0, 8192.0
    want = []
    for f in [500000.0 ** (-2 * d / 64) for d in range(32)]:
        wave = 2 * math.pi / f
        smooth = (original / wave - low) / (high - low)
        want.append(f if wave < original / high else f / factor if wave > original / low else (1 - smooth) * f / factor + smooth * f)
    same(kv8.rope_table(2, 64, theta=500000.0, device="cpu",
                        scaling={"type": "llama3", "factor": factor, "low_freq_factor": low, "high_freq_factor": high, "original": original}), want)
    # yarn: the ramp runs over the pairs between 32 turns and 1 turn over the original positions
    find = lambda turns: 64 * math.log(4096 / (turns * 2 * math.pi)) / (2 * math.log(10000.0))   # noqa: E731
    lo, hi = math.floor(find(32)), math.ceil(find(1))
    want = []
    for d, f in enumerate(plain):
        ramp = min(max((d - lo) / (hi - lo), 0), 1)
        want.append(f / 16 * ramp + f * (1 - ramp))
    same(kv8.rope_table(2, 64, device="cpu", scaling={"type": "yarn", "factor": 16, "original": 4096}), want, 0.1 * math.log(16) + 1)
    same(kv8.rope_table(2, 64, device="cpu", scaling={"type": "yarn", "factor": 16, "original": 4096, "attention": 1.0}), want)
    far = kv8.rope_table(131072, 64, theta=500000.0, device="cpu").double()
    for d in (0, 5, 31):
        a = 131071 * 500000.0 ** (-2 * d / 64)
        assert abs(float(far[131071, d, 0]) - math.cos(a)) < 1e-7 and abs(float(far[131071, d, 1]) - math.sin(a)) < 1e-7
    for bad in ({"type": "spiral", "factor": 2}, {"type": "linear", "factor": 2, "original": 5}):
        with pytest.raises(ValueError, match="^scaling: "):
            kv8.rope_table(2, 64, device="cpu", scaling=bad)


def test_blocks_f8_on_the_host():
    w = torch.randn(130, 200)
    codes, scale = L.blocks_f8(w)
    assert codes.shape == w.shape and codes.dtype == F8 and scale.shape == (2, 2) and codes.stride(0) % 16 == 0
    back = codes.float() * scale.repeat_interleave(128, 0)[:130].repeat_interleave(128, 1)[:, :200]
    assert ((back - w).abs() <= w.abs() * (2.0 ** -4 + 1e-6) + scale.max() * 2.0 ** -10).all()
