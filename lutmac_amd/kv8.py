"""The paged 8-bit key/value cache (include/lutmac_kv8.h) on torch tensors.

A program that serves many sequences keeps one ``KvCache8`` per layer, a page
table and the lengths of its sequences on the device, and per step calls
``append`` with the new tokens' keys, values and queries and ``attend`` with the
rotated queries:

    q = cache.append(k, v, offsets, lengths, pages, rope=rope, q=q)
    out = cache.attend(q, offsets, lengths, pages)

Rows of a call are tokens: those of sequence s are offsets[s] .. offsets[s + 1]
- 1, the last of its lengths[s] tokens; token j lies in page pages[s, j // 64].
offsets, lengths and pages are int32 and read when the work runs, so a captured
call follows what they hold at each replay.
"""
import ctypes
import functools

import torch

from . import (ERR_UNSUPPORTED_FORMAT, Kv8BatchC, Kv8CacheC, LmxError, _current_device, _stream_ptr, _types, check, lib)

PAGE, BLOCK = 64, 16


def rope_table(positions, head_dim, theta=10000.0, factor=1.0, device="cuda"):
    """(cos, sin) of (position / factor) * theta^(-2d / head_dim), the reference's
    apply_rope angles (embedding.cpp:36-75), as ``append`` takes them: fp32
    [positions, head_dim // 2, 2].  Angles are formed in 64 bits."""
    d = torch.arange(head_dim // 2, dtype=torch.float64)
    angle = (torch.arange(positions, dtype=torch.float64) / factor)[:, None] * theta ** (-2.0 * d / head_dim)
    return torch.stack([angle.cos(), angle.sin()], -1).float().to(device)


def _bad(name, t, want):
    raise ValueError(f"{name}: {t.dtype} {tuple(t.shape)} with strides {t.stride()} on {t.device}, expected {want}")


def _rows(name, t, dtype, heads, head_dim, rows):
    """Checks a row tensor [rows, heads, head_dim], rows any stride apart; returns its row stride."""
    # (written for speed: every call checks up to four of them)
    if t.dtype is not dtype or t.shape != (rows, heads, head_dim):
        _bad(name, t, f"{dtype} [{rows}, {heads}, {head_dim}]")
    row, head, one = t.stride()
    if (one != 1 or (head != head_dim and heads > 1)) and rows:
        _bad(name, t, "a row's heads side by side")
    return row if rows > 1 else heads * head_dim   # (a single row's stride says nothing)


@functools.lru_cache(maxsize=1024)   # (of sizes alone)
def _workspace(n_pages, n_kv_heads, head_dim, kind, rows, heads, n_seqs, max_pages):
    c = Kv8CacheC(None, None, None, None, n_pages, n_kv_heads, head_dim)
    b, n = Kv8BatchC(None, None, None, n_seqs, max_pages, rows), ctypes.c_size_t()
    check(lib().lmx_kv8_attention_workspace(ctypes.byref(c), ctypes.byref(b), kind, heads, ctypes.byref(n)))
    return n.value


class KvCache8:
    """One layer's cache on tensors that the caller may hold too: k int8 [pages,
    kv_heads, 64, head_dim], v int8 [pages, kv_heads, head_dim, 64], k_scale and
    v_scale fp32 [pages, kv_heads, 4]; value = code * scale."""

    def __init__(self, k, v, k_scale, v_scale):
        pages, heads, page, hd = k.shape if k.dim() == 4 else (0, 0, 0, 0)
        if page != PAGE or (hd != 64 and hd != 128) or k.dtype is not torch.int8 or not k.is_contiguous():
            _bad("k", k, f"contiguous int8 [pages, kv_heads, {PAGE}, 64 or 128]")
        if v.dtype is not torch.int8 or v.shape != (pages, heads, hd, PAGE) or not v.is_contiguous():
            _bad("v", v, f"contiguous int8 {(pages, heads, hd, PAGE)}")
        shape = (pages, heads, PAGE // BLOCK)
        if k_scale.dtype is not torch.float32 or k_scale.shape != shape or not k_scale.is_contiguous():
            _bad("k_scale", k_scale, f"contiguous float32 {shape}")
        if v_scale.dtype is not torch.float32 or v_scale.shape != shape or not v_scale.is_contiguous():
            _bad("v_scale", v_scale, f"contiguous float32 {shape}")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads, self.head_dim = pages, heads, hd
        self._device = k.get_device()
        if v.get_device() != self._device or k_scale.get_device() != self._device or v_scale.get_device() != self._device:
            raise ValueError("the cache's tensors must be on one device")
        self._c = Kv8CacheC(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads, hd)

    @classmethod
    def empty(cls, n_pages, n_kv_heads, head_dim, device="cuda"):
        """A cache of zeros."""
        def zeros(dtype, *shape):
            return torch.zeros(n_pages, n_kv_heads, *shape, dtype=dtype, device=device)
        return cls(zeros(torch.int8, PAGE, head_dim), zeros(torch.int8, head_dim, PAGE), zeros(torch.float32, PAGE // BLOCK),
                   zeros(torch.float32, PAGE // BLOCK))

    def _batch(self, offsets, lengths, pages, rows, *others):
        """The call's batch, after checking that all its tensors are on the current device."""
        int32 = torch.int32
        if pages.dtype is not int32 or pages.dim() != 2 or not pages.is_contiguous():
            _bad("pages", pages, "contiguous int32 of 2 dimensions")
        n, width = pages.shape
        if offsets.dtype is not int32 or offsets.shape != (n + 1,) or not offsets.is_contiguous():
            _bad("offsets", offsets, f"contiguous int32 [{n + 1}] beside {n} page table rows")
        if lengths.dtype is not int32 or lengths.shape != (n,) or not lengths.is_contiguous():
            _bad("lengths", lengths, f"contiguous int32 [{n}] beside {n} page table rows")
        device = self._device
        for t in (offsets, lengths, pages, *others):
            if t is not None and t.get_device() != device:
                raise ValueError(f"expected tensors on the cache's device, got one on {t.device}")
        if device < 0 or device != _current_device():
            raise ValueError(f"expected tensors on the current device, the cache is on {self.k.device}")
        return Kv8BatchC(offsets.data_ptr(), lengths.data_ptr(), pages.data_ptr(), n, width, rows)

    def append(self, k, v, offsets, lengths, pages, rope=None, q=None, q_out=None, stream=None):
        """lmx_kv8_append: k and v [rows, kv_heads, head_dim] rotated (k) to their
        positions and appended; returns q [rows, heads, head_dim] rotated, in q_out
        (which may be q; default a new tensor), or None without q.  rope: fp32
        [positions, head_dim // 2, 2] (rope_table), or None."""
        dtype, hd, rows = k.dtype, self.head_dim, k.shape[0] if k.dim() else 0
        kind = _types().get(dtype)
        if kind is None:
            raise LmxError(ERR_UNSUPPORTED_FORMAT, f"k is {k.dtype}: float32, float16 or bfloat16")
        ks = _rows("k", k, dtype, self.n_kv_heads, hd, rows)
        vs = _rows("v", v, dtype, self.n_kv_heads, hd, rows)
        heads = qs = os = 0
        qp = op = rp = None
        if q is not None:
            heads = q.shape[1] if q.dim() == 3 else 0
            qs = _rows("q", q, dtype, heads, hd, rows)
            if q_out is None:
                q_out, os = torch.empty_like(q, memory_format=torch.contiguous_format), heads * hd
            else:
                os = _rows("q_out", q_out, dtype, heads, hd, rows)
            qp, op = q.data_ptr(), q_out.data_ptr()
        elif q_out is not None:
            raise ValueError("q_out without q")
        positions = 0
        if rope is not None:
            positions = rope.shape[0] if rope.dim() else 0
            if rope.dtype is not torch.float32 or rope.shape != (positions, hd // 2, 2) or not rope.is_contiguous():
                _bad("rope", rope, f"contiguous float32 [positions, {hd // 2}, 2]")
            rp = rope.data_ptr()
        b = self._batch(offsets, lengths, pages, rows, k, v, q, q_out, rope)
        check(lib().lmx_kv8_append(ctypes.byref(self._c), ctypes.byref(b), kind, k.data_ptr(), ks, v.data_ptr(), vs, qp, qs, op,
                                   os, heads, rp, positions, _stream_ptr(stream)))
        return q_out

    def attend(self, q, offsets, lengths, pages, scale=None, out=None, workspace=None, stream=None):
        """lmx_kv8_attention: causal attention of q [rows, heads, head_dim] (rotated)
        over the sequences' cached tokens; scale defaults to head_dim ** -0.5.
        workspace: a uint8 tensor of at least attend_workspace bytes that no
        overlapping call uses (default: torch allocates one for the call)."""
        dtype, hd = q.dtype, self.head_dim
        kind = _types().get(dtype)
        if kind is None:
            raise LmxError(ERR_UNSUPPORTED_FORMAT, f"q is {q.dtype}: float32, float16 or bfloat16")
        rows, heads = q.shape[:2] if q.dim() == 3 else (0, 0)
        qs = _rows("q", q, dtype, heads, hd, rows)
        if out is None:
            out, os = torch.empty_like(q, memory_format=torch.contiguous_format), heads * hd
        else:
            os = _rows("out", out, dtype, heads, hd, rows)
        b = self._batch(offsets, lengths, pages, rows, q, out, workspace)
        c = ctypes.byref(self._c)
        if workspace is None:
            size = _workspace(self.n_pages, self.n_kv_heads, hd, kind, rows, heads, b.n_seqs, b.max_pages)
            if size:
                workspace = torch.empty(size, dtype=torch.uint8, device=q.device)
        else:
            size = workspace.numel() * workspace.element_size()
        check(lib().lmx_kv8_attention(c, ctypes.byref(b), kind, q.data_ptr(), qs, heads, hd ** -0.5 if scale is None else scale,
                                      out.data_ptr(), os, None if workspace is None else workspace.data_ptr(), size,
                                      _stream_ptr(stream)))
        return out

    def attend_workspace(self, dtype, rows, heads, n_seqs, max_pages):
        """Bytes of workspace of an attend call of these sizes."""
        return _workspace(self.n_pages, self.n_kv_heads, self.head_dim, _types()[dtype], rows, heads, n_seqs, max_pages)
