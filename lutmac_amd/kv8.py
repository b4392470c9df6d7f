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
import math

import torch

from . import (ERR_UNSUPPORTED_FORMAT, Kv8BatchC, Kv8CacheC, LmxError, _on_current_device, _stream_ptr, _types, check,
               lib)

PAGE, BLOCK = 64, 16


def rope_table(positions, head_dim, theta=10000.0, factor=1.0, device="cuda"):
    """(cos, sin) of (position / factor) * theta^(-2d / head_dim), the reference's
    apply_rope angles (embedding.cpp:36-75), as ``append`` takes them: fp32
    [positions, head_dim // 2, 2].  Angles are formed in 64 bits."""
    d = torch.arange(head_dim // 2, dtype=torch.float64)
    angle = (torch.arange(positions, dtype=torch.float64) / factor)[:, None] * theta ** (-2.0 * d / head_dim)
    return torch.stack([angle.cos(), angle.sin()], -1).float().to(device)


def _rows(name, t, kind, heads, head_dim, rows=None):
    """Checks a row tensor [rows, heads, head_dim], rows any stride apart; returns its row stride."""
    if _types().get(t.dtype) != kind:
        raise ValueError(f"{name} is {t.dtype}: the rows of a call have one type")
    if t.dim() != 3 or t.shape[2] != head_dim or (heads and t.shape[1] != heads) or (rows is not None and t.shape[0] != rows):
        raise ValueError(f"{name} {tuple(t.shape)}: expected [{rows if rows is not None else 'rows'}, {heads or 'heads'}, {head_dim}]")
    if t.numel() and (t.stride(2) != 1 or (t.shape[1] > 1 and t.stride(1) != head_dim)):
        raise ValueError(f"{name}: the heads of a row must lie side by side")
    # (a single row's stride says nothing)
    return t.stride(0) if t.shape[0] > 1 else t.shape[1] * head_dim


class KvCache8:
    """One layer's cache on tensors that the caller may hold too: k int8 [pages,
    kv_heads, 64, head_dim], v int8 [pages, kv_heads, head_dim, 64], k_scale and
    v_scale fp32 [pages, kv_heads, 4]; value = code * scale."""

    def __init__(self, k, v, k_scale, v_scale):
        if k.dim() != 4 or k.shape[2] != PAGE or k.shape[3] not in (64, 128):
            raise ValueError(f"k {tuple(k.shape)}: expected [pages, kv_heads, {PAGE}, 64 or 128]")
        pages, heads, _, hd = k.shape
        if v.shape != (pages, heads, hd, PAGE):
            raise ValueError(f"v {tuple(v.shape)}: expected {(pages, heads, hd, PAGE)}")
        if k.dtype != torch.int8 or v.dtype != torch.int8:
            raise ValueError("codes must be int8")
        for s in (k_scale, v_scale):
            if s.shape != (pages, heads, PAGE // BLOCK) or s.dtype != torch.float32:
                raise ValueError(f"scales must be float32 {(pages, heads, PAGE // BLOCK)}")
        for t in (k, v, k_scale, v_scale):
            if not t.is_contiguous():
                raise ValueError("cache tensors must be contiguous")
        self.k, self.v, self.k_scale, self.v_scale = k, v, k_scale, v_scale
        self.n_pages, self.n_kv_heads, self.head_dim = pages, heads, hd
        self._c = Kv8CacheC(k.data_ptr(), v.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), pages, heads, hd)

    @classmethod
    def empty(cls, n_pages, n_kv_heads, head_dim, device="cuda"):
        """A cache of zeros."""
        def zeros(dtype, *shape):
            return torch.zeros(n_pages, n_kv_heads, *shape, dtype=dtype, device=device)
        return cls(zeros(torch.int8, PAGE, head_dim), zeros(torch.int8, head_dim, PAGE), zeros(torch.float32, PAGE // BLOCK),
                   zeros(torch.float32, PAGE // BLOCK))

    def _batch(self, offsets, lengths, pages, rows):
        for name, t, dim in (("offsets", offsets, 1), ("lengths", lengths, 1), ("pages", pages, 2)):
            if t.dtype != torch.int32 or t.dim() != dim or not t.is_contiguous():
                raise ValueError(f"{name}: contiguous int32 of {dim} dimension(s)")
        n = lengths.shape[0]
        if offsets.shape[0] != n + 1 or pages.shape[0] != n:
            raise ValueError(f"{n} lengths need {n + 1} offsets and {n} page table rows")
        return Kv8BatchC(offsets.data_ptr(), lengths.data_ptr(), pages.data_ptr(), n, pages.shape[1], rows)

    def append(self, k, v, offsets, lengths, pages, rope=None, q=None, q_out=None, stream=None):
        """lmx_kv8_append: k and v [rows, kv_heads, head_dim] rotated (k) to their
        positions and appended; returns q [rows, heads, head_dim] rotated, in q_out
        (which may be q; default a new tensor), or None without q.  rope: fp32
        [positions, head_dim // 2, 2] (rope_table), or None."""
        kind = _types().get(k.dtype)
        if kind is None:
            raise LmxError(ERR_UNSUPPORTED_FORMAT, f"k is {k.dtype}: float32, float16 or bfloat16")
        hd, rows = self.head_dim, k.shape[0]
        ks, vs = _rows("k", k, kind, self.n_kv_heads, hd), _rows("v", v, kind, self.n_kv_heads, hd, rows)
        heads = qs = os = 0
        if q is not None:
            heads = q.shape[1]
            qs = _rows("q", q, kind, heads, hd, rows)
            if q_out is None:
                q_out = torch.empty(rows, heads, hd, dtype=q.dtype, device=q.device)
            os = _rows("q_out", q_out, kind, heads, hd, rows)
        elif q_out is not None:
            raise ValueError("q_out without q")
        if rope is not None and (rope.dtype != torch.float32 or rope.dim() != 3 or rope.shape[1:] != (hd // 2, 2)
                                 or not rope.is_contiguous()):
            raise ValueError(f"rope: contiguous float32 [positions, {hd // 2}, 2]")
        b = self._batch(offsets, lengths, pages, rows)
        _on_current_device(self.k, self.v, self.k_scale, self.v_scale, k, v, q, q_out, rope, offsets, lengths, pages)
        check(lib().lmx_kv8_append(ctypes.addressof(self._c), ctypes.addressof(b), kind, k.data_ptr(), ks, v.data_ptr(), vs,
                                   None if q is None else q.data_ptr(), qs, None if q is None else q_out.data_ptr(), os,
                                   heads, None if rope is None else rope.data_ptr(), 0 if rope is None else rope.shape[0],
                                   _stream_ptr(stream)))
        return q_out

    def attend(self, q, offsets, lengths, pages, scale=None, out=None, workspace=None, stream=None):
        """lmx_kv8_attention: causal attention of q [rows, heads, head_dim] (rotated)
        over the sequences' cached tokens; scale defaults to head_dim ** -0.5.
        workspace: a uint8 tensor of at least attend_workspace bytes that no
        overlapping call uses (default: torch allocates one for the call)."""
        kind = _types().get(q.dtype)
        if kind is None:
            raise LmxError(ERR_UNSUPPORTED_FORMAT, f"q is {q.dtype}: float32, float16 or bfloat16")
        hd, rows = self.head_dim, q.shape[0]
        qs = _rows("q", q, kind, 0, hd)
        heads = q.shape[1]
        if out is None:
            # rows behind the last sequence are left as they are: of a new tensor, zeros
            out = torch.empty(rows, heads, hd, dtype=q.dtype, device=q.device)
        os = _rows("out", out, kind, heads, hd, rows)
        b = self._batch(offsets, lengths, pages, rows)
        need = ctypes.c_size_t()
        check(lib().lmx_kv8_attention_workspace(ctypes.addressof(self._c), ctypes.addressof(b), heads, ctypes.byref(need)))
        if workspace is None and need.value:
            workspace = torch.empty(need.value, dtype=torch.uint8, device=q.device)
        _on_current_device(self.k, self.v, self.k_scale, self.v_scale, q, out, offsets, lengths, pages, workspace)
        check(lib().lmx_kv8_attention(ctypes.addressof(self._c), ctypes.addressof(b), kind, q.data_ptr(), qs, heads,
                                      1.0 / math.sqrt(hd) if scale is None else scale, out.data_ptr(), os,
                                      None if workspace is None else workspace.data_ptr(),
                                      0 if workspace is None else workspace.numel() * workspace.element_size(),
                                      _stream_ptr(stream)))
        return out

    def attend_workspace(self, rows, heads, n_seqs, max_pages):
        """Bytes of workspace of an attend call of these sizes."""
        b, n = Kv8BatchC(None, None, None, n_seqs, max_pages, rows), ctypes.c_size_t()
        check(lib().lmx_kv8_attention_workspace(ctypes.addressof(self._c), ctypes.addressof(b), heads, ctypes.byref(n)))
        return n.value
