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

import torch

from . import BF16, F16, F32, Kv8BatchC, Kv8CacheC, check, lib, on_stream, torch_module

PAGE, BLOCK = 64, 16


def rope_table(positions, head_dim, theta=10000.0, factor=1.0, device="cuda"):
    """(cos, sin) of (position / factor) * theta^(-2d / head_dim), the reference's
    apply_rope angles (embedding.cpp:36-75), as ``append`` takes them: fp32
    [positions, head_dim // 2, 2].  Angles are formed in 64 bits."""
    d = torch.arange(head_dim // 2, dtype=torch.float64)
    angle = (torch.arange(positions, dtype=torch.float64) / factor)[:, None] * theta ** (-2.0 * d / head_dim)
    return torch.stack([angle.cos(), angle.sin()], -1).float().to(device)


class KvCache8:
    """One layer's cache on tensors that the caller may hold too: k int8 [pages,
    kv_heads, 64, head_dim], v int8 [pages, kv_heads, head_dim, 64], k_scale and
    v_scale fp32 [pages, kv_heads, 4]; value = code * scale.  The cache holds its
    tensors, which are not replaced (another cache costs little to make)."""

    def __init__(self, k, v, k_scale, v_scale):
        self._ops = torch_module()
        self._c = self._ops.kv8_cache(k, v, k_scale, v_scale)   # (checks them)
        self._tensors = k, v, k_scale, v_scale

    k = property(lambda self: self._tensors[0])
    v = property(lambda self: self._tensors[1])
    k_scale = property(lambda self: self._tensors[2])
    v_scale = property(lambda self: self._tensors[3])
    n_pages = property(lambda self: self.k.shape[0])
    n_kv_heads = property(lambda self: self.k.shape[1])
    head_dim = property(lambda self: self.k.shape[3])

    @classmethod
    def empty(cls, n_pages, n_kv_heads, head_dim, device="cuda"):
        """A cache of zeros."""
        def zeros(dtype, *shape):
            return torch.zeros(n_pages, n_kv_heads, *shape, dtype=dtype, device=device)
        return cls(zeros(torch.int8, PAGE, head_dim), zeros(torch.int8, head_dim, PAGE), zeros(torch.float32, PAGE // BLOCK),
                   zeros(torch.float32, PAGE // BLOCK))

    def append(self, k, v, offsets, lengths, pages, rope=None, q=None, q_out=None, stream=None):
        """lmx_kv8_append: k and v [rows, kv_heads, head_dim] rotated (k) to their
        positions and appended; returns q [rows, heads, head_dim] rotated, in q_out
        (which may be q; default a new tensor), or None without q.  rope: fp32
        [positions, head_dim // 2, 2] (rope_table), or None.  Rows may lie any stride
        apart."""
        return on_stream(stream, self._ops.kv8_append, self._c, k, v, offsets, lengths, pages, rope, q, q_out)

    def attend(self, q, offsets, lengths, pages, scale=None, out=None, workspace=None, stream=None):
        """lmx_kv8_attention: causal attention of q [rows, heads, head_dim] (rotated)
        over the sequences' cached tokens; scale defaults to head_dim ** -0.5.
        workspace: a uint8 tensor of at least attend_workspace bytes that no
        overlapping call uses (default: torch allocates one for the call)."""
        return on_stream(stream, self._ops.kv8_attend, self._c, q, offsets, lengths, pages, scale, out, workspace)

    def attend_workspace(self, dtype, rows, heads, n_seqs, max_pages):
        """Bytes of workspace of an attend call of these sizes."""
        kind = {torch.float32: F32, torch.float16: F16, torch.bfloat16: BF16}[dtype]
        pages, kv_heads, _, head_dim = self.k.shape
        c, n = Kv8CacheC(None, None, None, None, pages, kv_heads, head_dim), ctypes.c_size_t()
        b = Kv8BatchC(None, None, None, n_seqs, max_pages, rows)
        check(lib().lmx_kv8_attention_workspace(ctypes.byref(c), ctypes.byref(b), kind, heads, ctypes.byref(n)))
        return n.value
