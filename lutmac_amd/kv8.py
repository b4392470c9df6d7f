"""The paged 8-bit key/value cache (include/lutmac_kv8.h) on torch tensors, its
page table on the device, and rotations.

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

``KvPages`` keeps the page table: per step it grants tokens their places and takes
back those that are dropped, without the host:

    offsets, granted, positions, _ = held.extend(new, positions)
    at = asked_rows(asked, offsets, rows)         # of tokens laid out by what was asked
    q, k = rotate(q, k, positions, rope)          # (or let append rotate)
    cache.append(k, v, offsets, held.lengths, held.pages)
    out = cache.attend(q, offsets, held.lengths, held.pages)
    held.trim(rejected)
"""
import ctypes
import math

import torch

from . import BF16, F16, F32, Kv8BatchC, Kv8CacheC, check, lib, on_stream, torch_module

PAGE, BLOCK = 64, 16


def rope_table(positions, head_dim, theta=10000.0, factor=1.0, device="cuda", scaling=None):
    """(cos, sin) of (position / factor) * theta^(-2d / head_dim), the reference's
    apply_rope angles (embedding.cpp:36-75), as ``append`` and ``rotate`` take them:
    fp32 [positions, head_dim // 2, 2].  Angles are formed in 64 bits.  For a rotation of
    part of the heads head_dim is that part.

    scaling: a dict, for models that were trained on `original` positions --
    {"type": "linear", "factor"}: positions divided by the factor;
    {"type": "ntk", "factor"}: theta times factor^(d / (d - 2)), so that the slowest
    pair turns as linear scaling has it and the fastest as before;
    {"type": "llama3", "factor", "low_freq_factor", "high_freq_factor", "original"}: pairs of
    more than original / low turns' wavelength as linear scaling has them, those below
    original / high as before, between them a blend (the decoder's LMX_ROPE_LLAMA3);
    {"type": "yarn", "factor", "original", "beta_fast" (32), "beta_slow" (1),
    "attention" (0.1 ln(factor) + 1)}: pairs that turn beta_fast times and more over
    `original` positions as before, those that turn beta_slow times and less as linear scaling has them, a ramp
    over their index between; cos and sin times `attention`."""
    half = head_dim // 2
    d = torch.arange(half, dtype=torch.float64)
    kind, times, scaling = None, 1.0, dict(scaling or {})
    if scaling:
        kind, by = scaling.pop("type"), float(scaling.pop("factor"))
    if kind == "ntk":
        theta = theta * by ** (head_dim / (head_dim - 2)) if head_dim > 2 else theta
    freq = theta ** (-2.0 * d / head_dim)
    if kind == "linear":
        freq = freq / by
    elif kind == "llama3":
        low, high, original = (float(scaling.pop(n)) for n in ("low_freq_factor", "high_freq_factor", "original"))
        turns = original * freq / (2 * math.pi)   # over the original positions
        blend = ((turns - low) / (high - low)).clamp(0.0, 1.0)
        freq = freq * (blend + (1 - blend) / by)
    elif kind == "yarn":
        original, times = float(scaling.pop("original")), float(scaling.pop("attention", 0.1 * math.log(by) + 1.0 if by > 1 else 1.0))

        def pair(turns):   # the (fractional) pair that turns so often over the original positions
            return head_dim * math.log(original / (turns * 2 * math.pi)) / (2 * math.log(theta))
        first = max(math.floor(pair(float(scaling.pop("beta_fast", 32.0)))), 0)
        last = min(math.ceil(pair(float(scaling.pop("beta_slow", 1.0)))), head_dim - 1)
        blend = ((d - first) / max(last - first, 0.001)).clamp(0.0, 1.0)
        freq = freq * (1 - blend) + freq / by * blend
    elif kind not in (None, "ntk"):
        raise ValueError(f"scaling: type {kind!r}, expected linear, ntk, llama3 or yarn")
    if scaling:
        raise ValueError(f"scaling: {sorted(scaling)} not known to type {kind!r}")
    angle = (torch.arange(positions, dtype=torch.float64) / factor)[:, None] * freq
    return torch.stack([angle.cos() * times, angle.sin() * times], -1).float().to(device)


def rotate(q, k, positions, rope, interleaved=False, inverse=False, q_out=None, k_out=None, stream=None):
    """lmx_rotary: q [rows, heads, head_dim] and k [rows, kv_heads, head_dim] (or None)
    turned to positions int32 [rows] by rope fp32 [positions, pairs, 2] (rope_table), the
    first 2 * pairs elements of each head, the rest copied; pairs lie half that apart or,
    interleaved, side by side.  inverse: by -sin, the gradient, which also turns back
    what a table with cos^2 + sin^2 = 1 turned (a yarn table's `attention` comes in twice).
    Returns (q_out, k_out), which may be q and k (default new tensors; rows whose
    position the table lacks are not written).  Rows may lie any stride apart."""
    return on_stream(stream, torch_module().rotate, q, k, positions, rope, interleaved, inverse, q_out, k_out)


def asked_rows(asked, offsets, rows):
    """Where each of a step's rows lies among rows that were laid out before it was known
    who is granted: offsets int32 [sequences + 1] as ``KvPages.extend`` gives them, asked
    int32 [sequences] the first row of each sequence there.  Returns int64 [rows] (0
    for rows behind the last), to index tokens and drafts with: a refused sequence's
    rows are left out and those behind it move up.  Nothing is read on the host."""
    if not asked.numel():
        return torch.zeros(rows, dtype=torch.int64, device=offsets.device)
    r = torch.arange(rows, dtype=offsets.dtype, device=offsets.device)
    s = (torch.searchsorted(offsets, r, right=True) - 1).clamp_(0, asked.numel() - 1)
    return torch.where(r < offsets[-1], asked[s] + r - offsets[s], 0).long()


class KvPages:
    """Whose pages are whose, on the device: pages int32 [sequences, max_pages] as
    ``append`` and ``attend`` take them, lengths int32 [sequences], free int32 [pages]
    with the free ones in its first n_free[0] (int32 [1]) places.  The tensors are the
    caller's and written in place."""

    def __init__(self, pages, lengths, free, n_free):
        self._ops = torch_module()
        self._tensors = pages, lengths, free, n_free
        self._ops.kv8_pages(*self._tensors)

    pages = property(lambda self: self._tensors[0])
    lengths = property(lambda self: self._tensors[1])
    free = property(lambda self: self._tensors[2])
    n_free = property(lambda self: self._tensors[3])

    @classmethod
    def empty(cls, n_seqs, max_pages, n_pages, device="cuda"):
        """Sequences without tokens; page 0 is given out first."""
        return cls(torch.full((n_seqs, max_pages), -1, dtype=torch.int32, device=device),
                   torch.zeros(n_seqs, dtype=torch.int32, device=device),
                   torch.arange(n_pages - 1, -1, -1, dtype=torch.int32, device=device),
                   torch.full((1,), n_pages, dtype=torch.int32, device=device))

    def extend(self, new, positions, slots=None, offsets=None, granted=None, stream=None):
        """lmx_kv8_extend: room for new int32 [sequences] tokens.  positions int32 [rows]
        (as many rows as the step has room for) and slots int64 [rows] (or None) receive
        each row's position and page * 64 + position % 64; rows past the last stay as they
        are.  Returns (offsets [sequences + 1], granted [sequences], positions, slots): a
        sequence gets all its tokens or none, and the rows of one that gets none are not
        there (asked_rows)."""
        offsets, granted = on_stream(stream, self._ops.kv8_extend, *self._tensors, new, positions, slots, offsets, granted)
        return offsets, granted, positions, slots

    def trim(self, drop, stream=None):
        """lmx_kv8_trim: takes the last drop int32 [sequences] tokens back, and frees the
        pages that hold none any more.  A sequence ends with drop = its length.  Entries
        of the table that are no pages (negative: given up by the caller) are not freed.  Caches
        are not touched: the last block of kept tokens stays rounded to the scale that the
        dropped ones had asked for (NaN, where they were not finite)."""
        on_stream(stream, self._ops.kv8_trim, *self._tensors, drop)


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
