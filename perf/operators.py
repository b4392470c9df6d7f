"""The 8-bit serving operators: their calls, and what they compute in plain torch.

*append*: keys and values of new tokens are rotated to their positions and
written into a paged cache that holds 8-bit codes with one fp32 scale per
block of 16 tokens and KV head; the queries are rotated on the way.

*attention*: grouped-query, causal attention of those queries over that cache,
one token per sequence or whole prompts.

*linear*: a linear layer in 8-bit integers, one scale per token (made in the
call from the largest magnitude) and one per output channel.

The cache of one layer: k [pages, kv_heads, 64, head_dim] and v [pages,
kv_heads, head_dim, 64] signed bytes, k_scale and v_scale [pages, kv_heads, 4]
fp32, value = code * scale.  Rows of a call are tokens, those of sequence s
being offsets[s] .. offsets[s + 1] - 1, the last of the lengths[s] tokens the
sequence then has; token j of it lies in page pages[s, j // 64].
"""
import math

import torch

own = False

PAGE, BLOCK = 64, 16
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
# The smallest scale a block is given: codes of smaller values lose bits.
LEAST_SCALE = 2.0 ** -100


def cached(name, op, dtype, heads, kv, hd, seqs, new_lo, new_hi, old_lo, old_hi):
    """`seqs` sequences with old_lo .. old_hi tokens before the call and new_lo .. new_hi in it."""
    return {"name": name, "op": op, "dtype": dtype, "heads": heads, "kv": kv, "hd": hd, "seqs": seqs,
            "new_lo": new_lo, "new_hi": new_hi, "old_lo": old_lo, "old_hi": old_hi}


def linear(name, dtype, batch, cols, rows, bias):
    return {"name": name, "op": "linear", "dtype": dtype, "batch": batch, "cols": cols, "rows": rows, "bias": bias}


def listed():
    return [
        # The decoder's step for 64 users of the 1.5B model, each at another position of its 2048.
        cached("append step 64", "append", "f32", 12, 2, 128, 64, 1, 1, 0, 2047),
        # Prompts of many lengths arriving together, some behind a cached prefix, some sequences without a new token.
        cached("append prompts", "append", "bf16", 32, 8, 64, 24, 0, 511, 0, 1500),
        # Four long documents of an 8-KV-head model read in one pass.
        cached("append long", "append", "bf16", 32, 8, 128, 4, 4000, 4096, 0, 9),
        # One user of the 1B model at the end of the benchmark's generation.
        cached("step 1", "attention", "f32", 32, 8, 64, 1, 1, 1, 319, 319),
        # The decoder's step for 64 users of the 1.5B model, each at another position.
        cached("step 64", "attention", "f32", 12, 2, 128, 64, 1, 1, 0, 2047),
        # Long contexts of 32 users, one token each: the largest read of the cache.
        cached("step long", "attention", "bf16", 32, 8, 128, 32, 1, 1, 20000, 32767),
        # A prompt of the 1B model as the decoder passes it, in fp32.
        cached("prompt 383", "attention", "f32", 32, 8, 64, 1, 383, 383, 0, 0),
        # The second halves of two 8192-token documents.
        cached("prompt long", "attention", "bf16", 32, 8, 128, 2, 4096, 4096, 4000, 4096),
        # One token through the 1B model's fused gate|up.
        linear("linear 1", "f32", 1, 2048, 16384, False),
        # 48 tokens through the 1.5B model's down projection, with a bias.
        linear("linear 48", "f16", 48, 8960, 1536, True),
        # An odd number of rows and columns and a batch that fills no tile.
        linear("linear odd", "f32", 517, 1400, 3001, True),
        # A long prompt's tokens through the 1B model's fused gate|up.
        linear("linear 8192", "bf16", 8192, 2048, 16384, False),
    ]


def log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def most(op):
    """Work of the largest listed case of an operator."""
    w = [work(c) for c in listed() if c["op"] == op]
    return max(x["bytes"] for x in w), max(x["flops"] for x in w)


def draw(rng):
    while True:
        op = rng.choice(["append", "attention", "attention", "linear"])
        dtype = rng.choice(["f32", "bf16", "f16"])
        if op == "linear":
            c = linear("", dtype, log_uniform(rng, 1, 8192), log_uniform(rng, 100, 8960), log_uniform(rng, 250, 40000),
                       rng.random() < 0.5)
        else:
            kv = rng.choice([1, 2, 4, 8])
            heads, hd = kv * rng.choice([1, 2, 3, 4, 6, 8]), rng.choice([64, 128])
            if rng.random() < 0.5:   # steps: one token, now and then a few, for each sequence
                n = rng.choice([1, 1, 1, 2, 5])
                old = log_uniform(rng, 30, 32000)
                c = cached("", op, dtype, heads, kv, hd, log_uniform(rng, 1, 200), 1, n, old // rng.choice([1, 3, 30]), old)
            else:
                new = log_uniform(rng, 20, 6000)
                old = rng.choice([0, log_uniform(rng, 10, 4000)])
                c = cached("", op, dtype, heads, kv, hd, log_uniform(rng, 1, 40), new // rng.choice([1, 2, 20]), new, old // 3,
                           old)
        if op != "linear":
            new, old = tokens(c)
            if sum(new) == 0 or len(new) * max(new) * (max(new) + max(old) + PAGE) * heads > 1 << 31 or \
                    len(new) * (max(new) + max(old)) * kv * hd > 1 << 30:
                continue
        w, (b, f) = work(c), most(op)
        if w["bytes"] <= b and w["flops"] <= f:
            del c["name"]
            return c


def tokens(case):
    """Each sequence's new tokens and those before them."""
    n = case["seqs"]
    step = next(s for s in (37, 41, 43, 47, 53) if math.gcd(s, n) == 1 or n == 1)   # visits every rank once

    def spread(lo, hi, by):
        return [lo + (hi - lo) * ((i * by + n - 1) % n) // max(1, n - 1) if n > 1 else hi for i in range(n)]
    return spread(case["new_lo"], case["new_hi"], step), spread(case["old_lo"], case["old_hi"], step + 2 * n)


def work(case):
    e = SIZE[case["dtype"]]
    if case["op"] == "linear":
        m, k, n = case["batch"], case["cols"], case["rows"]
        return {"bytes": m * k * e + n * k + 4 * n + (e * n if case["bias"] else 0) + m * n * e, "flops": 2 * m * n * k}
    new, old = tokens(case)
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    rows = sum(new)
    if case["op"] == "append":
        blocks = sum(-(-(o + n) // BLOCK) - o // BLOCK for n, o in zip(new, old) if n)
        return {"bytes": rows * (2 * h + 2 * kv) * hd * e + rows * 2 * kv * hd + blocks * 2 * kv * 4 + rows * hd * 4,
                "flops": rows * (h + kv) * hd * 3 + rows * 2 * kv * hd * 3}
    length = sum(o + n for n, o in zip(new, old) if n)
    pairs = sum(n * o + n * (n + 1) // 2 for n, o in zip(new, old))
    return {"bytes": 2 * rows * h * hd * e + length * 2 * kv * hd + -(-length // BLOCK) * 2 * kv * 4,
            "flops": 4 * h * hd * pairs}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dt = DTYPES[case["dtype"]]

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    if case["op"] == "linear":
        m, k, n = case["batch"], case["cols"], case["rows"]
        x = normal(m, k)
        x[:, torch.randperm(k, generator=g, device="cuda")[: max(1, k // 200)]] *= 20.0   # the few far channels of real activations
        width = -(-k // 16) * 16   # weight rows start on 16 bytes
        w = (normal(n, width) * 32).round_().clamp_(-127, 127).to(torch.int8)[:, :k]
        return {"op": "linear", "x": x.to(dt), "w": w, "w_scale": 0.02 / 32 * (0.5 + torch.rand(n, generator=g, device="cuda")),
                "bias": normal(n).mul_(0.1).to(dt) if case["bias"] else None}
    new, old = tokens(case)
    h, kv, hd = case["heads"], case["kv"], case["hd"]
    lengths = [o + n for n, o in zip(new, old)]
    width = max(1, -(-max(lengths) // PAGE))
    pool = sum(-(-l // PAGE) for l in lengths) + 3
    order = torch.randperm(pool, generator=g, device="cuda").to(torch.int32)
    pages = torch.full((len(new), width), -1, dtype=torch.int32)
    at = 0
    order = order.cpu()
    for s, l in enumerate(lengths):
        n = -(-l // PAGE)
        pages[s, :n] = order[at:at + n]
        at += n
    rows = sum(new)
    offsets = torch.tensor([sum(new[:s]) for s in range(len(new) + 1)], dtype=torch.int32)

    def scales():
        return 0.03 * torch.exp(0.3 * normal(pool, kv, PAGE // BLOCK))

    def codes(*shape):
        return (normal(*shape) * 32).round_().clamp_(-127, 127).to(torch.int8)
    s = {"op": case["op"], "q": normal(rows, h, hd).to(dt), "offsets": offsets.cuda(),
         "lengths": torch.tensor(lengths, dtype=torch.int32, device="cuda"), "pages": pages.cuda(), "most_new": max(new),
         "cache_k": codes(pool, kv, PAGE, hd), "cache_v": codes(pool, kv, hd, PAGE), "k_scale": scales(), "v_scale": scales()}
    if case["op"] == "append":
        angle = torch.arange(max(1, max(lengths)), dtype=torch.float64)[:, None] * \
            500000.0 ** (-torch.arange(hd // 2, dtype=torch.float64) / (hd // 2))
        s["rope"] = torch.stack([angle.cos(), angle.sin()], -1).float().cuda()   # [position, pair, (cos, sin)]
        loud = 1 + 7 * (torch.rand(kv, hd, generator=g, device="cuda") < 0.04)     # keys have a few loud channels
        s["k"], s["v"] = (normal(rows, kv, hd) * loud).to(dt), normal(rows, kv, hd).to(dt)
    return s


def run(s):
    if own:
        if s["op"] == "linear":
            import lutmac_amd as L
            return L.linear_i8(s["x"], s["w"], s["w_scale"], bias=s["bias"])
        from lutmac_amd.kv8 import KvCache8
        cache = KvCache8(s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"])
        if s["op"] == "append":
            q = cache.append(s["k"], s["v"], s["offsets"], s["lengths"], s["pages"], rope=s["rope"], q=s["q"])
            return q, s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"]
        return cache.attend(s["q"], s["offsets"], s["lengths"], s["pages"])
    return {"linear": plain_linear, "append": plain_append, "attention": plain_attention}[s["op"]](s)


# ---- the plain forms -------------------------------------------------------

def plain_linear(s):
    x = s["x"].double()
    most = x.abs().amax(1, keepdim=True)
    codes = (x * 127.0 / most.clamp_min(1e-300)).round()   # to the even one of two equally near; 64 bits: borders
    y = codes.float() @ s["w"].float().t()
    y = y * (most / 127.0).float() * s["w_scale"]
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def rotated(x, rope, at):
    """Pairs (d, d + hd / 2) of x [rows, heads, hd] rotated by their positions' angles, in 64 bits."""
    c, n = rope[at].double().unbind(-1)
    a, b = x.double().chunk(2, -1)
    c, n = c[:, None], n[:, None]
    return torch.cat([a * c - b * n, a * n + b * c], -1)


def rows_of(s):
    """Each row's sequence and its position in it."""
    off, n = s["offsets"].long(), s["q"].shape[0]
    row = torch.arange(n, device="cuda")
    seq = torch.searchsorted(off[1:].contiguous(), row, right=True)
    return seq, s["lengths"].long()[seq] - off[seq + 1] + row


def plain_append(s):
    seq, at = rows_of(s)
    page, slot = s["pages"].long()[seq, at // PAGE], at % PAGE
    pool, kv = s["k_scale"].shape[:2]
    block = page * 4 + slot // BLOCK
    # the block that each sequence begins in, and how many of its tokens stay
    count = (s["offsets"][1:] - s["offsets"][:-1]).long()
    start = s["lengths"].long() - count
    kept = torch.where(count > 0, start % BLOCK, 0)
    first = s["pages"].long().gather(1, (start // PAGE).clamp(max=s["pages"].shape[1] - 1)[:, None])[:, 0] * 4 + start % PAGE // BLOCK
    has = kept > 0
    first = first.clamp_min(0)

    def scales(x, scale):
        """New scales of every block that the rows touch; the factor of the kept codes."""
        top = torch.zeros(pool * 4, kv, dtype=torch.float64, device="cuda")
        top.scatter_reduce_(0, block[:, None].expand(-1, kv), x.abs().amax(-1), "amax")
        flat = scale.transpose(1, 2).reshape(pool * 4, kv)   # [page, block] by head
        before = torch.zeros_like(flat).index_put_((first,), torch.where(has[:, None], flat[first], 0), accumulate=True)
        touched = torch.zeros(pool * 4, dtype=torch.bool, device="cuda").index_fill_(0, block, True)
        fresh = torch.maximum((top / 127.0).float(), before).clamp_min(LEAST_SCALE)
        after = torch.where(touched[:, None], fresh, flat)
        was = flat[first]
        scale.copy_(after.view(pool, 4, kv).transpose(1, 2))
        return after, was

    k, v = rotated(s["k"], s["rope"], at), s["v"].double()
    inside = torch.arange(BLOCK, device="cuda")
    stays = has[:, None] & (inside < kept[:, None])   # [sequence, token of its first block]
    fp, fs = (first // 4)[:, None].expand(-1, BLOCK), (first % 4 * BLOCK)[:, None] + inside
    fp, fs = fp[stays], fs[stays]
    owner = torch.arange(len(kept), device="cuda")[:, None].expand(-1, BLOCK)[stays]
    for codes, scale, x, values_last in ((s["cache_k"], s["k_scale"], k, True), (s["cache_v"], s["v_scale"], v, False)):
        after, was = scales(x, scale)
        view = codes if values_last else codes.transpose(2, 3)   # [page, head, token, dim]
        old = view[fp, :, fs].double() * was[owner].double()[:, :, None] / after[first][owner].double()[:, :, None]
        view[fp, :, fs] = old.round().to(torch.int8)
        view[page, :, slot] = (x / after[block].double()[:, :, None]).round().to(torch.int8)
    return rotated(s["q"], s["rope"], at).to(s["q"].dtype), s["cache_k"], s["cache_v"], s["k_scale"], s["v_scale"]


def plain_attention(s):
    q, off, length = s["q"], s["offsets"].long(), s["lengths"].long()
    rows, h, hd = q.shape
    kv = s["cache_k"].shape[1]
    n, width, most = len(length), s["pages"].shape[1], s["most_new"]
    page = s["pages"].long().clamp_min(0)
    k = s["cache_k"][page].float() * s["k_scale"][page].repeat_interleave(BLOCK, -1)[..., None]       # [n, width, kv, 64, hd]
    v = s["cache_v"][page].float() * s["v_scale"][page].repeat_interleave(BLOCK, -1)[:, :, :, None]   # [n, width, kv, hd, 64]
    k = k.transpose(1, 2).reshape(n, kv, width * PAGE, hd)
    v = v.permute(0, 2, 1, 4, 3).reshape(n, kv, width * PAGE, hd)
    t = torch.arange(most, device="cuda")
    count = off[1:] - off[:-1]
    pick = (off[:-1, None] + t).clamp(max=rows - 1)
    qs = q[pick].float().view(n, most, kv, h // kv, hd).permute(0, 2, 3, 1, 4).reshape(n, kv, h // kv * most, hd)
    score = (qs @ k.transpose(2, 3)).view(n, kv, h // kv, most, width * PAGE) * (1.0 / math.sqrt(hd))
    last = (length - count)[:, None] + t   # the position of each query
    hidden = torch.arange(width * PAGE, device="cuda") > torch.minimum(last, length[:, None] - 1)[:, :, None]
    score = score.masked_fill_(hidden[:, None, None], -math.inf)
    score = (score - score.amax(-1, keepdim=True)).exp_()
    out = (score.view(n, kv, h // kv * most, width * PAGE) @ v).view(n, kv, h // kv, most, hd)
    out = out / score.sum(-1, keepdim=True)
    seq, at = rows_of(s)
    return out.permute(0, 3, 1, 2, 4)[seq, at - (length - count)[seq]].reshape(rows, h, hd).to(q.dtype)


# ---- the definitions in 64 bits --------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": exact_linear, "append": exact_append, "attention": exact_attention}[case["op"]](s)


def exact_linear(s):
    x, w = s["x"].double(), s["w"].double()
    out = []
    for part in x.split(1024):
        top = part.abs().max(1).values
        codes = torch.where(top[:, None] > 0, torch.round(part * 127 / top[:, None]), 0.0)
        y = torch.matmul(codes, w.T) * torch.outer(top / 127, s["w_scale"].double())
        out.append(y if s["bias"] is None else y + s["bias"].double())
    return torch.cat(out)


def exact_append(s):
    q = torch.empty(s["q"].shape, dtype=torch.float64, device="cuda")
    cache = {n: s[n].clone() for n in ("cache_k", "cache_v")}
    scale = {n: s[n].double() for n in ("k_scale", "v_scale")}
    off, lengths, pages = s["offsets"].tolist(), s["lengths"].tolist(), s["pages"].tolist()
    turn = torch.complex(s["rope"][..., 0].double(), s["rope"][..., 1].double())
    half = s["q"].shape[-1] // 2

    def turned(x, lo):
        z = torch.complex(x[..., :half].double(), x[..., half:].double()) * turn[lo:lo + x.shape[0], None]
        return torch.cat([z.real, z.imag], -1)
    for i, length in enumerate(lengths):
        a, b = off[i], off[i + 1]
        if a == b:
            continue
        lo = length - (b - a)
        q[a:b] = turned(s["q"][a:b], lo)
        values = {"cache_k": turned(s["k"][a:b], lo), "cache_v": s["v"][a:b].double()}
        for start in range(lo // BLOCK * BLOCK, length, BLOCK):
            page, part = pages[i][start // PAGE], start % PAGE // BLOCK
            kept = max(0, lo - start)
            fresh = slice(max(0, start - lo), min(length, start + BLOCK) - lo)
            for name, which in (("cache_k", "k_scale"), ("cache_v", "v_scale")):
                x = values[name][fresh].transpose(0, 1)   # [head, token, dim]
                codes = cache[name][page] if name == "cache_k" else cache[name][page].transpose(1, 2)
                codes = codes[:, part * BLOCK:(part + 1) * BLOCK]
                was = scale[which][page, :, part].clone()
                now = x.abs().flatten(1).max(1).values / 127
                now = now.float().double()   # the scale is an fp32 number by definition
                if kept:
                    now = torch.maximum(now, was)
                now = now.clamp(min=LEAST_SCALE)
                if kept:
                    codes[:, :kept] = torch.round(codes[:, :kept].double() * was[:, None, None] / now[:, None, None]).to(torch.int8)
                codes[:, kept:kept + x.shape[1]] = torch.round(x / now[:, None, None]).to(torch.int8)
                scale[which][page, :, part] = now
    return q, cache["cache_k"], cache["cache_v"], scale["k_scale"], scale["v_scale"]


def exact_attention(s):
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    h, hd = s["q"].shape[1:]
    kv = s["cache_k"].shape[1]
    off, lengths = s["offsets"].tolist(), s["lengths"].tolist()
    for i, length in enumerate(lengths):
        a, b = off[i], off[i + 1]
        if a == b:
            continue
        page = s["pages"][i, : -(-length // PAGE)].long()
        for head in range(kv):
            block = torch.arange(length, device="cuda") % PAGE // BLOCK
            at = torch.arange(length, device="cuda") // PAGE
            ks, vs = (s[n][page, head][at, block].double() for n in ("k_scale", "v_scale"))
            k = s["cache_k"][page, head].flatten(0, 1)[:length].double() * ks[:, None]
            v = s["cache_v"][page, head].transpose(1, 2).flatten(0, 1)[:length].double() * vs[:, None]
            mine = slice(head * (h // kv), (head + 1) * (h // kv))
            x = s["q"][a:b, mine].double().transpose(0, 1)   # [group, row, dim]
            see = torch.arange(length, device="cuda") <= torch.arange(length - (b - a), length, device="cuda")[:, None]
            p = torch.softmax(torch.where(see, torch.matmul(x, k.T) / hd ** 0.5, -math.inf), -1)
            out[a:b, mine] = torch.matmul(p, v).transpose(0, 1)
    return out
