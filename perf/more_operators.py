"""A serving step that checks drafted tokens: its operators' calls, and what they compute in plain torch.

*pages*: rows of a step are granted and given their places in a paged cache --
offsets, positions, slots, new pages from a stack of free ones -- and taken
back again.

*rotary*: queries and keys turned to their positions; pairs a half head apart or
side by side, the whole head or its first dimensions.

*linear*: a linear layer in 8-bit floating point (e4m3), weights with one scale
per block of 128 x 128, activations with one, a power of two, per row and 128
columns.

*verify*: drafted tokens accepted or replaced so that what comes out is
distributed as the target's own tokens are, from given random numbers.

Rows of sequence s are offsets[s] .. offsets[s + 1] - 1.
"""
import math

import torch

own = False

PAGE, BLOCK = 64, 128
DTYPES = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
SIZE = {"f32": 4, "f16": 2, "bf16": 2}
E4M3_MOST = 448.0
LEAST_EXPONENT = -126   # of an activation scale


def linear(name, dtype, batch, cols, rows, bias):
    return {"name": name, "op": "linear", "dtype": dtype, "batch": batch, "cols": cols, "rows": rows, "bias": bias}


def verify(name, dtype, seqs, least, most, vocab, probs, temperature):
    """`seqs` sequences of least .. most drafted tokens each; temperature below 0: 0, 0.7 and 1 in turn."""
    return {"name": name, "op": "verify", "dtype": dtype, "seqs": seqs, "least": least, "most": most, "vocab": vocab,
            "probs": probs, "temperature": temperature}


def paged(name, seqs, new_lo, new_hi, old, share):
    """`seqs` sequences of 0 .. old tokens that get new_lo .. new_hi; the free pages are `share` of what that takes."""
    return {"name": name, "op": "pages", "seqs": seqs, "new_lo": new_lo, "new_hi": new_hi, "old": old, "share": share}


def turned(name, dtype, rows, heads, kv, hd, rd, interleaved, positions):
    return {"name": name, "op": "rotary", "dtype": dtype, "rows": rows, "heads": heads, "kv": kv, "hd": hd, "rd": rd,
            "interleaved": interleaved, "positions": positions}


def listed():
    return [
        # One token through the 1B model's fused gate|up.
        linear("linear 1", "bf16", 1, 2048, 16384, False),
        # 48 tokens through the 1.5B model's down projection, with a bias.
        linear("linear 48", "f16", 48, 8960, 1536, True),
        # An odd number of rows and columns and a batch that fills no tile, in fp32.
        linear("linear odd", "f32", 517, 1400, 3001, True),
        # A long prompt's tokens through the 1B model's fused gate|up.
        linear("linear 8192", "bf16", 8192, 2048, 16384, False),
        # One user of the 1B model; drafts looked up in the text, so that nothing is known of their probabilities.
        verify("verify 1", "f32", 1, 4, 4, 128256, False, 0.7),
        # 64 users of the 1.5B model, drafts of a smaller model with its probabilities.
        verify("verify 64", "bf16", 64, 0, 7, 151936, True, 1.0),
        # A few users of a small vocabulary, greedy and sampled ones together.
        verify("verify odd", "f16", 9, 1, 3, 32003, True, -1.0),
        # The step of 64 users, each with one token and up to 4 drafts.
        paged("pages 64", 64, 1, 5, 2047, 1.5),
        # Prompts of 1000 users arriving together, more than the free pages hold.
        paged("pages prompts", 1000, 0, 4000, 500, 0.98),
        # The step of 64 users of the 1.5B model.
        turned("rotary 64", "f32", 64, 12, 2, 128, 128, False, 2048),
        # A long prompt of an 8-KV-head model whose pairs lie side by side.
        turned("rotary long", "bf16", 16384, 32, 8, 128, 128, True, 131072),
        # Heads of 80 of which 32 turn.
        turned("rotary part", "f16", 2051, 32, 32, 80, 32, False, 8192),
    ]


def log_uniform(rng, lo, hi):
    return min(hi, max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    while True:
        op = rng.choice(["linear", "linear", "verify", "verify", "pages", "rotary"])
        dtype = rng.choice(["f32", "bf16", "f16"])
        if op == "linear":
            c = linear("", dtype, log_uniform(rng, 1, 8192), log_uniform(rng, 100, 8960), log_uniform(rng, 250, 40000),
                       rng.random() < 0.5)
        elif op == "verify":
            most = rng.randint(0, 8)
            c = verify("", dtype, log_uniform(rng, 1, 80), rng.randint(0, most), most, log_uniform(rng, 2000, 152000),
                       rng.random() < 0.6, rng.choice([-1.0, 0.0, 0.6, 1.0, 1.0]))
        elif op == "pages":
            hi = rng.choice([1, rng.randint(2, 9), log_uniform(rng, 10, 6000)])
            c = paged("", log_uniform(rng, 1, 2000), hi // rng.choice([1, 3, 30]), hi, log_uniform(rng, 1, 4000),
                      rng.choice([1.1, 1.5, 0.9]))
        else:
            hd = rng.choice([64, 80, 96, 128, 256])
            kv = rng.choice([1, 2, 4, 8, 16])
            c = turned("", dtype, log_uniform(rng, 1, 20000), kv * rng.choice([1, 2, 3, 4, 8]), kv, hd,
                       rng.choice([hd, hd, hd // 2, 32]), rng.random() < 0.5, log_uniform(rng, 100, 131072))
        w = work(c)
        most = [work(x) for x in listed() if x["op"] == op]
        if w["bytes"] <= max(x["bytes"] for x in most) and w["flops"] <= max(x["flops"] for x in most):
            del c["name"]
            return c


def spread(lo, hi, n, by):
    """n numbers from lo to hi, in an order that looks like none."""
    step = next(s for s in (37, 41, 43, 47, 53) if math.gcd(s, n) == 1 or n == 1) + by * n
    return [lo + (hi - lo) * ((i * step + n - 1) % n) // max(1, n - 1) if n > 1 else hi for i in range(n)]


def pages_of(tokens):
    return -(-tokens // PAGE)


def work(case):
    op = case["op"]
    if op == "linear":
        e, m, k, n = SIZE[case["dtype"]], case["batch"], case["cols"], case["rows"]
        return {"bytes": m * k * e + n * k + 4 * -(-n // BLOCK) * -(-k // BLOCK) + (e * n if case["bias"] else 0) + m * n * e,
                "flops": 2 * m * n * k}
    if op == "verify":
        n = case["seqs"]
        rows = n + sum(spread(case["least"], case["most"], n, 0))
        # every row's logits; the draft's probabilities of one row of each sequence
        return {"bytes": rows * case["vocab"] * SIZE[case["dtype"]] + (4 * n * case["vocab"] if case["probs"] else 0) + 16 * rows,
                "flops": 3 * rows * case["vocab"]}
    if op == "pages":
        new = spread(case["new_lo"], case["new_hi"], case["seqs"], 0)
        # counts in and out twice; a position and a slot a row; new pages into the table, and back
        return {"bytes": 28 * case["seqs"] + 12 * sum(new) + 16 * sum(pages_of(n) for n in new), "flops": sum(new)}
    rows, heads = case["rows"], case["heads"] + case["kv"]
    return {"bytes": 2 * rows * heads * case["hd"] * SIZE[case["dtype"]] + rows * (4 * case["rd"] + 4),
            "flops": 3 * rows * heads * case["rd"]}


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)

    def normal(*shape):
        return torch.randn(*shape, generator=g, device="cuda")
    return {"linear": prepare_linear, "verify": prepare_verify, "pages": prepare_pages, "rotary": prepare_rotary}[case["op"]](case, g, normal)


def prepare_linear(case, g, normal):
    dt, m, k, n = DTYPES[case["dtype"]], case["batch"], case["cols"], case["rows"]
    x = normal(m, k)
    x[:, torch.randperm(k, generator=g, device="cuda")[: max(1, k // 200)]] *= 20.0   # the few far channels of real activations
    width = -(-k // 16) * 16   # weight rows start on 16 bytes
    w = (normal(n, width) * 100).clamp_(-E4M3_MOST, E4M3_MOST).to(torch.float8_e4m3fn)[:, :k]
    scale = 0.02 / 100 * torch.exp(0.3 * normal(-(-n // BLOCK), -(-k // BLOCK)))
    return {"op": "linear", "x": x.to(dt), "w": w, "w_scale": scale, "bias": normal(n).mul_(0.1).to(dt) if case["bias"] else None}


def prepare_verify(case, g, normal):
    n, vocab = case["seqs"], case["vocab"]
    drafts = spread(case["least"], case["most"], n, 0)
    rows = n + sum(drafts)
    logits = (normal(rows, vocab) * 2.5).to(DTYPES[case["dtype"]])
    logits[:, :: 1000] += 4   # the words that come up everywhere
    t = [case["temperature"] if case["temperature"] >= 0 else (0.0, 0.7, 1.0)[i % 3] for i in range(n)]
    offsets = torch.tensor([sum(drafts[:i]) + i for i in range(n + 1)], dtype=torch.int32, device="cuda")
    # the draft's distribution: the target's with an error
    near = logits.float() + 0.6 * normal(rows, vocab)
    probs = torch.softmax(near, -1)
    race = torch.rand(rows, vocab, generator=g, device="cuda").clamp_(1e-30).log_().neg_()
    token = (probs / race).argmax(-1)   # a sample of it
    cold = torch.tensor([v == 0 for v in t], device="cuda").repeat_interleave((offsets[1:] - offsets[:-1]).long())
    token = torch.where(cold, near.argmax(-1), token).to(torch.int32)
    return {"op": "verify", "logits": logits, "drafts": token, "offsets": offsets, "probs": probs if case["probs"] else None,
            "uniforms": torch.rand(rows, 2, generator=g, device="cuda"),
            "temperature": torch.tensor(t, dtype=torch.float32, device="cuda")}


def prepare_pages(case, g, normal):
    n = case["seqs"]
    new, old = spread(case["new_lo"], case["new_hi"], n, 0), spread(0, case["old"], n, 2)
    width = max(1, max(pages_of(a + b) for a, b in zip(new, old)))
    held, needs = sum(pages_of(o) for o in old), sum(pages_of(a + b) - pages_of(b) for a, b in zip(new, old))
    free = max(1, int(needs * case["share"]))
    order = torch.randperm(held + free, generator=g, device="cuda").to(torch.int32)
    shuffle = torch.randperm(n, generator=g, device="cuda")   # who comes with how many
    new, old = torch.tensor(new, dtype=torch.int32, device="cuda")[shuffle], torch.tensor(old, dtype=torch.int32, device="cuda")
    has = torch.arange(width, device="cuda") < ((old + PAGE - 1) // PAGE)[:, None]
    pages = torch.full((n, width), -1, dtype=torch.int32, device="cuda")
    pages[has] = order[:held]
    stack = torch.cat([order[held:], torch.full((held,), -1, dtype=torch.int32, device="cuda")])
    rows = int(case["new_hi"] * n)   # what the program makes room for
    return {"op": "pages", "new": new, "lengths": old, "pages": pages, "free": stack,
            "n_free": torch.tensor([free], dtype=torch.int32, device="cuda"),
            "positions": torch.full((rows,), -1, dtype=torch.int32, device="cuda"),
            "slots": torch.full((rows,), -1, dtype=torch.int64, device="cuda")}


def prepare_rotary(case, g, normal):
    dt, rows, hd, rd = DTYPES[case["dtype"]], case["rows"], case["hd"], case["rd"]
    angle = torch.arange(case["positions"], dtype=torch.float64, device="cuda")[:, None] * \
        500000.0 ** (-torch.arange(rd // 2, dtype=torch.float64, device="cuda") / (rd // 2))
    return {"op": "rotary", "q": normal(rows, case["heads"], hd).to(dt), "k": normal(rows, case["kv"], hd).to(dt),
            "rope": torch.stack([angle.cos(), angle.sin()], -1).float(), "interleaved": case["interleaved"],
            "positions": torch.randint(0, case["positions"], (rows,), generator=g, device="cuda", dtype=torch.int32)}


def run(s):
    if own:
        import lutmac_amd as L
        if s["op"] == "linear":
            return L.linear_f8(s["x"], s["w"], s["w_scale"], bias=s["bias"])
        if s["op"] == "verify":
            return L.verify_drafts(s["logits"], s["drafts"], s["offsets"], s["uniforms"], probs=s["probs"],
                                   temperature=s["temperature"])
        from lutmac_amd import kv8
        if s["op"] == "rotary":
            return kv8.rotate(s["q"], s["k"], s["positions"], s["rope"], interleaved=s["interleaved"])
        held = kv8.KvPages(s["pages"], s["lengths"], s["free"], s["n_free"])
        offsets, granted, positions, slots = held.extend(s["new"], s["positions"], s["slots"])
        held.trim(granted)   # (all drafts rejected: the next pass finds what this one found)
        return offsets, granted, positions, slots, s["pages"], s["lengths"], s["free"], s["n_free"]
    return {"linear": plain_linear, "verify": plain_verify, "pages": plain_pages, "rotary": plain_rotary}[s["op"]](s)


# ---- the plain forms -------------------------------------------------------

def power_of_two(e):
    """2^e in fp32, exactly (a power function may be off in its last bit)."""
    return ((e + 127) << 23).view(torch.float32)


def plain_linear(s):
    x, w, scale = s["x"].float(), s["w"].float(), s["w_scale"]
    m, k, n = x.shape[0], x.shape[1], w.shape[0]
    blocks = -(-k // BLOCK)
    x = torch.nn.functional.pad(x, (0, blocks * BLOCK - k)).view(m, blocks, BLOCK)
    top = x.abs().amax(-1, keepdim=True)
    half, e = torch.frexp(top)                       # top = half * 2^e, half in [0.5, 1)
    e = (e - 9 + (half > E4M3_MOST / 512).int()).clamp_min(LEAST_EXPONENT)   # the least with top <= 448 * 2^e
    e = torch.where(top > 0, e, LEAST_EXPONENT).int()
    code = (x * power_of_two(-e)).to(torch.float8_e4m3fn).float()
    x = (code * power_of_two(e)).view(m, blocks * BLOCK)[:, :k]
    w = w * scale.repeat_interleave(BLOCK, 0)[:n].repeat_interleave(BLOCK, 1)[:, :k]
    y = x @ w.t()
    if s["bias"] is not None:
        y = y + s["bias"].float()
    return y.to(s["x"].dtype)


def plain_rotary(s):
    c, n = s["rope"][s["positions"].long()][:, None].unbind(-1)   # [rows, 1, pairs]
    rd = 2 * c.shape[-1]

    def turn(x):
        y = x[..., :rd].float()
        if s["interleaved"]:
            a, b = y[..., 0::2], y[..., 1::2]
            y = torch.stack([a * c - b * n, a * n + b * c], -1).flatten(-2)
        else:
            a, b = y.chunk(2, -1)
            y = torch.cat([a * c - b * n, a * n + b * c], -1)
        return torch.cat([y.to(x.dtype), x[..., rd:]], -1)
    return turn(s["q"]), turn(s["k"])


def plain_pages(s):
    pages, lengths, free, n_free = s["pages"], s["lengths"], s["free"], s["n_free"]
    room, width, most = s["positions"].shape[0], pages.shape[1], free.shape[0]
    new, old, have = s["new"].long().clamp_min(0), lengths.long(), n_free.long()
    fits = (new > 0) & (old + new <= width * PAGE)
    new = torch.where(fits, new, 0)
    need = (old + new + PAGE - 1) // PAGE - (old + PAGE - 1) // PAGE
    taken = need.cumsum(0)
    granted = torch.where((new.cumsum(0) <= room) & ((need == 0) | (taken <= have)), new, 0)
    given = torch.where(granted > 0, need, 0)
    ends = granted.cumsum(0)
    offsets = torch.cat([torch.zeros_like(ends[:1]), ends])
    # the new pages, from the top of the stack in the order of the sequences
    at = torch.arange(width, device="cuda")
    first = (old + PAGE - 1) // PAGE
    fresh = (at >= first[:, None]) & (at < (first + given)[:, None])
    place = have - 1 - ((taken - need)[:, None] + at - first[:, None])
    table = torch.where(fresh, free.long()[place.clamp(0, most - 1)], pages.long())
    # every row's position and slot
    row = torch.arange(room, device="cuda")
    seq = torch.searchsorted(ends, row, right=True)
    inside = seq < len(ends)
    seq = seq.clamp_max(len(ends) - 1)
    position = old[seq] + row - offsets[seq]
    slot = table[seq, (position // PAGE).clamp(0, width - 1)] * PAGE + position % PAGE
    s["positions"].copy_(torch.where(inside, position, s["positions"].long()))
    s["slots"].copy_(torch.where(inside, slot, s["slots"]))
    have = have - given.sum()
    # and back: the same tokens dropped, their pages pushed so that the first of the first sequence is on top
    length = old + granted
    drop = granted
    keep = (length - drop).clamp_min(0)
    last, kept = (length + PAGE - 1) // PAGE, (keep + PAGE - 1) // PAGE
    gone = (at >= kept[:, None]) & (at < last[:, None])
    count = last - kept
    total = count.sum()
    place = have + total - 1 - ((count.cumsum(0) - count)[:, None] + at - kept[:, None])
    stack = torch.cat([free, free[:1]])   # (its last place takes what is no page)
    stack.scatter_(0, torch.where(gone, place, most).flatten(), table.flatten().to(free.dtype))
    free.copy_(stack[:most])
    pages.copy_(torch.where(gone, -1, table))
    lengths.copy_(keep)
    n_free.copy_(have + total)
    i32 = torch.int32
    return offsets.to(i32), granted.to(i32), s["positions"], s["slots"], pages, lengths, free, n_free


def plain_verify(s):
    # (in 64 bits: a token is chosen by which side of a border a number lies)
    logits, off = s["logits"].double(), s["offsets"].long()
    rows, vocab = logits.shape
    n = len(off) - 1
    row = torch.arange(rows, device="cuda")
    seq = torch.searchsorted(off[1:].contiguous(), row, right=True)
    t = s["temperature"].double()[seq][:, None]
    top, best = logits.max(-1, keepdim=True)
    best = (logits == top).int().argmax(-1, keepdim=True)   # the first of equals
    weight = torch.exp((logits - top) / torch.where(t > 0, t, 1.0))
    greedy = torch.zeros_like(weight).scatter_(1, best, 1.0)
    weight = torch.where(t > 0, weight, greedy)
    total = weight.sum(-1)
    token = s["drafts"].long()
    known = (token >= 0) & (token < vocab)
    token = token.clamp(0, vocab - 1)[:, None]
    probs = s["probs"]
    q = probs.double().gather(1, token)[:, 0] if probs is not None else torch.ones_like(total)
    yes = known & (s["uniforms"][:, 0].double() * q * total < weight.gather(1, token)[:, 0])
    last = off[1:] - 1
    yes[last] = False   # (nothing drafted there)
    stop = torch.full((n,), rows, device="cuda").scatter_reduce_(0, seq, torch.where(yes, rows, row), "amin")
    accepted = stop - off[:-1]
    # the token of the row where each sequence stops
    w, all_ = weight[stop], total[stop][:, None]
    drawn = (stop < last)[:, None] & known[stop][:, None]
    if probs is not None:
        rest = (w - probs[stop].double() * all_).clamp_min(0.0)
        rest = torch.where((stop < last)[:, None], rest, w)
    else:
        rest = torch.where(drawn & (torch.arange(vocab, device="cuda") == token[stop]), 0.0, w)
    rest = torch.where(rest.sum(-1, keepdim=True) > 0, rest, w)
    sums = rest.cumsum(-1)
    pick = (sums > s["uniforms"][stop, 1:2].double() * sums[:, -1:]).int().argmax(-1)
    out = torch.where(row < stop[seq], s["drafts"].long(), torch.where(row == stop[seq], pick[seq], -1))
    return accepted.to(torch.int32), out.to(torch.int32)


# ---- the definitions in 64 bits --------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"linear": exact_linear, "verify": exact_verify, "pages": lambda s: None, "rotary": exact_rotary}[case["op"]](s)


def exact_power(e):
    return (e + 1023 << 52).view(torch.float64)


def exact_linear(s):
    x, w, scale = s["x"].double(), s["w"].float().double(), s["w_scale"].double()
    out = []
    for part in x.split(2048):
        y = torch.zeros(part.shape[0], w.shape[0], dtype=torch.float64, device="cuda")
        for b in range(scale.shape[1]):
            cols = slice(b * BLOCK, min((b + 1) * BLOCK, x.shape[1]))
            block = part[:, cols]
            top = block.abs().max(1).values
            least = torch.full_like(top, LEAST_EXPONENT, dtype=torch.int64)
            for e in range(LEAST_EXPONENT, 120):
                least += (top > E4M3_MOST * 2.0 ** e).long()
            unit = exact_power(least)[:, None]
            value = block / unit
            # e4m3: 4 bits from the first on, down to 2^-9
            bits = value.abs().clamp_min(2.0 ** -6).view(torch.int64) >> 52
            step = exact_power(bits - 1023 - 3)
            value = torch.round(value / step) * step * unit
            rows = scale[:, b].repeat_interleave(BLOCK)[: w.shape[0]]
            y += torch.matmul(value, w[:, cols].T.contiguous()) * rows
        out.append(y if s["bias"] is None else y + s["bias"].double())
    return torch.cat(out)


def exact_rotary(s):
    turn = torch.complex(s["rope"][..., 0].double(), s["rope"][..., 1].double())[s["positions"].long()][:, None]
    half = turn.shape[-1]
    got = []
    for x in (s["q"], s["k"]):
        y = x.double()
        step = 1 if s["interleaved"] else half
        i = torch.arange(half, device="cuda") * (2 if s["interleaved"] else 1)
        z = torch.complex(y[..., i], y[..., i + step]) * turn
        y[..., i], y[..., i + step] = z.real, z.imag
        got.append(y)
    return tuple(got)


def exact_verify(s):
    off, drafts = s["offsets"].tolist(), s["drafts"].tolist()
    accepted, out = [], [-1] * len(drafts)
    for i, t in enumerate(s["temperature"].tolist()):
        at = off[i]
        while True:
            x = s["logits"][at].double()
            p = torch.softmax(x / t, 0) if t > 0 else (torch.arange(len(x), device="cuda") == torch.nonzero(x == x.max())[0]).double()
            if at == off[i + 1] - 1:
                break
            q = s["probs"][at].double() if s["probs"] is not None else (torch.arange(len(x), device="cuda") == drafts[at]).double()
            if not float(s["uniforms"][at, 0].double() * q[drafts[at]]) < float(p[drafts[at]]):
                rest = torch.relu(p - q)
                p = rest if float(rest.sum()) > 0 else p
                break
            out[at] = drafts[at]
            at += 1
        upto = torch.cumsum(p, 0)
        out[at] = int(torch.searchsorted(upto, s["uniforms"][at, 1].double() * upto[-1], right=True))
        accepted.append(at - off[i])
    return torch.tensor(accepted, dtype=torch.int32, device="cuda"), torch.tensor(out, dtype=torch.int32, device="cuda")
