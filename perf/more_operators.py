"""Performance cases of what keeps long contexts cheap in a paged cache: keys and
values held in 4 bits, and attention over the pages that a cheap score selects.

A case is a plain dict.  Its "op" says what one pass does:

  append    rotate q and k of every new token, write k and v into a 4-bit cache
  attend    attention of every new token over its sequence's 4-bit pages
  bounds    bring the keys' bounds of the pages that new tokens are in up to date
  select    the pages that each new token is to read, for each kv head, by the bounds
  selected  attention of every new token over its selected pages

"batch" sequences bring "q" new tokens each.  They hold "kv" tokens with the new ones,
or with "ragged" between one eighth of that and all of it.  "window" > 0: a token sees
that many positions, its own included, and pages wholly before the first window are
not in the table any more (-1), as in a server that has freed them.  "count": pages
that a token reads, the sequence's first and the last two it sees always among them.
"""
import math

import torch

own = False

THETA = 10000.0
FIRST, LAST = 1, 2  # pages that are always selected


def _case(name, op, **kw):
    c = {"name": name, "op": op, "batch": 1, "q": 1, "kv": 1, "ragged": False, "heads": 32,
         "kv_heads": 8, "dim": 128, "page": 64, "cache": "fp4", "window": 0, "count": 0}
    if op == "append":
        c.update({"rot": kw.get("dim", 128), "style": "halves"})
    c.update(kw)
    return c


def listed():
    return [
        # A serving step of 64 sequences.
        _case("append_decode_batch", "append", batch=64, kv=4096, ragged=True, page=16, window=1),
        # A prompt of ordinary length.
        _case("append_prompt", "append", q=2048, kv=2048),
        # One token of a 1.1B model (TinyLlama's heads) in a chat of some hundred tokens.
        _case("attend_one_short", "attend", kv=700, kv_heads=4, dim=64),
        # One token over a very long context.
        _case("attend_one_long", "attend", kv=131072),
        # A serving step: 64 sequences of all lengths.
        _case("attend_batch", "attend", batch=64, kv=8192, ragged=True, page=32),
        # The next chunk of a long prompt.
        _case("attend_chunk", "attend", q=512, kv=16384),
        # A serving step of long contexts: the smallest call there is for 64 sequences.
        _case("bounds_decode", "bounds", batch=64, kv=16384, ragged=True, cache="fp16"),
        # After a long prompt: all of its pages.
        _case("bounds_prompt", "bounds", q=8192, kv=8192),
        # One token over a very long context.
        _case("select_one_long", "select", kv=131072, count=64),
        # A chunk of a long prompt, each token with pages of its own.
        _case("select_chunk", "select", q=512, kv=32768, count=32),
        # A serving step of long contexts.
        _case("selected_batch", "selected", batch=16, kv=65536, ragged=True, count=64,
              cache="fp16"),
        # A chunk of a long prompt, 8-bit cache, odd sizes.
        _case("selected_chunk_int8", "selected", q=251, kv=30011, count=31, heads=35, kv_heads=5,
              dim=80, page=32, cache="int8"),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["append", "attend", "attend", "bounds", "select", "selected", "selected"])
    cache = "fp4" if op in ("append", "attend") else rng.choice(["fp16", "int8", "fp4"])
    heads = [(32, 4, 64), (32, 8, 128), (16, 16, 128), (12, 6, 96), (35, 5, 128), (14, 2, 64),
             (8, 1, 256), (20, 4, 160), (9, 3, 32)]
    if cache != "fp4":  # (4-bit heads are whole groups of 32)
        heads += [(35, 5, 80), (9, 3, 40), (12, 6, 80)]
    heads, kv_heads, dim = rng.choice(heads)
    c = {"op": op, "heads": heads, "kv_heads": kv_heads, "dim": dim, "cache": cache,
         "page": rng.choice([16, 32, 64, 128, 256]), "ragged": rng.random() < 0.7, "window": 0,
         "count": 0}
    few = rng.random() < 0.6  # single tokens, or a few (drafts to be verified)
    batch = _log(rng, 1, 64 if few else 6)
    q = rng.choice([1, 1, 1, 2, 5]) if few else _log(rng, 6, 1024)
    c.update({"batch": batch, "q": q})
    if op == "append":
        c.update({"kv": max(q, _log(rng, 1, 200000)), "style": rng.choice(["halves", "pairs"]),
                  "rot": rng.choice([dim, dim, dim // 2 // 8 * 8]), "window": 1})
    elif op == "attend":
        c.update({"kv": q + _log(rng, 1, 131072 // batch if few else 16384 // batch),
                  "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)])})
    elif op == "bounds":
        c.update({"kv": q + _log(rng, 1, 262144 // batch)})
    else:
        kv = q + _log(rng, 1, 262144 // batch)
        if op == "selected":  # (what the plain form gathers: at most 1024 tokens' 512 positions)
            c["q"] = q = min(q, 512 // batch + 1)
            count = _log(rng, 3, max(3, min(128, 2 ** 19 // (batch * q * c["page"]))))
        else:
            count = _log(rng, 3, 128)
        c.update({"kv": kv, "count": count})
    return c


# --- sizes ------------------------------------------------------------------------

def _lengths(c):
    """(new tokens, cached tokens with them) of each sequence; from the case alone."""
    out = []
    for b in range(c["batch"]):
        kv = c["kv"]
        if c["ragged"] and b:  # spread evenly over [kv / 8, kv]
            kv = max(c["q"], int(kv * (0.125 + 0.875 * ((b * 0.6180339887498949) % 1.0))))
        out.append((c["q"], kv))
    return out


def _first_position(c, q, kv):
    """The first position that any of a sequence's new tokens reads (or, appending, writes)."""
    return max(0, kv - q - c["window"] + 1) if c["window"] else 0


def _visible(c):
    """(query, position) pairs of one head, and positions read, over all sequences."""
    pairs = tokens = 0
    for q, kv in _lengths(c):
        tokens += kv - _first_position(c, q, kv)
        w = c["window"] or kv
        lo = kv - q + 1  # positions that the first new token could see, itself included
        full = max(0, min(q, q - (w - lo)))  # tokens that see a whole window
        pairs += full * w + (q - full) * (lo + (lo + q - full - 1)) // 2
    return pairs, tokens


def _token_bytes(c):
    """Of one token and kv head in K (or V)."""
    d = c["dim"]
    return {"fp16": 2 * d, "int8": d + 4, "fp4": d // 2 + d // 16}[c["cache"]]


def work(case):
    c = case
    lens = _lengths(c)
    rows = sum(q for q, _ in lens)
    H, KV, D, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    ints = 4 * (2 * c["batch"] + 1)
    if c["op"] == "append":
        n = rows * ((2 * H + 2 * KV) * D * 4 + 2 * KV * _token_bytes(c))
        return {"bytes": n + ints, "flops": 3 * rows * (H + KV) * c["rot"]}
    if c["op"] == "attend":
        pairs, tokens = _visible(c)
        return {"bytes": 2 * rows * H * D * 4 + ints + 2 * tokens * KV * _token_bytes(c),
                "flops": 4 * pairs * H * D}
    if c["op"] == "bounds":
        pages = read = 0
        for q, kv in lens:
            first = (kv - q) // ps
            pages += -(-kv // ps) - first
            read += kv - first * ps
        return {"bytes": read * KV * _token_bytes(c) + pages * KV * (2 * D + 4) + ints,
                "flops": 2 * read * KV * D}
    if c["op"] == "select":
        pages = scored = 0
        for q, kv in lens:
            pages += max(0, (kv - 1) // ps + 1 - FIRST - LAST)
            scored += sum(max(0, p // ps + 1 - FIRST - LAST) for p in range(kv - q, kv))
        return {"bytes": rows * (H * D * 4 + KV * c["count"] * 4) + pages * KV * (2 * D + 4) + ints,
                "flops": 2 * scored * H * D}
    # Tokens of a sequence may share their pages: what is read once is the smaller of both.
    read = pairs = 0
    for q, kv in lens:
        here = [min(c["count"], p // ps + 1) for p in range(kv - q, kv)]
        here = [n * ps - (ps - 1 - p % ps) for n, p in zip(here, range(kv - q, kv))]
        pairs += sum(here)
        read += min(sum(here), kv)
    return {"bytes": rows * (2 * H * D * 4 + KV * c["count"] * 4) +
            2 * read * KV * _token_bytes(c) + ints, "flops": 4 * pairs * H * D}


# --- inputs ------------------------------------------------------------------------

def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = _lengths(c)
    rows = sum(q for q, _ in lens)
    ps, kvh, dim = c["page"], c["kv_heads"], c["dim"]
    # Pages in no order, a few more than are in use; one table row a sequence.
    spans = [(_first_position(c, q, kv) // ps, -(-kv // ps)) for q, kv in lens]
    pages = sum(hi - lo for lo, hi in spans) + 3
    perm = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)
    table = torch.full((c["batch"], max(hi for _, hi in spans)), -1, dtype=torch.int32,
                       device="cuda")
    at = 0
    for b, (lo, hi) in enumerate(spans):
        table[b, lo:hi] = perm[at:at + hi - lo]
        at += hi - lo
    cu = [0]
    for q, _ in lens:
        cu.append(cu[-1] + q)

    def normal(*shape, std=1.0):
        return torch.randn(shape, generator=g, device="cuda").mul_(std)

    s = {"case": c, "table": table, "max_kv": max(kv for _, kv in lens),
         "cu": torch.tensor(cu, dtype=torch.int32, device="cuda"),
         "lens": torch.tensor([kv for _, kv in lens], dtype=torch.int32, device="cuda")}
    # Queries and keys: a few channels an order larger than the rest.
    if c["op"] != "bounds":
        s["q"] = normal(rows, c["heads"], dim, std=2.0)
        s["q"][..., ::37] *= 3.0
    shape = (pages, kvh, ps, dim)
    if c["op"] == "append":
        s["k"] = normal(rows, kvh, dim)
        s["k"][..., ::37] *= 6.0
        s["v"] = normal(rows, kvh, dim)
        s["inv_freq"] = (THETA ** -(torch.arange(0, c["rot"], 2, device="cuda").double() /
                                    c["rot"])).float() if c["rot"] else None
        s["kc"], s["vc"] = (torch.zeros(shape[:3] + (dim // 2,), dtype=torch.uint8, device="cuda")
                            for _ in range(2))
        s["ks"], s["vs"] = (torch.zeros((pages, kvh, dim // 32, ps), dtype=torch.float16,
                                        device="cuda") for _ in range(2))
        return s
    if c["op"] == "select":
        # The smallest and largest of a page's keys in each channel, in 8 bits.
        hi, lo = normal(pages, kvh, dim, std=0.4) + 2.4, normal(pages, kvh, dim, std=0.4) - 2.4
        both = torch.stack([lo, hi], 2)
        both[..., ::37] *= 6.0
        s["bs"] = both.abs().amax((2, 3)) / 127
        s["bc"] = (both / s["bs"][..., None, None]).round_().to(torch.int8)
        return s
    names = [("kc", "ks")] if c["op"] == "bounds" else [("kc", "ks"), ("vc", "vs")]
    for code, scale in names:
        s[scale] = None
        if c["cache"] == "fp16":
            s[code] = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
            if code == "kc":
                s[code][..., ::37] *= 3.0
            # What past the ends was never written holds anything.
            for b, ((_, kv), (_, hi)) in enumerate(zip(lens, spans)):
                if kv % ps:
                    s[code][table[b, hi - 1].long(), :, kv % ps:] = float("nan")
        elif c["cache"] == "int8":
            s[code] = torch.randint(-127, 128, shape, generator=g, device="cuda",
                                    dtype=torch.int8)
            s[scale] = torch.rand(shape[:3], generator=g, device="cuda").mul_(0.02).add_(0.01)
        else:
            s[code] = torch.randint(0, 256, shape[:3] + (dim // 2,), generator=g, device="cuda",
                                    dtype=torch.uint8)
            s[scale] = torch.rand((pages, kvh, dim // 32, ps), generator=g,
                                  device="cuda").mul_(0.5).add_(0.1).half()
    if c["op"] == "bounds":
        s["bc"] = torch.zeros((pages, kvh, 2, dim), dtype=torch.int8, device="cuda")
        s["bs"] = torch.zeros((pages, kvh), device="cuda")
    else:
        # The first page, the last two, and others by chance, in order; -1 behind.
        pos = torch.cat([torch.arange(kv - q, kv, device="cuda") for q, kv in lens])
        here = (pos // ps)[:, None, None]
        p = torch.arange(s["table"].shape[1], device="cuda")
        rank = torch.rand((rows, kvh, len(p)), generator=g, device="cuda")
        rank = torch.where((p < FIRST) | (p > here - LAST), 2.0, rank)
        rank = torch.where(p > here, -1.0, rank)
        top = rank.topk(min(c["count"], len(p)), -1)
        pick = torch.where(top.values < 0, len(p), top.indices).sort(-1).values
        pick = torch.where(pick == len(p), -1, pick)
        s["pick"] = torch.full((rows, kvh, c["count"]), -1, dtype=torch.int32, device="cuda")
        s["pick"][..., :pick.shape[-1]] = pick
    return s


# --- the plain forms -------------------------------------------------------------------

def _rows(s):
    """Sequence, index in it and position of every new token."""
    cu, t = s["cu"].long(), torch.arange(int(s["case"]["batch"] * s["case"]["q"]), device="cuda")
    seq = torch.searchsorted(cu[1:], t, right=True)
    i = t - cu[seq]
    return seq, i, s["lens"].long()[seq] - (cu[seq + 1] - cu[seq]) + i


def _rotate(x, pos, s):
    """Angles and products in 64 bits: far positions, and values next to a border of
    the 4-bit grid; rounded to 32 bits once."""
    c = s["case"]
    if not c["rot"]:
        return x.clone()
    r, ang = c["rot"], pos.double()[:, None] * s["inv_freq"].double()
    co, si = torch.cos(ang)[:, None], torch.sin(ang)[:, None]
    y = x.double()
    if c["style"] == "halves":
        a, b = y[..., :r // 2], y[..., r // 2:r]
        turned = torch.cat([a * co - b * si, b * co + a * si], -1)
    else:
        a, b = y[..., 0:r:2], y[..., 1:r:2]
        turned = torch.stack([a * co - b * si, b * co + a * si], -1).flatten(-2)
    return torch.cat([turned, y[..., r:]], -1).float()


GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def _to_fp4(x):
    """Codes [..., D / 2] and scales [..., D / 32] of rows x."""
    y = x.unflatten(-1, (-1, 32))
    scale = y.abs().amax(-1)
    scale = (scale / torch.full_like(scale, 6.0)).half()
    y = (y / scale.float()[..., None]).flatten(-2)
    a = y.abs()
    code = ((a > 0.25).byte() + (a >= 0.75).byte() + (a > 1.25).byte() + (a >= 1.75).byte() +
            (a > 2.5).byte() + (a >= 3.5).byte() + (a > 5.0).byte() + torch.signbit(y).byte() * 8)
    return code[..., 0::2] | code[..., 1::2] << 4, scale


def _pairs():
    """[256, 2] fp16: the two values of a byte, low four bits first."""
    grid = torch.tensor(GRID + [-x for x in GRID], device="cuda", dtype=torch.float16)
    return torch.stack([grid.repeat(16), grid.repeat_interleave(16)], -1)


def _values4(codes, scale):
    """fp16 values of codes [..., slots, D / 2] with scales [..., D / 32, slots]."""
    v = _pairs()[codes.int()].flatten(-2)
    v = v.unflatten(-1, (-1, 32)) * scale.transpose(-1, -2)[..., None]
    return v.flatten(-2)


def _plain_append(s):
    c = s["case"]
    seq, _, pos = _rows(s)
    q, k, v = _rotate(s["q"], pos, s), _rotate(s["k"], pos, s), s["v"]
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    s["kc"][page, :, slot], s["ks"][page, :, :, slot] = _to_fp4(k)
    s["vc"][page, :, slot], s["vs"][page, :, :, slot] = _to_fp4(v)
    return q


def _cached(s, name, page, slot):
    """Values of tokens in (page, slot), which have one shape: [*shape, kv_heads, dim]."""
    codes, scale = s[name + "c"], s[name + "s"]
    x = codes[page, :, slot]
    if s["case"]["cache"] == "fp16":
        return x.float()
    if s["case"]["cache"] == "int8":
        return x.float() * scale[page, :, slot][..., None]
    x = _pairs()[x.int()].flatten(-2).unflatten(-1, (-1, 32))
    return (x * scale[page, :, :, slot][..., None]).flatten(-2).float()


def _plain_attend(s):
    c = s["case"]
    seq, i, pos = _rows(s)
    B, H, KV, D, qm = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["q"]
    lens = s["lens"].long()
    p = torch.arange(s["max_kv"], device="cuda")
    page = s["table"][:, p // c["page"]].long()  # [B, L]
    there = (p < lens[:, None]) & (page >= 0)
    page, slot = page.clamp(min=0), (p % c["page"])[None].expand(B, -1)
    keep = there[:, :, None, None]
    k = torch.where(keep, _cached(s, "k", page, slot), 0.0).permute(0, 2, 3, 1)
    v = torch.where(keep, _cached(s, "v", page, slot), 0.0).permute(0, 2, 1, 3)
    q = torch.zeros(B, qm, H, D, device="cuda")
    at = torch.full((B, qm), -1, device="cuda")
    q[seq, i], at[seq, i] = s["q"], pos
    # [B, kv_heads, qm * group, D]
    q = q.view(B, qm, KV, H // KV, D).permute(0, 2, 1, 3, 4).reshape(B, KV, -1, D)
    sees = there[:, None] & (p <= at[..., None])
    if c["window"]:
        sees &= p > at[..., None] - c["window"]
    sees = sees[:, None, :, None]  # [B, 1, qm, 1, L]
    x = torch.matmul(q, k.contiguous()).mul_(D ** -0.5).view(B, KV, qm, H // KV, -1)
    x.masked_fill_(~sees, -math.inf)
    m = x.amax(-1, keepdim=True).clamp(min=-3e38)
    x.sub_(m).exp_()
    o = torch.matmul(x.view(B, KV, qm * (H // KV), -1), v.contiguous())
    o = (o.view(B, KV, qm, H // KV, D) / x.sum(-1, keepdim=True)).permute(0, 2, 1, 3, 4)
    return o.reshape(B, qm, H, D)[seq, i]


def _to_codes(x, dims):
    """8-bit codes of x with one scale over `dims`: rounded, halves away from zero."""
    scale = x.abs().amax(dims, keepdim=True)
    scale = scale / torch.full_like(scale, 127.0)  # (a division: by a number torch multiplies)
    y = torch.where(scale > 0, x / scale, 0.0)
    return torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)), scale


def _plain_bounds(s):
    c = s["case"]
    seq, _, pos = _rows(s)
    ps = c["page"]
    key = torch.unique(seq * s["table"].shape[1] + pos // ps)  # (sequence, page of it)
    seq, at = key // s["table"].shape[1], key % s["table"].shape[1]
    page = s["table"][seq, at].long()
    there = at[:, None] * ps + torch.arange(ps, device="cuda") < s["lens"].long()[seq, None]
    if c["cache"] == "fp4":
        k = _values4(s["kc"][page], s["ks"][page]).float()
    else:
        k = s["kc"][page].float()
        if c["cache"] == "int8":
            k = k * s["ks"][page][..., None]
    there = there[:, None, :, None]
    both = torch.stack([torch.where(there, k, math.inf).amin(2),
                        torch.where(there, k, -math.inf).amax(2)], 2)
    codes, scale = _to_codes(both, (2, 3))
    s["bc"][page], s["bs"][page] = codes.to(torch.int8), scale[:, :, 0, 0]


def _plain_select(s):
    c = s["case"]
    seq, i, pos = _rows(s)
    B, H, KV, D, qm, ps = c["batch"], c["heads"], c["kv_heads"], c["dim"], c["q"], c["page"]
    codes, scale = _to_codes(s["q"], (2,))
    q = torch.zeros(B, qm, H, 2 * D, device="cuda")
    q[seq, i] = torch.cat([codes.clamp(max=0.0), codes.clamp(min=0.0)], -1)
    qs = torch.zeros(B, qm, H, 1, device="cuda")
    qs[seq, i] = scale
    here = torch.full((B, qm), -1, device="cuda")
    here[seq, i] = pos // ps
    group = (B, qm, KV, H // KV, -1)
    q = q.view(group).permute(0, 2, 1, 3, 4).reshape(B, KV, -1, 2 * D)
    qs = qs.view(group).permute(0, 2, 1, 3, 4)
    page = s["table"].long().clamp(min=0)  # [B, P]
    bounds = s["bc"][page].float().flatten(-2)  # [B, P, KV, 2 D]
    # (whole numbers below 2^23: exact in 32 bits, in any order)
    x = torch.matmul(q, bounds.permute(0, 2, 3, 1).contiguous())
    x = x.view(B, KV, qm, H // KV, -1).mul_(qs).amax(3)  # [B, KV, qm, P]
    x = x * s["bs"][page].permute(0, 2, 1)[:, :, None]
    p, here = torch.arange(x.shape[-1], device="cuda"), here[:, None, :, None]
    x = torch.where(s["table"][:, None, None] >= 0, x, -math.inf)
    x = torch.where((p < FIRST) | (p > here - LAST), math.inf, x)
    x = torch.where(p > here, -math.inf, x)
    top = torch.sort(x, dim=-1, descending=True, stable=True)
    n = min(c["count"], len(p))
    pick = torch.where(top.values == -math.inf, len(p), top.indices)[..., :n].sort(-1).values
    pick = torch.where(pick == len(p), -1, pick).permute(0, 2, 1, 3)[seq, i]
    out = torch.full((len(seq), KV, c["count"]), -1, dtype=torch.int32, device="cuda")
    out[..., :n] = pick
    return out


def _plain_selected(s):
    c = s["case"]
    seq, _, pos = _rows(s)
    T, KV, ps, D = len(seq), c["kv_heads"], c["page"], c["dim"]
    pick = s["pick"].long()  # [T, KV, n]
    page = s["table"][seq[:, None, None], pick.clamp(min=0)].long()
    slot = torch.arange(ps, device="cuda")
    sees = (pick >= 0)[..., None] & (pick[..., None] * ps + slot <= pos[:, None, None, None])
    page, sees = page.clamp(min=0)[..., None], sees.view(T, KV, -1)
    head = torch.arange(KV, device="cuda")[:, None, None]

    def values(name):
        codes, scale = s[name + "c"], s[name + "s"]
        x = codes[page, head, slot].view(T, KV, -1, codes.shape[-1])
        if c["cache"] == "fp16":
            x = x.float()
        elif c["cache"] == "int8":
            x = x.float() * scale[page, head, slot].view(T, KV, -1, 1)
        else:
            block = torch.arange(D // 32, device="cuda")
            by = scale[page[..., None], head[..., None], block, slot[:, None]]
            x = _pairs()[x.int()].view(T, KV, -1, D // 32, 32) * by.view(T, KV, -1, D // 32, 1)
            x = x.flatten(-2).float()
        return torch.where(sees[..., None], x, 0.0)

    q = s["q"].view(T, KV, -1, D)
    x = torch.matmul(q, values("k").transpose(-1, -2).contiguous()).mul_(D ** -0.5)
    x.masked_fill_(~sees[:, :, None], -math.inf)
    x = (x - x.amax(-1, keepdim=True).clamp(min=-3e38)).exp()
    return (torch.matmul(x, values("v")) / x.sum(-1, keepdim=True)).view(T, c["heads"], D)


# --- one pass -----------------------------------------------------------------------

def run(state):
    s = state
    c = s["case"]
    if own:
        import hypno_amd as hk
        batch = dict(page_table=s["table"], kv_lens=s["lens"], cu_q=s["cu"])
    if c["op"] == "attend":
        if own:
            return hk.paged_attention(s["q"], s["kc"], s["vc"], **batch, window=c["window"],
                                      k_scale=s["ks"], v_scale=s["vs"], max_kv_len=s["max_kv"])
        return _plain_attend(s)
    if c["op"] == "select":
        if own:
            return hk.select_pages(s["q"], s["bc"], s["bs"], c["page"], **batch,
                                   count=c["count"], first=FIRST, last=LAST,
                                   max_kv_len=s["max_kv"])
        return _plain_select(s)
    if c["op"] == "selected":
        if own:
            return hk.selected_attention(s["q"], s["kc"], s["vc"], s["pick"], **batch,
                                         k_scale=s["ks"], v_scale=s["vs"])
        return _plain_selected(s)
    if c["op"] == "bounds":
        if own:
            hk.key_bounds(s["kc"], s["bc"], s["bs"], **batch, k_scale=s["ks"])
        else:
            _plain_bounds(s)
        # (the values that the codes stand for)
        return s["bc"] * s["bs"][..., None, None]
    if own:
        q = hk.append_kv(s["q"], s["k"], s["v"], s["kc"], s["vc"], **batch,
                         inv_freq=s["inv_freq"], style=c["style"], k_scale=s["ks"],
                         v_scale=s["vs"])
    else:
        q = _plain_append(s)
    return {"q": q, "k": _values4(s["kc"], s["ks"]), "v": _values4(s["vc"], s["vs"])}


# --- the definitions in 64 bits ----------------------------------------------------------

def _exact_fp4(x):
    """The values that the 4-bit codes of rows x stand for (x: of 32 bits, held in 64):
    quotients are defined in 32 bits, scales and values in 16."""
    y = x.unflatten(-1, (-1, 32))
    scale = (y.abs().amax(-1, keepdim=True) / 6).float().half().double()
    y = torch.where(scale > 0, (y / scale).float().double(), 0.0)
    a = y.abs().clamp(max=6.0)
    step = torch.where(a < 2, 0.5, torch.where(a < 4, 1.0, 2.0))
    a = torch.round(a / step) * step  # (halves to even)
    return (a * y.sign() * scale).half().double().flatten(-2)


def _exact_read(s, name, g, page, slot):
    x = s[name + "c"][page, g, slot]
    if s["case"]["cache"] == "fp16":
        return x.double()
    if s["case"]["cache"] == "int8":
        return x.double() * s[name + "s"][page, g, slot, None].double()
    code = torch.stack([x & 15, x >> 4], -1).flatten(-2).long()
    exponent, fraction = code >> 1 & 3, (code & 1).double()
    value = torch.where(exponent > 0, torch.exp2(exponent.double() - 1) * (1 + fraction / 2),
                        fraction / 2)
    value = torch.where(code > 7, -value, value)
    scale = s[name + "s"][page, g, :, slot].double().repeat_interleave(32, -1)
    return (value * scale).half().double()


def _exact_codes(x, scale):
    return ((x / scale).float().double().abs() + 0.5).floor() * x.sign()


def _exact_pick(c, pos, score, ids):
    """The pages of one token: score [P] of the sequence's pages, their ids."""
    here = pos // c["page"]
    kept = {p for p in range(here + 1) if p < FIRST or p > here - LAST}
    free = [p for p in range(here + 1) if p not in kept and ids[p] >= 0]
    free.sort(key=lambda p: (-score[p], p))
    pick = sorted(list(kept) + free[:max(0, c["count"] - len(kept))])
    return pick + [-1] * (c["count"] - len(pick))


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    out, t0 = [], 0
    H, KV, D, ps = c["heads"], c["kv_heads"], c["dim"], c["page"]
    G = H // KV
    if c["op"] == "append":
        kc, vc = (torch.zeros(s["kc"].shape[:3] + (D,), dtype=torch.float64, device="cuda")
                  for _ in range(2))
    if c["op"] == "bounds":
        bounds = torch.zeros(s["bc"].shape, dtype=torch.float64, device="cuda")
    for b, (n, kv) in enumerate(_lengths(c)):
        pos = torch.arange(kv - n, kv, device="cuda")
        q = s["q"][t0:t0 + n].double() if "q" in s else None
        if c["op"] == "append":
            turned = []
            for x in (q, s["k"][t0:t0 + n].double()):
                if c["rot"]:
                    # As complex numbers: (x0 + i x1) times e^(i angle).
                    half = c["rot"] // 2
                    near = 2 * torch.arange(half, device="cuda")
                    i0, i1 = ((near // 2, near // 2 + half) if c["style"] == "halves"
                              else (near, near + 1))
                    angle = pos[:, None, None] * s["inv_freq"].double()
                    z = torch.complex(x[..., i0], x[..., i1]) * torch.polar(
                        torch.ones_like(angle), angle)
                    x[..., i0], x[..., i1] = z.real, z.imag
                turned.append(x)
            out.append(turned[0])
            page, slot = s["table"][b].long()[pos // ps], pos % ps
            kc[page, :, slot] = _exact_fp4(turned[1].float().double())
            vc[page, :, slot] = _exact_fp4(s["v"][t0:t0 + n].double())
        elif c["op"] == "bounds":
            for at in range((kv - n) // ps, -(-kv // ps)):
                page, slot = s["table"][b, at].long(), torch.arange(min(ps, kv - at * ps),
                                                                    device="cuda")
                for g in range(KV):
                    k = _exact_read(s, "k", g, page.expand(len(slot)), slot).float().double()
                    both = torch.stack([k.amin(0), k.amax(0)])
                    scale = (both.abs().amax() / 127).float().double()
                    bounds[page, g] = _exact_codes(both, scale) * scale
        elif c["op"] == "select":
            page = s["table"][b].long()[:-(-kv // ps)]
            score = torch.empty(n, KV, len(page), device="cuda")
            for g in range(KV):
                for h in range(g * G, g * G + G):
                    scale = (q[:, h].abs().amax(-1) / 127).float().double()
                    x = _exact_codes(q[:, h], scale[:, None])
                    lo, hi = (s["bc"][page, g, j].double() for j in (0, 1))
                    # sum over the channels of max(x lo, x hi)
                    y = ((x[:, None] + x[:, None].abs()) / 2 * hi +
                         (x[:, None] - x[:, None].abs()) / 2 * lo).sum(-1)
                    y = (y * scale[:, None]).float()
                    score[:, g] = y if h == g * G else torch.maximum(score[:, g], y)
            score, ids = (score * s["bs"][page].T).tolist(), page.tolist()
            out.append(torch.tensor([[_exact_pick(c, kv - n + i, score[i][g], ids)
                                      for g in range(KV)] for i in range(n)],
                                    dtype=torch.int32, device="cuda"))
        else:
            first = _first_position(c, n, kv)
            p = torch.arange(first, kv, device="cuda")
            page, slot = s["table"][b].long()[p // ps], p % ps
            o = torch.empty(n, H, D, dtype=torch.float64, device="cuda")
            hidden = p > pos[:, None]
            if c["window"]:
                hidden |= p <= pos[:, None] - c["window"]
            for g in range(KV):
                k, v = (_exact_read(s, name, g, page, slot) for name in "kv")
                if c["op"] == "selected":
                    pick = s["pick"][t0:t0 + n, g].long()
                    seen = torch.zeros(n, len(s["table"][b]) + 1, dtype=torch.bool, device="cuda")
                    seen.scatter_(1, torch.where(pick < 0, seen.shape[1] - 1, pick), True)
                    hide = hidden | ~seen[:, p // ps]
                else:
                    hide = hidden
                # (NaN in places that nobody sees)
                k, v = (torch.where(hide.all(0)[:, None], 0.0, y) for y in (k, v))
                for h in range(g * G, g * G + G):
                    x = (q[:, h] @ k.T) / math.sqrt(D)
                    x[hide] = -math.inf
                    x = torch.exp(x - x.max(-1, keepdim=True).values)
                    o[:, h] = (x / x.sum(-1, keepdim=True)) @ v
            out.append(o)
        t0 += n
    if c["op"] == "append":
        return {"q": torch.cat(out), "k": kc, "v": vc}
    return bounds if c["op"] == "bounds" else torch.cat(out)
