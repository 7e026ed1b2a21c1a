"""Performance cases of the attention between a layer's q/k/v projections and its
output projection: rotated keys and values appended to a paged cache
(hypno_amd.append_kv), and attention of the new tokens over that cache
(hypno_amd.paged_attention), from one token of one sequence to long prompts.

A case is a plain dict.  Its "op" says what one pass does:

  append  rotate q and k of every new token, write k and v into their pages
  attend  attention of every new token over its sequence's pages

"batch" sequences bring new tokens: "q" each, or with "mix" the first one "q"
and the others one.  They hold "kv" tokens with the new ones, or with "ragged"
between one eighth of that and all of it.  "window" > 0: a token sees that many
positions, its own included, and pages wholly before the first window are not
in the table any more (-1), as in a server that has freed them.
"""
import math

import torch

own = False

THETA = 10000.0


def _case(name, op, **kw):
    c = {"name": name, "op": op, "batch": 1, "q": 1, "mix": False, "kv": 1, "ragged": False,
         "heads": 32, "kv_heads": 8, "dim": 128, "page": 64, "cache": "fp16", "window": 0}
    if op == "append":
        c.update({"rot": kw.get("dim", 128), "style": "halves"})
    c.update(kw)
    return c


def listed():
    return [
        # The smallest call: a one-token step of a 1.1B model (TinyLlama's heads).
        _case("append_one_token", "append", kv=700, heads=32, kv_heads=4, dim=64, window=1),
        # A serving step of 64 sequences.
        _case("append_decode_batch", "append", batch=64, kv=4096, ragged=True, page=16, window=1),
        # A prompt of ordinary length, pairs of neighbours rotated.
        _case("append_prompt", "append", q=2048, kv=2048, style="pairs"),
        # Chunks of several long prompts into an 8-bit cache, far positions, a
        # rotation of a part of an odd head.
        _case("append_chunks_int8", "append", batch=3, q=333, kv=90001, ragged=True, heads=12,
              kv_heads=6, dim=80, rot=32, page=32, cache="int8", window=1),
        # One token of a 1.1B model in a chat of some hundred tokens.
        _case("decode_one_short", "attend", kv=700, heads=32, kv_heads=4, dim=64),
        # One token over a very long context.
        _case("decode_one_long", "attend", kv=131072),
        # A serving step: 64 sequences of all lengths.
        _case("decode_batch", "attend", batch=64, kv=8192, ragged=True, page=16),
        # The same with the cache in 8 bits.
        _case("decode_batch_int8", "attend", batch=64, kv=8192, ragged=True, page=32,
              cache="int8"),
        # A prompt of ordinary length.
        _case("prompt", "attend", q=2048, kv=2048),
        # The next chunk of a long prompt.
        _case("chunk_of_long_prompt", "attend", q=512, kv=16384),
        # A mixed batch under a sliding window: a chunk beside single tokens, an odd
        # head size and group, 8 bits.
        _case("mixed_window_int8", "attend", batch=7, q=333, mix=True, kv=5003, ragged=True,
              heads=35, kv_heads=5, dim=80, page=16, cache="int8", window=1024),
        # The largest: a whole long prompt.
        _case("long_prompt", "attend", q=8192, kv=8192),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    heads, kv_heads, dim = rng.choice([(32, 4, 64), (32, 8, 128), (16, 16, 128), (12, 6, 80),
                                       (35, 5, 80), (14, 2, 64), (8, 1, 256), (24, 8, 96),
                                       (9, 3, 40)])
    c = {"heads": heads, "kv_heads": kv_heads, "dim": dim,
         "page": rng.choice([8, 16, 32, 64, 128, 256]), "cache": rng.choice(["fp16", "int8"])}
    few = rng.random() < 0.5  # single tokens, or a few (drafts to be verified)
    batch = _log(rng, 1, 64 if few else 6)
    q = rng.choice([1, 1, 1, 2, 5]) if few else _log(rng, 6, 2048)
    c.update({"batch": batch, "q": q, "mix": not few and rng.random() < 0.4,
              "ragged": rng.random() < 0.7})
    if rng.random() < 0.35:
        rot = rng.choice([dim, dim, dim // 2 // 8 * 8])
        c.update({"op": "append", "kv": max(q, _log(rng, 1, 200000)), "rot": rot,
                  "style": rng.choice(["halves", "pairs"]), "window": 1})
    else:
        kv = q + _log(rng, 1, 131072 // batch if few else 16384 // batch)
        c.update({"op": "attend", "kv": kv,
                  "window": rng.choice([0, 0, 0, _log(rng, 1, 4096)])})
    return c


# --- sizes ------------------------------------------------------------------------

def _lengths(c):
    """(new tokens, cached tokens with them) of each sequence; from the case alone."""
    out = []
    for b in range(c["batch"]):
        q = c["q"] if b == 0 or not c["mix"] else 1
        kv = c["kv"]
        if c["ragged"] and b:  # spread evenly over [kv / 8, kv]
            kv = max(q, int(kv * (0.125 + 0.875 * ((b * 0.6180339887498949) % 1.0))))
        out.append((q, kv))
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


def work(case):
    c = case
    rows = sum(q for q, _ in _lengths(c))
    item = 2 if c["cache"] == "fp16" else 1
    scale = 0 if c["cache"] == "fp16" else 4
    ints = 4 * (2 * c["batch"] + 1)
    if c["op"] == "append":
        n = rows * ((2 * c["heads"] + 2 * c["kv_heads"]) * c["dim"] * 4 +
                    2 * c["kv_heads"] * (c["dim"] * item + scale))
        return {"bytes": n + ints, "flops": 3 * rows * (c["heads"] + c["kv_heads"]) * c["rot"]}
    pairs, tokens = _visible(c)
    return {"bytes": 2 * rows * c["heads"] * c["dim"] * 4 + ints +
            2 * tokens * c["kv_heads"] * (c["dim"] * item + scale),
            "flops": 4 * pairs * c["heads"] * c["dim"]}


# --- inputs ------------------------------------------------------------------------

def prepare(case, seed):
    c = case
    g = torch.Generator(device="cuda").manual_seed(seed)
    lens = _lengths(c)
    rows = sum(q for q, _ in lens)
    ps, kvh, dim = c["page"], c["kv_heads"], c["dim"]
    # Pages in no order, a few more than are in use; one table row a sequence.
    spans = [(_first_position(c, q, kv) // ps, -(-kv // ps)) for q, kv in lens]
    used = sum(hi - lo for lo, hi in spans)
    pages = used + 3
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
    s["q"] = normal(rows, c["heads"], dim, std=2.0)
    s["q"][..., ::37] *= 3.0
    shape = (pages, kvh, ps, dim)
    if c["op"] == "append":
        s["k"] = normal(rows, kvh, dim)
        s["k"][..., ::37] *= 6.0
        s["v"] = normal(rows, kvh, dim)
        s["inv_freq"] = (THETA ** -(torch.arange(0, c["rot"], 2, device="cuda").double() /
                                    c["rot"])).float() if c["rot"] else None
        if c["cache"] == "fp16":
            s["kc"], s["vc"] = (torch.zeros(shape, dtype=torch.float16, device="cuda")
                                for _ in range(2))
            s["ks"] = s["vs"] = None
        else:
            s["kc"], s["vc"] = (torch.zeros(shape, dtype=torch.int8, device="cuda")
                                for _ in range(2))
            s["ks"], s["vs"] = (torch.zeros(shape[:3], device="cuda") for _ in range(2))
        return s
    if c["cache"] == "fp16":
        s["kc"] = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
        s["vc"] = torch.randn(shape, generator=g, device="cuda", dtype=torch.float16)
        s["kc"][..., ::37] *= 3.0
        s["ks"] = s["vs"] = None
        # What past the ends and in unused pages was never written holds anything.
        for b, ((_, kv), (_, hi)) in enumerate(zip(lens, spans)):
            if kv % ps:
                p = table[b, hi - 1].long()
                s["kc"][p, :, kv % ps:] = float("nan")
                s["vc"][p, :, kv % ps:] = float("nan")
    else:
        s["kc"], s["vc"] = (torch.randint(-127, 128, shape, generator=g, device="cuda",
                                          dtype=torch.int8) for _ in range(2))
        s["ks"], s["vs"] = (torch.rand(shape[:3], generator=g, device="cuda").mul_(0.02)
                            .add_(0.01) for _ in range(2))
    return s


# --- one pass -----------------------------------------------------------------------

def _rows(s):
    """Sequence, index in it and position of every new token."""
    cu, t = s["cu"].long(), torch.arange(s["q"].shape[0], device="cuda")
    seq = torch.searchsorted(cu[1:], t, right=True)
    i = t - cu[seq]
    return seq, i, s["lens"].long()[seq] - (cu[seq + 1] - cu[seq]) + i


def _rotate(x, pos, s):
    """Angles and products in 64 bits: far positions, and values next to a border of
    the 8-bit grid; rounded to 32 bits once."""
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


def _to_int8(x):
    scale = x.abs().amax(-1, keepdim=True)
    scale = scale / torch.full_like(scale, 127.0)  # (a division: by a number torch multiplies)
    y = x / scale
    return torch.trunc(y + torch.copysign(torch.full_like(y, 0.5), y)).to(torch.int8), scale[..., 0]


def _plain_append(s):
    c = s["case"]
    seq, _, pos = _rows(s)
    q, k, v = _rotate(s["q"], pos, s), _rotate(s["k"], pos, s), s["v"]
    page, slot = s["table"][seq, pos // c["page"]].long(), pos % c["page"]
    if c["cache"] == "fp16":
        s["kc"][page, :, slot], s["vc"][page, :, slot] = k.half(), v.half()
    else:
        s["kc"][page, :, slot], s["ks"][page, :, slot] = _to_int8(k)
        s["vc"][page, :, slot], s["vs"][page, :, slot] = _to_int8(v)
    return q


def _cached(s, cache, scales, page, slot):
    x = cache[page, :, slot].float()  # [B, L, kv_heads, dim]
    return x if scales is None else x * scales[page, :, slot][..., None]


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
    k = torch.where(keep, _cached(s, s["kc"], s["ks"], page, slot), 0.0).permute(0, 2, 3, 1)
    v = torch.where(keep, _cached(s, s["vc"], s["vs"], page, slot), 0.0).permute(0, 2, 1, 3)
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


def run(state):
    s = state
    c = s["case"]
    if c["op"] == "attend":
        if own:
            import hypno_amd as hk
            return hk.paged_attention(s["q"], s["kc"], s["vc"], s["table"], s["lens"], s["cu"],
                                      window=c["window"], k_scale=s["ks"], v_scale=s["vs"],
                                      max_kv_len=s["max_kv"])
        return _plain_attend(s)
    if own:
        import hypno_amd as hk
        q = hk.append_kv(s["q"], s["k"], s["v"], s["kc"], s["vc"], s["table"], s["lens"], s["cu"],
                         inv_freq=s["inv_freq"], style=c["style"], k_scale=s["ks"],
                         v_scale=s["vs"])
    else:
        q = _plain_append(s)
    if c["cache"] == "fp16":
        return {"q": q, "k": s["kc"], "v": s["vc"]}
    # The 8-bit caches as the values that they stand for.
    return {"q": q, "k": s["kc"] * s["ks"][..., None], "v": s["vc"] * s["vs"][..., None]}


# --- the definition in 64 bits ----------------------------------------------------------

def _exact_codes(x):
    """The 8-bit format of rows x (values of 32 bits, held in 64): its scale and its
    quotients are defined in 32 bits.  Returns the values that the codes stand for."""
    scale = (x.abs().amax(-1, keepdim=True) / 127).float().double()
    quotient = (x / scale).float().double()
    return (quotient.abs() + 0.5).floor() * quotient.sign() * scale


def exact(case, seed):
    c = case
    s = prepare(case, seed)
    out, t0 = [], 0
    if c["op"] == "append":
        kc, vc = (torch.zeros(s["kc"].shape, dtype=torch.float64, device="cuda")
                  for _ in range(2))
    for b, (n, kv) in enumerate(_lengths(c)):
        pos = torch.arange(kv - n, kv, device="cuda")
        q = s["q"][t0:t0 + n].double()
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
            page, slot = s["table"][b].long()[pos // c["page"]], pos % c["page"]
            k, v = turned[1], s["v"][t0:t0 + n].double()
            if c["cache"] == "int8":  # (of the values in 32 bits)
                k, v = _exact_codes(k.float().double()), _exact_codes(v)
            kc[page, :, slot], vc[page, :, slot] = k, v
        else:
            first = _first_position(c, n, kv)
            p = torch.arange(first, kv, device="cuda")
            page, slot = s["table"][b].long()[p // c["page"]], p % c["page"]
            o = torch.empty(n, c["heads"], c["dim"], dtype=torch.float64, device="cuda")
            hidden = p > pos[:, None]
            if c["window"]:
                hidden |= p <= pos[:, None] - c["window"]
            for h in range(c["heads"]):
                g = h // (c["heads"] // c["kv_heads"])
                k, v = s["kc"][page, g, slot].double(), s["vc"][page, g, slot].double()
                if s["ks"] is not None:
                    k = k * s["ks"][page, g, slot, None].double()
                    v = v * s["vs"][page, g, slot, None].double()
                x = (q[:, h] @ k.T) / math.sqrt(c["dim"])
                x[hidden] = -math.inf
                x = torch.exp(x - x.max(-1, keepdim=True).values)
                o[:, h] = (x / x.sum(-1, keepdim=True)) @ v
            out.append(o)
        t0 += n
    if c["op"] == "attend":
        return torch.cat(out)
    return {"q": torch.cat(out), "k": kc, "v": vc}
