"""A decoder layer on the GPU with a paged KV cache: Q4_0 projections, keys and values
appended with their rotation, attention over the pages, the gated MLP.  A prompt goes
through in two chunks and tokens follow one by one (each the layer's last output, in
place of an embedded token); the same rows as one prompt have to give the same outputs.

    python examples/paged_decode.py [--prompt 500] [--tokens 20] [--int8 | --fp4] [--pages N]

With --pages, tokens after the prompt read only the N pages of their context that
score highest (the first and the last two always), and each one's attention has to be
that of a plain computation over its pages; while N is all of them the outputs are the
same.  The layer has TinyLlama-1.1B's sizes and random weights.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import hypno_amd as hk  # noqa: E402

HIDDEN, HEADS, KV_HEADS, DIM, INTER, EPS, PAGE = 2048, 32, 4, 64, 5632, 1e-5, 16


class Layer:
    def __init__(self, seed=0):
        g = torch.Generator(device="cuda").manual_seed(seed)

        def weight(n, m):
            w = torch.randn(n * m, generator=g, device="cuda").mul_(m ** -0.5)
            return hk.quantize_f32_to_q4_0(w), n, m

        # q, k and v are one matrix: their rows lie side by side in its output.
        self.qkv = weight((HEADS + 2 * KV_HEADS) * DIM, HIDDEN)
        self.o, self.down = weight(HIDDEN, HEADS * DIM), weight(HIDDEN, INTER)
        self.gate, self.up = weight(INTER, HIDDEN), weight(INTER, HIDDEN)
        self.norms = [torch.rand(HIDDEN, generator=g, device="cuda") + 0.5 for _ in range(2)]
        self.inv_freq = 10000.0 ** (-torch.arange(0, DIM, 2, device="cuda").float() / DIM)

    def product(self, x, w):
        q, n, m = w
        y = torch.empty(x.shape[0], n, device="cuda")
        hk.batch_matmul(y, q, hk.DType.Q4_0, x, n, m, x.shape[0])
        return y

    def __call__(self, x, cache, bounds, table, kv_lens, cu_q, max_kv_len, pages=0):
        """x: the new tokens' rows; kv_lens counts them already.  bounds: of the cache's keys,
        or None where no token selects pages; pages: that each token reads (0: all)."""
        t = x.shape[0]
        y = self.product(hk.rms_norm(x, self.norms[0], EPS, t), self.qkv).view(t, -1, DIM)
        q, k, v = y.split([HEADS, KV_HEADS, KV_HEADS], 1)
        batch = dict(page_table=table, kv_lens=kv_lens, cu_q=cu_q)
        q = hk.append_kv(q, k, v, inv_freq=self.inv_freq, **batch, **cache)
        if bounds:
            hk.key_bounds(cache["k_cache"], *bounds, **batch, k_scale=cache.get("k_scale"))
        if pages:
            chosen = hk.select_pages(q, *bounds, PAGE, **batch, count=pages, last=2,
                                     max_kv_len=max_kv_len)
            a = hk.selected_attention(q, selected=chosen, **batch, **cache)
            check(a[0], q[0], cache, table[0], chosen[0].tolist(), max_kv_len)
        else:
            a = hk.paged_attention(q, max_kv_len=max_kv_len, **batch, **cache)
        x = x + self.product(a.view(t, -1), self.o)
        y = hk.rms_norm(x, self.norms[1], EPS, t)
        return x + self.product(hk.silu_mul(self.product(y, self.gate), self.product(y, self.up)),
                                self.down)


def new_cache(pages, kind):
    """A cache and the bounds of its keys."""
    shape, scales = (pages, KV_HEADS, PAGE, DIM), None
    dtype = {"fp16": torch.float16, "int8": torch.int8, "fp4": torch.uint8}[kind]
    if kind == "int8":
        scales = torch.zeros(shape[:3], device="cuda")
    elif kind == "fp4":
        shape = (*shape[:3], DIM // 2)
        scales = torch.zeros(pages, KV_HEADS, DIM // 32, PAGE, dtype=torch.float16, device="cuda")
    c = {n: torch.zeros(shape, dtype=dtype, device="cuda") for n in ("k_cache", "v_cache")}
    if scales is not None:
        c.update({n: scales.clone() for n in ("k_scale", "v_scale")})
    return c, (torch.zeros(pages, KV_HEADS, 2, DIM, dtype=torch.int8, device="cuda"),
               torch.zeros(pages, KV_HEADS, device="cuda"))


GRID = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]


def cached(cache, name, g, page, slots):
    """Values of a page's slots for kv head g, float64."""
    x, scale = cache[f"{name}_cache"][page, g, slots], cache.get(f"{name}_scale")
    if x.dtype is torch.float16:
        return x.double()
    if x.dtype is torch.int8:
        return x.double() * scale[page, g, slots, None].double()
    grid = torch.tensor(GRID + [-v for v in GRID], dtype=torch.float64, device=x.device)
    v = grid[torch.stack([x & 15, x >> 4], -1).flatten(-2).long()].unflatten(-1, (-1, 32))
    return (v * scale[page, g, :, slots].T[..., None].double()).half().double().flatten(-2)


def over_pages(q, cache, table, chosen, kv):
    """Attention of one token, the last of kv, over the chosen pages for each kv head, and
    the same of |v|: float64."""
    group = q.shape[0] // len(chosen)
    page_size = cache["k_cache"].shape[2]
    out = []
    for g, pages in enumerate(chosen):
        k, v = (torch.cat([cached(cache, n, g, table[p], slice(0, min(page_size, kv - p * page_size)))
                           for p in pages if p >= 0]) for n in "kv")
        s = q[g * group:(g + 1) * group].double() @ k.T / q.shape[-1] ** 0.5
        w = s.softmax(-1)
        out.append(torch.stack([w @ v, w @ v.abs()]))
    return torch.cat(out, 1)


def check(a, q, cache, table, chosen, kv):
    """That `a` is one token's attention over the pages chosen for it, and that these are
    as many as there can be, in order, the first and the last two among them."""
    own = (kv - 1) // cache["k_cache"].shape[2]
    for pages in chosen:
        n = min(len(pages), own + 1)
        if pages[:n] != sorted({*pages[:n], 0, max(own - 1, 0), own}) or pages[n:] != [-1] * (
                len(pages) - n):
            sys.exit(f"pages {pages} for position {kv - 1}")
    # A score is a sum of 64 products of a size of up to 15 here, off by some 72 roundings of
    # it; a weight by twice that, numerator and denominator, and their sums by 16 roundings
    # times the root of the positions, 1024 pages at most: 4200 times 2^-24.
    want, size = over_pages(q, cache, table, chosen, kv)
    if not ((a - want).abs() <= 2.5e-4 * size).all():
        sys.exit(f"attention over pages {chosen} differs at position {kv - 1}")


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--tokens", type=int, default=20)
    kinds = ap.add_mutually_exclusive_group()
    kinds.add_argument("--int8", dest="kind", action="store_const", const="int8", default="fp16")
    kinds.add_argument("--fp4", dest="kind", action="store_const", const="fp4")
    ap.add_argument("--pages", type=int, default=0)
    a = ap.parse_args()
    total = a.prompt + a.tokens
    pages = -(-total // PAGE)
    layer = Layer()
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(a.prompt, HIDDEN, generator=g, device="cuda")
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None].contiguous()

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    (cache, bounds), out, done = new_cache(pages, a.kind), [], 0
    half = a.prompt // 2
    chunks = [rows[:half], rows[half:]] if half else [rows]
    if not a.pages:
        bounds = None
    for i in range(len(chunks) + a.tokens):
        x = chunks[i] if i < len(chunks) else out[-1][-1:] / out[-1][-1:].abs().amax()
        if i >= len(chunks):
            rows = torch.cat([rows, x])
        done += x.shape[0]
        out.append(layer(x, cache, bounds, table, ints(done), ints(0, x.shape[0]), done,
                         a.pages if i >= len(chunks) else 0))
    out = torch.cat(out)
    whole = layer(rows, new_cache(pages, a.kind)[0], None, table, ints(total), ints(0, total),
                  total)
    # The products of many rows take activations in fp16 (2e-3 in the L2 norm), those of
    # one row in fp32; 8-bit codes of values that differ so differ by a step at most, and
    # one in a hundred 4-bit ones by a step, half of a value: 5e-2 in the L2 norm.
    err = ((out - whole).norm() / whole.norm()).item()
    print(f"prompt of {a.prompt} and {a.tokens} tokens against one prompt: {err:.1e}")
    if 0 < a.pages < pages:  # (other outputs; each token's attention was checked)
        print(f"with {a.pages} of {pages} pages")
        if not out.isfinite().all():
            sys.exit("outputs are not finite")
    elif not err < (5e-2 if a.kind == "fp4" else 1e-2):
        sys.exit("outputs differ")
    print("agree")


if __name__ == "__main__":
    main()
