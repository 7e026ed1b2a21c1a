"""A decoder layer on the GPU with a paged KV cache: Q4_0 projections, keys and values
appended with their rotation, attention over the pages, the gated MLP.  A prompt goes
through in two chunks and tokens follow one by one (each the layer's last output, in
place of an embedded token); the same rows as one prompt have to give the same outputs.

    python examples/paged_decode.py [--prompt 500] [--tokens 20] [--int8]

The layer has TinyLlama-1.1B's sizes and random weights.
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

    def __call__(self, x, cache, table, kv_lens, cu_q, max_kv_len):
        """x: the new tokens' rows; kv_lens counts them already."""
        t = x.shape[0]
        y = self.product(hk.rms_norm(x, self.norms[0], EPS, t), self.qkv).view(t, -1, DIM)
        q, k, v = y.split([HEADS, KV_HEADS, KV_HEADS], 1)
        q = hk.append_kv(q, k, v, page_table=table, kv_lens=kv_lens, cu_q=cu_q,
                         inv_freq=self.inv_freq, **cache)
        a = hk.paged_attention(q, page_table=table, kv_lens=kv_lens, cu_q=cu_q,
                               max_kv_len=max_kv_len, **cache)
        x = x + self.product(a.view(t, -1), self.o)
        y = hk.rms_norm(x, self.norms[1], EPS, t)
        return x + self.product(hk.silu_mul(self.product(y, self.gate), self.product(y, self.up)),
                                self.down)


def new_cache(pages, int8):
    shape = (pages, KV_HEADS, PAGE, DIM)
    dtype = torch.int8 if int8 else torch.float16
    c = {n: torch.zeros(shape, dtype=dtype, device="cuda") for n in ("k_cache", "v_cache")}
    if int8:
        c.update({n: torch.zeros(shape[:3], device="cuda") for n in ("k_scale", "v_scale")})
    return c


def main():
    ap = argparse.ArgumentParser()
    ap.add_argument("--prompt", type=int, default=500)
    ap.add_argument("--tokens", type=int, default=20)
    ap.add_argument("--int8", action="store_true")
    a = ap.parse_args()
    total = a.prompt + a.tokens
    pages = -(-total // PAGE)
    layer = Layer()
    g = torch.Generator(device="cuda").manual_seed(1)
    rows = torch.randn(a.prompt, HIDDEN, generator=g, device="cuda")
    table = torch.randperm(pages, generator=g, device="cuda").to(torch.int32)[None].contiguous()

    def ints(*x):
        return torch.tensor(x, dtype=torch.int32, device="cuda")

    cache, out, done = new_cache(pages, a.int8), [], 0
    half = a.prompt // 2
    chunks = [rows[:half], rows[half:]] if half else [rows]
    for i in range(len(chunks) + a.tokens):
        x = chunks[i] if i < len(chunks) else out[-1][-1:] / out[-1][-1:].abs().amax()
        if i >= len(chunks):
            rows = torch.cat([rows, x])
        done += x.shape[0]
        out.append(layer(x, cache, table, ints(done), ints(0, x.shape[0]), done))
    out = torch.cat(out)
    whole = layer(rows, new_cache(pages, a.int8), table, ints(total), ints(0, total), total)
    # The products of many rows take activations in fp16 (2e-3 in the L2 norm), those of
    # one row in fp32; 8-bit codes of values that differ so differ by a step at most.
    err = ((out - whole).norm() / whole.norm()).item()
    print(f"prompt of {a.prompt} and {a.tokens} tokens against one prompt: {err:.1e}")
    if not err < 1e-2:
        sys.exit("outputs differ")
    print("agree")


if __name__ == "__main__":
    main()
