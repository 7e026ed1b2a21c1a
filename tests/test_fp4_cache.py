"""append_kv into a 4-bit cache and paged_attention over it, against their definitions, at
the sizes, masks and values where they can go wrong, and their refusals."""
import ctypes

import numpy as np
import pytest

import hypno_amd as hk
from hypno_amd import _lib
from test_paged_attention import F, K, O, Q, SEQS, V, Batch, _kv, attend, check, queries, run_attend

GRID = np.array([0, 0.5, 1, 1.5, 2, 3, 4, 6], np.float32)
GRID = np.concatenate([GRID, -GRID])


def values4(codes, scale):
    """float64 values of codes [..., slots, D / 2] with scales [..., D / 32, slots]: code *
    scale (exact in fp32) rounded to fp16."""
    c = np.stack([codes & 15, codes >> 4], -1).reshape(*codes.shape[:-1], -1)
    s = np.repeat(np.swapaxes(scale, -1, -2), 32, -1).astype(np.float32)
    with np.errstate(over="ignore", invalid="ignore"):
        return (GRID[c] * s).astype(np.float16).astype(np.float64)


def quantize4(x):
    """Codes and scales [..., D / 32] of float32 rows [..., D], by the definition."""
    y = x.astype(np.float32).reshape(*x.shape[:-1], -1, 32)
    with np.errstate(all="ignore"):
        s = (np.abs(y).max(-1) / np.float32(6)).astype(np.float16)
        s[~np.isfinite(s)] = np.nan
        a = np.abs(y / s[..., None].astype(np.float32)).astype(np.float64)
        # nearest of the grid: among equally near ones the even code
        off = np.abs(a[..., None] - GRID[:8].astype(np.float64))
        near = off == off.min(-1, keepdims=True)
        even = near & (np.arange(8) % 2 == 0)
        code = np.where(even.any(-1), even.argmax(-1), near.argmax(-1))
        code = np.where(a >= 6, 7, code) + 8 * np.signbit(y)
    code = np.where((s > 0)[..., None], code, 0).reshape(x.shape).astype(np.uint8)
    return code[..., 0::2] | code[..., 1::2] << 4, s


class Batch4(Batch):
    def __init__(self, seqs, page, seed, kv_heads=2, dim=64, **kw):
        super().__init__(seqs, page, seed, kv_heads=kv_heads, dim=dim, **kw)
        rng = np.random.default_rng(seed + 77)
        shape = (self.pages, kv_heads, page, dim // 2)
        self.kind = "fp4"
        self.k, self.v = (rng.integers(0, 256, shape).astype(np.uint8) for _ in range(2))
        shape = (self.pages, kv_heads, dim // 32, page)
        self.ks, self.vs = ((rng.random(shape) * 0.5 + 0.1).astype(np.float16) for _ in range(2))

    def values(self, b, g, p):
        pg, sl = self.place(b, p)
        return tuple(values4(c[pg, g, sl][:, None], s[pg, g, :, sl][..., None])[:, 0]
                     for c, s in ((self.k, self.ks), (self.v, self.vs)))

    def as_fp16(self):
        """The same values in an fp16 cache."""
        other = Batch(self.seqs, self.page, 0, kv_heads=self.kv_heads, dim=self.dim)
        other.table, other.pages = self.table, self.pages
        other.k, other.v = (values4(c, s).astype(np.float16)
                            for c, s in ((self.k, self.ks), (self.v, self.vs)))
        return other


HEADS = [(4, 2, 64), (8, 1, 128), (3, 3, 32), (10, 2, 160), (7, 1, 96), (2, 1, 256), (5, 1, 192),
         (20, 1, 64), (33, 1, 128)]
MORE = {**SEQS, "one sequence": [(1, 1500)], "drafts": [(3, 900), (2, 40), (5, 17), (1, 600)],
        "run ends": [(1, n) for n in (15, 16, 17, 32, 33, 47, 48, 49, 127, 128, 129, 255, 257)]}


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("seqs", list(MORE))
def test_attention(seqs, heads, kv_heads, dim):
    page = {"one token": 16, "single tokens": 32, "few tokens": 32, "empty and short": 16,
            "chunks": 16, "long": 128}.get(seqs, 64)
    bt = Batch4(MORE[seqs], page, 5, kv_heads=kv_heads, dim=dim)
    q = queries(bt.tokens, heads, dim, 5)
    check(run_attend(bt, q), *attend(q, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("window", [1, 2, 15, 16, 17, 63, 64, 100, 1000])
def test_window(window):
    bt = Batch4([(1, 1), (1, 700), (3, 200), (40, 300), (1, 64)], 16, 6)
    q = queries(bt.tokens, 4, 64, 6)
    ref, tol = attend(q, bt, window=window)
    check(run_attend(bt, q, window=window), ref, tol)
    # Pages before the windows are not looked at.
    for b, (n, kv) in enumerate(bt.seqs):
        bt.table[b, :max(0, kv - n - window + 1) // bt.page] = -1
    check(run_attend(bt, q, window=window), ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [1.0, -0.3, 0.0, 1e-30])
def test_scale(scale):
    bt = Batch4([(1, 90), (20, 50)], 16, 7)
    q = queries(bt.tokens, 4, 64, 7, std=0.3)
    check(run_attend(bt, q, scale=scale), *attend(q, bt, scale=scale))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 30])
def test_what_masks_hide(n):
    """Infinities and NaN behind the last position, and ahead of a window, do no harm; seen,
    they give what the definition gives; a page that is none is NaN."""
    bt = Batch4([(n, 75), (n, 200), (n, 75)], 16, 8)
    q = queries(bt.tokens, 4, 64, 8)
    ref, tol = attend(q, bt)
    for b, (_, kv) in enumerate(bt.seqs):
        page = bt.table[b, kv // 16]
        bt.ks[page, :, :, kv % 16:] = np.nan
        bt.vs[page, :, :, kv % 16:] = np.inf
    check(run_attend(bt, q), ref, tol)
    bt.vs[bt.table[1, 3], 1, 1, 5] = np.nan  # position 53 of kv head 1, elements 32 to 63
    got = run_attend(bt, q)
    bad = np.zeros_like(got, bool)
    bad[n:2 * n, 2:, 32:] = True
    assert np.isnan(got[bad]).all()
    check(np.where(bad, 0, got), np.where(bad, 0, ref), tol)
    bt.vs[bt.table[1, 3], 1, 1, 5] = 0.5
    for none in (-1, bt.pages, 2 ** 31 - 1, -2 ** 31):
        bt.table[2, 1] = none
        got = run_attend(bt, q)
        assert np.isnan(got[2 * n:]).all() and not np.isnan(got[:2 * n]).any()


@pytest.mark.gpu
def test_values_of_the_format():
    """Scales of every size, infinities of the product, scales of 0: as the fp16 cache of
    the same values; a value past fp16 is an infinity."""
    bt = Batch4([(1, 40), (18, 40)], 16, 9, dim=128)
    rng = np.random.default_rng(1)
    bt.ks = (2.0 ** rng.uniform(-24, -2, bt.ks.shape)).astype(np.float16)
    bt.vs = (2.0 ** rng.uniform(-24, 13, bt.vs.shape)).astype(np.float16)
    bt.ks[..., ::5], bt.vs[..., ::7] = 0, 0
    q = queries(bt.tokens, 4, 128, 9, std=30.0)
    ref, tol = attend(q, bt)
    # Weights are held to 2^-37 of a row's largest: of values 2^37 apart that adds as much
    # of the sum of all that are seen.
    for b in range(2):
        for h in range(4):
            v = bt.values(b, h // 2, np.arange(40))[1]
            tol[bt.cu[b]:bt.cu[b + 1], h] += 2.0 ** -37 * np.abs(v).sum(0)
    check(run_attend(bt, q), ref, tol)
    bt.vs[bt.table[0, 0], 0, 0, 3] = 30000.0
    bt.v[bt.table[0, 0], 0, 3, 0] = 0x17  # 6 and 0.5 of it
    got = run_attend(bt, q)
    assert (got[0, :2, 0] == np.inf).all() and np.isfinite(got[0, :2, 1]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [20, 200])
def test_same_as_fp16(n):
    """A prompt's kernel is the same one: the same bits as an fp16 cache of the values."""
    bt = Batch4([(n, n + 100), (n, n)], 16, 10, kv_heads=1, dim=96)
    q = queries(bt.tokens, 2, 96, 10)
    assert np.array_equal(run_attend(bt, q), run_attend(bt.as_fp16(), q))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 48])
def test_strides(n):
    """Queries out of a fused projection, a pool of pages and layers."""
    import torch
    bt = Batch4([(n, 100), (n, 61)], 16, 16)
    q = queries(bt.tokens, 4, 64, 16)
    ref, tol = attend(q, bt)
    a = bt.gpu()
    fused = torch.randn(bt.tokens, 4 * 64 + 2 * 2 * 64 + 3, device="cuda")
    view = fused[:, 1:257].view(bt.tokens, 4, 64)
    view.copy_(torch.from_numpy(q))
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        pool = torch.zeros((bt.pages, 3, *a[name].shape[1:]), dtype=a[name].dtype, device="cuda")
        pool[:, 1].copy_(a[name])
        a[name] = pool[:, 1]
    check(hk.paged_attention(view, **a).cpu().numpy(), ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 30])
def test_far_pages(n):
    """Pages past 4 GB of the cache."""
    import torch
    bt = Batch4([(n, 150)], 64, 17, kv_heads=8, dim=128)
    q = queries(n, 8, 128, 17)
    ref, tol = attend(q, bt)
    a = bt.gpu()
    pages = 2 ** 32 // (8 * 64 * 64) + 200
    move = torch.arange(bt.pages, device="cuda") + (pages - bt.pages)
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        big = torch.empty((pages, *a[name].shape[1:]), dtype=a[name].dtype, device="cuda")
        big[move] = a[name]
        a[name] = big
    a["page_table"] = torch.where(a["page_table"] >= 0, a["page_table"] + (pages - bt.pages),
                                  a["page_table"]).to(torch.int32)
    check(hk.paged_attention(torch.from_numpy(q).cuda(), **a).cpu().numpy(), ref, tol)


@pytest.mark.gpu
def test_long_context():
    """Ranges of one sequence's positions, and of several of different lengths."""
    for seqs in ([(1, 20011)], [(1, 9001), (1, 3), (1, 5005), (1, 64)], [(2, 6000), (7, 4100)],
                 [(5, 60000)]):
        bt = Batch4(seqs, 64, 18, kv_heads=1, dim=128)
        q = queries(bt.tokens, 4, 128, 18)
        ref, tol = attend(q, bt)
        check(run_attend(bt, q), ref, tol)
        check(run_attend(bt, q, max_kv_len=max(kv for _, kv in seqs)), ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("page", [16, 32])
@pytest.mark.parametrize("window", [0, 3000, 4999])
def test_ranges(page, window):
    """Ranges where pages are a run or two, and from the start of a window on; sequences of
    several tokens among as many as there are tokens."""
    for seqs in ([(1, 7777)], [(1, 9000), (1, 33), (1, 4100)],
                 [(5, 5300), (0, 10), (0, 0), (3, 6001), (0, 5), (0, 7), (1, 40), (0, 3), (0, 1)]):
        for heads, kv_heads, dim in ((4, 1, 64), (7, 1, 128), (9, 1, 32)):
            bt = Batch4(seqs, page, 20, kv_heads=kv_heads, dim=dim)
            q = queries(bt.tokens, heads, dim, 20)
            check(run_attend(bt, q, window=window), *attend(q, bt, window=window))


@pytest.mark.gpu
def test_cu_q_that_does_not_ascend():
    """Nothing is read or written out of place; what the outputs hold is not said."""
    import torch
    bt = Batch4([(1, 100), (1, 40), (2, 60)], 16, 21)
    q = torch.from_numpy(queries(4, 4, 64, 21)).cuda()
    x = torch.randn(4, 2, 64, device="cuda")
    sel = torch.zeros(4, 2, 3, dtype=torch.int32, device="cuda")
    for cu in ([0, 3, 1, 4], [4, 3, 2, 1], [0, -5, 90, 4], [2, 2, 0, 2 ** 31 - 1]):
        a = bt.gpu()
        a["cu_q"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
        hk.append_kv(q, x, x, **a)
        hk.paged_attention(q, **a)
        hk.selected_attention(q, selected=sel, **a)
    torch.cuda.synchronize()


@pytest.mark.gpu
def test_captured():
    """append and attention in a graph, replayed over other tokens with eager work between."""
    import torch
    bt = Batch4([(1, 300), (1, 2000)], 16, 19, dim=128)
    a = bt.gpu()
    x = torch.randn(2, 8, 128, device="cuda")
    inv = torch.linspace(1, 0.01, 64, device="cuda")

    def step():
        q = hk.append_kv(x[:, :4].contiguous(), x[:, 4:6], x[:, 6:], inv_freq=inv, **a)
        return hk.paged_attention(q, **a)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        out = step()
    for i in range(4):
        x.copy_(torch.randn(2, 8, 128, device="cuda"))
        graph.replay()
        torch.cuda.synchronize()
        got = out.clone()
        want = step()
        # (the graph's positions may be split into other ranges)
        assert torch.allclose(got, want, rtol=1e-4, atol=1e-5)


# --- append ------------------------------------------------------------------------------------

def run_append(bt, x, heads, **kw):
    """Codes and scales of tokens x [T, heads + 2 kv_heads, dim] in a fresh cache, and q."""
    import torch
    a = bt.gpu()
    for n in ("k_cache", "v_cache"):
        a[n].fill_(0x5A)
    for n in ("k_scale", "v_scale"):
        a[n].fill_(7.25)
    g = torch.from_numpy(x).cuda()
    q, k, v = g.split([heads, bt.kv_heads, bt.kv_heads], 1)
    q = hk.append_kv(q, k, v, **a, **kw)
    torch.cuda.synchronize()
    return (q.cpu().numpy(), *(a[n].cpu().numpy() for n in ("k_cache", "v_cache", "k_scale",
                                                          "v_scale")))


@pytest.mark.gpu
@pytest.mark.parametrize("kv_heads,dim", [(2, 64), (1, 128), (3, 32), (1, 160), (2, 256), (4, 96)])
def test_append(kv_heads, dim):
    """Bit for bit the definition's codes and scales; nothing else is written."""
    bt = Batch4([(3, 50), (1, 1), (40, 40), (0, 7), (2, 18)], 16, 30, kv_heads=kv_heads, dim=dim)
    rng = np.random.default_rng(30)
    x = rng.standard_normal((bt.tokens, 2 + 2 * kv_heads, dim)).astype(np.float32)
    x *= (10.0 ** rng.uniform(-6, 3, (bt.tokens, 2 + 2 * kv_heads, dim // 32))).repeat(32, -1)
    x = x.astype(np.float32)
    x[::5, :, 32 * (dim // 64):] = 0  # groups of zeros
    x[1::4] = np.round(x[1::4] / np.abs(x[1::4]).max() * 24) / 4  # many halves between codes
    _, kc, vc, ks, vs = run_append(bt, x, 2)
    want = [np.full_like(kc, 0x5A), np.full_like(vc, 0x5A), np.full_like(ks, 7.25),
            np.full_like(vs, 7.25)]
    for b, (n, kv) in enumerate(bt.seqs):
        for i in range(n):
            pg, sl = bt.place(b, kv - n + i)
            t = bt.cu[b] + i
            for j, part in enumerate((x[t, 2:2 + kv_heads], x[t, 2 + kv_heads:])):
                want[j][pg, :, sl], want[2 + j][pg, :, :, sl] = quantize4(part)
    for got, ref in zip((kc, vc, ks, vs), want):
        assert np.array_equal(got, ref)


@pytest.mark.gpu
def test_append_odd_values():
    """Halves between codes both ways, infinities, NaN, the ends of fp16's range."""
    bt = Batch4([(12, 12)], 16, 31, kv_heads=1, dim=64)
    x = np.zeros((12, 3, 64), np.float32)
    halves = np.array([0.25, 0.75, 1.25, 1.75, 2.5, 3.5, 5.0, 6.0], np.float32)
    x[0, 1, :8], x[0, 1, 32:40] = halves, -halves * 2.0 ** 9
    x[1, 1, :16] = np.concatenate([np.nextafter(halves, 9), np.nextafter(halves, 0)])
    x[1, 1, 15] = 6
    x[2, 1, 3], x[3, 1, 3], x[4, 1, 40] = np.inf, np.nan, -np.inf
    x[2:5, 1, 0] = 1
    x[5, 1, :2] = 65504, 60000
    x[6, 1, :2] = 393000, 60000      # a scale of 65504 at most: 6 of it is an infinity
    x[7, 1, :2] = 3.4e38, 1          # a scale past fp16
    x[8, 1, :2] = 2.0 ** -23, 2.0 ** -25
    x[9, 1, :2] = 2.0 ** -24, 2.0 ** -25   # a scale of 2^-26.6: 0
    x[10, 1, :2] = 1e-40, -1e-41
    x[11, 1, :2] = -0.0, 0.0
    x[:, 2] = x[:, 1]
    _, kc, vc, ks, vs = run_append(bt, x, 1)
    codes, scale = quantize4(x[:, 1])
    page = bt.table[0, 0]
    assert np.array_equal(ks[page, 0, :, :12].T, scale, equal_nan=True)
    assert np.array_equal(kc[page, 0, :12], codes)
    assert np.array_equal(vc, kc) and np.array_equal(vs, ks, equal_nan=True)
    assert list(kc[page, 0, 0, :4]) == [0x20, 0x42, 0x64, 0x76]  # 0 1 1 2 2 4 4 6: even codes
    assert np.isnan(ks[page, 0, 0, [2, 3, 7]]).all() and np.isnan(ks[page, 0, 1, 4])
    assert (kc[page, 0, [2, 3, 7], :16] == 0).all() and ks[page, 0, 0, 9] == 0


@pytest.mark.gpu
@pytest.mark.parametrize("style", ["halves", "pairs"])
def test_append_rotated(style):
    """The rotated keys' codes: those of the formula in 64 bits, rounded to fp32."""
    import torch
    bt = Batch4([(5, 100000), (30, 3000)], 256, 32, kv_heads=2, dim=96)
    rng = np.random.default_rng(32)
    x = rng.standard_normal((35, 8, 96)).astype(np.float32)
    rot = 64
    inv = (10000.0 ** (-np.arange(rot // 2) / (rot // 2))).astype(np.float32)
    q, kc, vc, ks, vs = run_append(bt, x, 4, inv_freq=torch.from_numpy(inv).cuda(), style=style)
    pos = np.concatenate([np.arange(kv - n, kv) for n, kv in bt.seqs])
    ang = pos[:, None] * inv.astype(np.float64)
    j = np.arange(rot // 2)
    i0, i1 = (j, j + rot // 2) if style == "halves" else (2 * j, 2 * j + 1)
    y = x.astype(np.float64)
    co, si = np.cos(ang)[:, None], np.sin(ang)[:, None]
    y[..., i0], y[..., i1] = (y[..., i0] * co - y[..., i1] * si, y[..., i1] * co + y[..., i0] * si)
    y = y.astype(np.float32)
    y[:, 6:] = x[:, 6:]
    # (64-bit sines and products may differ in the last place: half a step of fp32 beyond)
    assert np.abs(q - y[:, :4]).max() <= 2.0 ** -22
    for b, (n, kv) in enumerate(bt.seqs):
        pg, sl = bt.place(b, np.arange(kv - n, kv))
        for c, s, part in ((kc, ks, y[:, 4:6]), (vc, vs, y[:, 6:])):
            codes, scale = quantize4(part[bt.cu[b]:bt.cu[b + 1]])
            assert np.array_equal(c[pg, :, sl], codes) and np.array_equal(s[pg, :, :, sl], scale)


@pytest.mark.gpu
def test_append_bad_places():
    """Pages that are none, negative positions, positions past the table, rows of no
    sequence: nothing is written for them."""
    bt = Batch4([(4, 40), (5, 3), (2, 16)], 16, 33)
    bt.table[0, 2] = -1           # positions 32 on
    bt.table[2, 0] = bt.pages
    x = np.random.default_rng(33).standard_normal((bt.tokens + 3, 6, 64)).astype(np.float32)
    q, kc, vc, ks, vs = run_append(bt, x, 2)
    want = np.full_like(kc, 0x5A)
    for i in range(2, 5):  # (tokens 4 and 5 are at positions -2 and -1)
        want[bt.table[1, 0], :, i - 2] = quantize4(x[4 + i, 2:4])[0]
    assert np.array_equal(kc, want)
    assert np.array_equal(q[:bt.tokens], x[:bt.tokens, :2])


@pytest.mark.gpu
def test_append_then_attend():
    """A prompt, then tokens one by one, against the formula over the values appended."""
    import torch
    bt = Batch4([(0, 0)], 16, 34, extra=8, kv_heads=2, dim=64)
    bt.table = np.random.default_rng(2).permutation(bt.pages)[None].astype(np.int32)
    rng = np.random.default_rng(34)
    x = rng.standard_normal((90, 8, 64)).astype(np.float32)
    a, done = bt.gpu(), 0
    for n in (70, 1, 1, 3, 15):
        bt.seqs, bt.cu = [(n, done + n)], np.array([0, n], np.int32)
        a["kv_lens"] = torch.tensor([done + n], dtype=torch.int32, device="cuda")
        a["cu_q"] = torch.tensor([0, n], dtype=torch.int32, device="cuda")
        g = torch.from_numpy(x[done:done + n]).cuda()
        q, k, v = g.split([4, 2, 2], 1)
        got = hk.paged_attention(hk.append_kv(q, k, v, **a), **a).cpu().numpy()
        bt.k, bt.v, bt.ks, bt.vs = (a[m].cpu().numpy() for m in ("k_cache", "v_cache", "k_scale",
                                                                 "v_scale"))
        check(got, *attend(x[done:done + n, :4], bt))
        done += n


# --- refusals (no GPU) --------------------------------------------------------------------------

GOOD = dict(dtype=2, k_scale=6 << 40, v_scale=7 << 40)
BAD = [dict(head_dim=48), dict(head_dim=40), dict(page_size=8), dict(k_scale=None),
       dict(v_scale=None), dict(k_scale=(6 << 40) + 8), dict(v_scale=(7 << 40) + 2),
       dict(k_page_stride=2 * 16 * 32 + 8), dict(v_page_stride=2 * 16 * 32 - 16),
       dict(k_scale_page_stride=60), dict(v_scale_page_stride=68), dict(dtype=3)]


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_c_refuses(bad):
    lib = _lib.load()
    c, b = (ctypes.byref(x) for x in _kv(**{**GOOD, **bad}))
    d = bad.get("head_dim", 64)
    assert lib.hypno_hip_append_kv_dev(c, b, O, 4 * d, Q, 4 * d, 4, K, 2 * d, V, 2 * d, F, 0, 0,
                                       None) == 22
    assert b"append_kv" in lib.hypno_hip_last_error()
    assert lib.hypno_hip_paged_attention_dev(O, Q, 4 * d, 4, c, b, 0.1, 0, 0, None) == 22
    assert b"paged_attention" in lib.hypno_hip_last_error()


def test_c_refuses_overlaps():
    """The codes take half a byte an element, the scales two bytes a group."""
    lib = _lib.load()
    c, b = (ctypes.byref(x) for x in _kv(**GOOD))
    codes, scales = 4 * 2 * 16 * 32, 4 * 2 * 2 * 16 * 2
    for o in ((1 << 40) + codes - 4, (2 << 40), (6 << 40) + scales - 4, 7 << 40):
        assert lib.hypno_hip_paged_attention_dev(o, Q, 256, 4, c, b, 0.1, 0, 0, None) == 22
        assert b"overlaps" in lib.hypno_hip_last_error()
        assert lib.hypno_hip_append_kv_dev(c, b, o, 256, Q, 256, 4, K, 128, V, 128, F, 0, 0,
                                           None) == 22


@pytest.mark.gpu
def test_python_refuses():
    import torch
    bt = Batch4([(2, 30), (1, 25)], 16, 70)
    q = torch.from_numpy(queries(3, 4, 64, 70)).cuda()
    for change, text in (({"k_scale": None}, "k_scale"), ({"v_scale": None}, "v_scale"),
                         ({"k_scale": bt.gpu()["k_scale"].float()}, "float16"),
                         ({"v_scale": bt.gpu()["v_scale"].transpose(2, 3).contiguous()}, "v_scale"),
                         ({"v_cache": bt.gpu()["v_cache"].view(torch.int8)}, "one type"),
                         ({"k_cache": bt.gpu()["k_cache"][..., :31]}, "one type")):
        with pytest.raises(ValueError, match=text):
            hk.paged_attention(q, **{**bt.gpu(), **change})
        with pytest.raises(ValueError, match=text):
            hk.append_kv(q, q[:, :2], q[:, 2:], **{**bt.gpu(), **change})
