"""append_kv and paged_attention against their formulas in 64 bits, at the sizes and
masks where they can go wrong, and their refusals."""
import ctypes
import math

import numpy as np
import pytest

import hypno_amd as hk
from hypno_amd import _lib

EPS = 2.0 ** -24  # half a step of fp32, relative


# --- a ragged batch over a paged cache, in 64 bits ------------------------------------

class Batch:
    """Sequences of (new tokens, cached tokens with them); pages in a shuffled order."""

    def __init__(self, seqs, page, seed, extra=2, kv_heads=2, dim=64, kind="fp16", freed=None):
        rng = np.random.default_rng(seed)
        self.seqs, self.page, self.kind = seqs, page, kind
        self.kv_heads, self.dim = kv_heads, dim
        need = [-(-max(kv, 0) // page) for _, kv in seqs]
        self.pages = sum(need) + extra
        self.table = np.full((len(seqs), max(max(need, default=0), 1)), -1, np.int32)
        perm, at = rng.permutation(self.pages).astype(np.int32), 0
        for b, n in enumerate(need):
            self.table[b, :n] = perm[at:at + n]
            at += n
        self.cu = np.cumsum([0] + [q for q, _ in seqs]).astype(np.int32)
        self.lens = np.array([kv for _, kv in seqs], np.int32)
        self.tokens = int(self.cu[-1])
        shape = (self.pages, kv_heads, page, dim)
        if kind == "fp16":
            self.k = rng.standard_normal(shape).astype(np.float16)
            self.v = rng.standard_normal(shape).astype(np.float16)
            self.ks = self.vs = None
        else:
            self.k = rng.integers(-127, 128, shape).astype(np.int8)
            self.v = rng.integers(-127, 128, shape).astype(np.int8)
            self.ks = (rng.random(shape[:3]) * 0.02 + 0.01).astype(np.float32)
            self.vs = (rng.random(shape[:3]) * 0.02 + 0.01).astype(np.float32)

    def place(self, b, p):
        return self.table[b, p // self.page], p % self.page

    def values(self, b, g, p):
        """K and V of kv head g at positions p of sequence b, float64."""
        pg, sl = self.place(b, p)
        k, v = self.k[pg, g, sl].astype(np.float64), self.v[pg, g, sl].astype(np.float64)
        if self.ks is not None:
            k *= self.ks[pg, g, sl].astype(np.float64)[:, None]
            v *= self.vs[pg, g, sl].astype(np.float64)[:, None]
        return k, v

    def gpu(self):
        import torch
        up = lambda a: None if a is None else torch.from_numpy(a).cuda()  # noqa: E731
        return dict(k_cache=up(self.k), v_cache=up(self.v), page_table=up(self.table),
                    kv_lens=up(self.lens), cu_q=up(self.cu), k_scale=up(self.ks),
                    v_scale=up(self.vs))


def attend(q, bt, scale=None, window=0):
    """The formula in 64 bits, and how far an fp32 computation may be from it.

    A score of D products is off by at most about sqrt(D) roundings of its sum of
    |products| (random signs; 8 sigma), q's parts add 4, the exponent's scaling 4; a
    weight is off by the score's error, numerator and denominator both, and their sums
    over n positions by sqrt(n) roundings each."""
    T, H, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, tol = np.zeros((T, H, D)), np.zeros((T, H, D))
    per = H // bt.kv_heads
    for b, (n, kv) in enumerate(bt.seqs):
        for i in range(n):
            pos, t = kv - n + i, bt.cu[b] + i
            p = np.arange(max(0, pos - window + 1) if window else 0, pos + 1)
            if not len(p):
                continue
            for h in range(H):
                k, v = bt.values(b, h // per, p)
                x = q[t, h].astype(np.float64)
                s = (k @ x) * scale
                size = (np.abs(k) @ np.abs(x)).max() * abs(scale)
                w = np.exp(s - s.max())
                w /= w.sum()
                out[t, h] = w @ v
                off = 2 * size * (8 * math.sqrt(D) + 8) + 16 * math.sqrt(len(p)) + 16
                tol[t, h] = EPS * off * (w @ np.abs(v)) + 1e-37
    return out, tol


def run_attend(bt, q, **kw):
    import torch
    out = torch.full(q.shape, 7.25, device="cuda")
    args = {k: v for k, v in bt.gpu().items()}
    got = hk.paged_attention(torch.from_numpy(q).cuda(), out=out, **args, **kw)
    torch.cuda.synchronize()
    assert got is out
    return got.cpu().numpy()


def check(got, ref, tol):
    worst = np.max(np.abs(got - ref) / np.maximum(tol, 1e-300))
    assert np.all(np.abs(got - ref) <= tol), f"{worst:.3g} of the tolerance"


def queries(T, H, D, seed, std=2.0):
    return (np.random.default_rng(seed + 1000).standard_normal((T, H, D)) * std).astype(np.float32)


HEADS = [(4, 2, 64), (8, 1, 128), (3, 3, 40), (10, 2, 80), (7, 1, 96), (2, 1, 256), (4, 4, 8),
         (5, 1, 192)]
SEQS = {
    "one token": [(1, 1)],
    "single tokens": [(1, 1), (1, 2), (1, 31), (1, 64), (1, 65), (1, 300)],
    "few tokens": [(2, 2), (3, 50), (5, 129), (4, 4)],
    "empty and short": [(0, 10), (1, 0), (3, 1), (0, 0), (2, 2), (4, 2)],
    "chunks": [(33, 33), (64, 200), (1, 77), (130, 131)],
    "long": [(1, 2500), (17, 1100)],
}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", HEADS)
@pytest.mark.parametrize("seqs", list(SEQS))
def test_attention(seqs, heads, kv_heads, dim, kind):
    page = {"one token": 16, "single tokens": 8, "few tokens": 32, "empty and short": 1,
            "chunks": 16, "long": 128}[seqs]
    bt = Batch(SEQS[seqs], page, 5, kv_heads=kv_heads, dim=dim, kind=kind)
    q = queries(bt.tokens, heads, dim, 5)
    check(run_attend(bt, q), *attend(q, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("window", [1, 2, 63, 64, 100, 5000])
@pytest.mark.parametrize("seqs", ["single tokens", "chunks", "long", "empty and short"])
def test_window(seqs, window, kind):
    bt = Batch(SEQS[seqs], 16, 6, kind=kind)
    q = queries(bt.tokens, 4, 64, 6)
    check(run_attend(bt, q, window=window), *attend(q, bt, window=window))


@pytest.mark.gpu
@pytest.mark.parametrize("max_kv", [None, 1, 300, 100000])
@pytest.mark.parametrize("page", [1, 4, 64, 1024])
def test_pages_and_bounds(page, max_kv):
    """Pages of one slot to one page for all; an upper bound that is none."""
    bt = Batch([(1, 700), (40, 300), (2, 1), (1, 64)], page, 7)
    q = queries(bt.tokens, 6, 64, 7)
    check(run_attend(bt, q, max_kv_len=max_kv), *attend(q, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0, 4.0])
def test_scale(scale):
    bt = Batch([(1, 200), (40, 90)], 16, 8)
    q = queries(bt.tokens, 4, 64, 8, std=1.0)
    check(run_attend(bt, q, scale=scale), *attend(q, bt, scale=scale))


@pytest.mark.gpu
@pytest.mark.parametrize("size", [1e-30, 1e-6, 30.0, 3e4])
def test_query_sizes(size):
    """Tokens of every magnitude keep fp32's precision (scaled back for the softmax)."""
    bt = Batch([(1, 200), (40, 90)], 16, 9)
    q = queries(bt.tokens, 4, 64, 9, std=size)
    q[:, :, 5] *= 1000.0
    scale = 0.125 / (size * 100)
    check(run_attend(bt, q, scale=scale), *attend(q, bt, scale=scale))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
def test_large_and_small_values(kind):
    """Values of one cache from the smallest to the largest: small ones beside one that
    holds all the weight, and whole sequences of either."""
    bt = Batch([(1, 700), (33, 400), (1, 300)], 32, 10, kind=kind)
    rng = np.random.default_rng(1)
    if kind == "fp16":
        bt.v[:] = bt.v * 10.0 ** rng.integers(-6, 4, bt.v.shape[:3])[..., None].astype(np.float32)
    else:
        bt.vs[:] = bt.vs * 10.0 ** rng.integers(-30, 30, bt.vs.shape).astype(np.float32)
        bt.ks[:, :, ::3] = 0.0
    q = queries(bt.tokens, 4, 64, 10)
    check(run_attend(bt, q), *attend(q, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 20])
@pytest.mark.parametrize("kind", ["fp16", "int8"])
def test_weight_in_many_small_ones(kind, n):
    """A first token of weight 1 and a value of zero beside 20000 of weight e^-9: what
    comes out is the sum of the small ones."""
    bt = Batch([(n, 20000)], 64, 11, kv_heads=1, kind=kind)
    pg, sl = bt.place(0, np.arange(20000))
    q = np.zeros((n, 2, 64), np.float32)
    q[:, :, 0] = 8.0
    if kind == "fp16":
        bt.k[pg, 0, sl, 0] = 0.0
        bt.k[pg[0], 0, sl[0], 0] = 9.0
        bt.v[pg, 0, sl] = np.abs(bt.v[pg, 0, sl])
        bt.v[pg[0], 0, sl[0]] = 0.0
    else:
        bt.ks[:] = 9.0 / 127
        bt.k[pg, 0, sl, 0] = 0
        bt.k[pg[0], 0, sl[0], 0] = 127
        bt.v[pg, 0, sl] = np.abs(bt.v[pg, 0, sl].astype(np.int32)).astype(np.int8)
        bt.v[pg[0], 0, sl[0]] = 0
    check(run_attend(bt, q), *attend(q, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("what", [float("nan"), float("inf"), -float("inf")])
@pytest.mark.parametrize("seqs", [[(1, 70)], [(40, 70)], [(5, 70), (1, 9)], [(150, 150)]])
@pytest.mark.parametrize("window", [0, 20])
@pytest.mark.parametrize("kind", ["fp16", "int8"])
def test_masked_places(kind, window, seqs, what):
    """Infinities and NaN past the ends, before windows and in positions that some of a
    chunk's tokens do not see reach the tokens that see them, no other."""
    bt = Batch(seqs, 16, 12, kind=kind)
    k, v = (bt.k, bt.v) if kind == "fp16" else (bt.ks, bt.vs)
    spoilt = {}
    for b, (n, kv) in enumerate(seqs):
        pg, sl = bt.place(b, np.arange(kv, bt.table.shape[1] * 16))
        ok = pg >= 0
        k[pg[ok], :, sl[ok]], v[pg[ok], :, sl[ok]] = what, what
        if window and kv - n - window > 0:
            pg, sl = bt.place(b, np.arange(0, kv - n - window + 1))
            k[pg, :, sl], v[pg, :, sl] = what, what
        if n > 4:
            spoilt[b] = kv - 3  # seen by the last three tokens only
            pg, sl = bt.place(b, spoilt[b])
            v[pg, 0, sl] = what
    q = queries(bt.tokens, 4, 64, 12)
    with np.errstate(invalid="ignore"):
        ref, tol = attend(q, bt, window=window)
    got = run_attend(bt, q, window=window)
    hit = np.zeros(q.shape[:2], bool)
    for b, p in spoilt.items():
        hit[bt.cu[b + 1] - 3:bt.cu[b + 1], :2] = True  # heads of kv head 0
    check(got[~hit], ref[~hit], tol[~hit])
    if hit.any():
        if kind == "int8" and not math.isnan(what):  # (a code of 0 times infinity is NaN)
            assert not np.isfinite(got[hit]).any()
        else:
            assert np.array_equal(got[hit], np.full_like(got[hit], what), equal_nan=True)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40])
def test_scores_without_weight(n):
    """Keys of -inf score have no weight; where all are, the output is zero."""
    bt = Batch([(n, 100), (n, 100)], 16, 13, kv_heads=1)
    bt.k[..., 0] = 1.0
    for b, seen in ((0, np.arange(0, 100, 2)), (1, np.arange(100))):
        pg, sl = bt.place(b, seen)
        bt.k[pg, 0, sl, 0] = -np.inf
    q = np.abs(queries(bt.tokens, 2, 64, 13)) + 0.1
    got = run_attend(bt, q)
    live = Batch([(n, 100), (n, 100)], 16, 13, kv_heads=1)
    live.k, live.v, live.table = bt.k.copy(), bt.v, bt.table
    pg, sl = bt.place(0, np.arange(0, 100, 2))
    live.k[pg, 0, sl] = 0.0
    live.k[pg, 0, sl, 0] = -60000.0
    ref, tol = attend(q, live)
    half = bt.cu[1]
    # (the formula's own tolerance, without the stand-in's large products)
    size = np.abs(live.k[live.k > -1000].astype(np.float64)).max() * np.abs(q).sum(-1).max()
    lim = EPS * (2 * size * (8 * 8 + 8) + 16 * 10 + 16) * np.abs(bt.v.astype(np.float64)).max()
    assert np.max(np.abs(got[:half] - ref[:half])) <= lim
    assert not got[half:].any()


@pytest.mark.gpu
def test_bad_pages_and_lengths():
    """Pages that are none, and a sequence longer than its table: NaN for the tokens
    that see them, no access elsewhere; their neighbours are as they were."""
    bt = Batch([(3, 40), (1, 40), (50, 60), (1, 64), (2, 30), (1, 30)], 16, 14)
    q = queries(bt.tokens, 4, 64, 14)
    ref, tol = attend(q, bt)
    bt.table[0, 1], bt.table[1, 0], bt.table[2, 3] = -1, bt.pages, 2 ** 31 - 1
    bt.lens[3], bt.lens[4] = 2 ** 31 - 1, -7
    got = run_attend(bt, q)
    bad = np.zeros(bt.tokens, bool)
    bad[0:4], bad[54] = True, True
    bad[4 + 38:54] = True     # positions 48 and up are in the third sequence's fourth page
    assert np.isnan(got[bad]).all()
    zero = np.zeros(bt.tokens, bool)
    zero[55:57] = True        # a negative length holds nothing
    assert not got[zero].any()
    fine = ~bad & ~zero
    check(got[fine], ref[fine], tol[fine])
    # Windows that begin after the bad page do not see it.
    bt = Batch([(3, 70), (30, 70)], 16, 14)
    q = queries(bt.tokens, 4, 64, 14)
    ref, tol = attend(q, bt, window=20)
    bt.table[0, :2], bt.table[1, 0] = -1, 1 << 30
    check(run_attend(bt, q, window=20), ref, tol)


@pytest.mark.gpu
def test_rows_of_no_sequence():
    """Rows past cu_q's end, and a cu_q that goes down, leave out alone and lead nowhere."""
    bt = Batch([(2, 30), (3, 20)], 16, 15)
    q = queries(9, 4, 64, 15)
    ref, tol = attend(q[:5], bt)
    got = run_attend(bt, q)
    check(got[:5], ref, tol)
    assert (got[5:] == 7.25).all()
    bt.cu[:] = [0, 9, -4]
    got = run_attend(bt, q)
    assert (got[9:] == 7.25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("n", [1, 48])
def test_strides(kind, n):
    """Queries out of a fused projection, a pool of pages and layers."""
    import torch
    bt = Batch([(n, 100), (n, 61)], 16, 16, kind=kind)
    q = queries(bt.tokens, 4, 64, 16)
    ref, tol = attend(q, bt)
    a = bt.gpu()
    fused = torch.randn(bt.tokens, 4 * 64 + 2 * 2 * 64 + 3, device="cuda")
    view = fused[:, 1:257].view(bt.tokens, 4, 64)
    view.copy_(torch.from_numpy(q))
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        if a[name] is not None:
            pool = torch.zeros((bt.pages, 3, *a[name].shape[1:]), dtype=a[name].dtype,
                               device="cuda")
            pool[:, 1].copy_(a[name])
            a[name] = pool[:, 1]
    check(hk.paged_attention(view, **a).cpu().numpy(), ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 70])
def test_far_pages(n):
    """Pages past 4 GB of the cache."""
    import torch
    bt = Batch([(n, 200)], 64, 17, kv_heads=8, dim=128)
    q = queries(n, 8, 128, 17)
    ref, tol = attend(q, bt)
    a = bt.gpu()
    pages = (5 << 30) // (8 * 64 * 128 * 2)
    for name in ("k_cache", "v_cache"):
        big = torch.empty((pages, 8, 64, 128), dtype=torch.float16, device="cuda")
        big[pages - bt.pages:].copy_(a[name])
        a[name] = big
    a["page_table"] += pages - bt.pages
    check(hk.paged_attention(torch.from_numpy(q).cuda(), **a).cpu().numpy(), ref, tol)


@pytest.mark.gpu
def test_streams_and_graph():
    """A step of append and attention captured once and replayed as the sequences
    grow, with eager calls between the replays: every replay is the eager result."""
    import torch
    # (capacity for 4 steps more)
    bt = Batch([(1, 2004), (1, 37), (1, 133)], 16, 18, kv_heads=2)
    bt.lens -= 4
    a = bt.gpu()
    inv = torch.tensor(10000.0 ** (-np.arange(32) / 32), dtype=torch.float32, device="cuda")
    side = torch.cuda.Stream()
    x = [torch.zeros(3, h, 64, device="cuda") for h in (4, 2, 2)]

    def step(c):
        q = hk.append_kv(*x, inv_freq=inv, **c)
        return hk.paged_attention(q, max_kv_len=2004, **c)

    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        step(a)
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            out = step(a)
    eager = {k: None if v is None else v.clone() for k, v in a.items()}
    for i in range(4):
        gen = torch.Generator(device="cuda").manual_seed(i)
        for t in x:
            t.copy_(torch.randn(t.shape, generator=gen, device="cuda"))
        a["kv_lens"] += 1
        eager["kv_lens"] += 1
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        want = step(eager)
        torch.cuda.synchronize()
        assert torch.equal(out, want)
        for name in ("k_cache", "v_cache"):
            assert torch.equal(a[name], eager[name])


# --- append ---------------------------------------------------------------------------

def rotate(x, pos, inv, style):
    x, r = x.astype(np.float64), 2 * len(inv)
    ang = (pos[:, None] * inv.astype(np.float64))[:, None]
    c, s = np.cos(ang), np.sin(ang)
    i = np.arange(r // 2)
    i0, i1 = (i, i + r // 2) if style == "halves" else (2 * i, 2 * i + 1)
    y = x.copy()
    y[..., i0], y[..., i1] = x[..., i0] * c - x[..., i1] * s, x[..., i1] * c + x[..., i0] * s
    return y


def codes(x):
    """The int8 codes and scales of rows x (fp32)."""
    amax = np.abs(x).max(-1)
    s = np.where(np.isfinite(x).all(-1), amax / np.float32(127), np.float32("nan"))
    y = x / np.where(s > 0, s, np.float32(1))[..., None]
    c = np.trunc(y + np.copysign(np.float32(0.5), y))
    c = np.where((s > 0)[..., None], np.clip(c, -127, 127), 0)
    return c.astype(np.int8), s.astype(np.float32)


def run_append(bt, q, k, v, inv, style, **kw):
    import torch
    a = bt.gpu()
    up = lambda t: None if t is None else torch.from_numpy(t).cuda()  # noqa: E731
    got = hk.append_kv(up(q), up(k), up(v), inv_freq=up(inv), style=style, **a, **kw)
    torch.cuda.synchronize()
    return got, a


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("style", ["halves", "pairs"])
@pytest.mark.parametrize("heads,kv_heads,dim,rot", [(4, 2, 64, 64), (3, 3, 40, 40), (10, 2, 80, 32),
                                                    (7, 1, 96, 18), (1, 1, 256, 256), (4, 4, 8, 2),
                                                    (32, 8, 128, 128), (4, 2, 64, 0)])
def test_append(heads, kv_heads, dim, rot, style, kind):
    seqs = [(1, 1), (5, 37), (0, 9), (1, 100), (3, 1), (20, 20)]
    bt = Batch(seqs, 8, 20, kv_heads=kv_heads, dim=dim, kind=kind)
    rng = np.random.default_rng(20)
    q, k, v = (rng.standard_normal((bt.tokens, h, dim)).astype(np.float32)
               for h in (heads, kv_heads, kv_heads))
    inv = (10000.0 ** (-np.arange(0, rot, 2) / max(rot, 1))).astype(np.float32) if rot else None
    got, a = run_append(bt, q, k, v, inv, style)
    none = np.zeros(0, np.float32)
    pos = np.concatenate([np.arange(kv - n, kv) for n, kv in seqs])
    ref = rotate(q, pos, none if inv is None else inv, style)
    # one rounding to fp32 (the 64-bit roundings before it are 2^-29 of that)
    assert np.all(np.abs(got.cpu().numpy() - ref) <= EPS * np.abs(ref) * 1.000001 + 1e-14)
    rk = rotate(k, pos, none if inv is None else inv, style).astype(np.float32)
    want = {"k": bt.k.copy(), "v": bt.v.copy()}
    scales = {} if kind == "fp16" else {"k": bt.ks.copy(), "v": bt.vs.copy()}
    for b, (n, kv) in enumerate(seqs):
        for i in range(n):
            p, t = kv - n + i, bt.cu[b] + i
            if p < 0:
                continue  # no place
            pg, sl = bt.place(b, p)
            for name, x in (("k", rk[t]), ("v", v[t])):
                if kind == "fp16":
                    want[name][pg, :, sl] = x.astype(np.float16)
                else:
                    want[name][pg, :, sl], scales[name][pg, :, sl] = codes(x)
    for name in ("k", "v"):
        c = a[name + "_cache"].cpu().numpy()
        if kind == "fp16" and name == "k":
            # a value within 2^-53 of the middle of two fp32 may go either way, and its
            # fp16 with it
            d = np.abs(c.astype(np.float64) - want[name].astype(np.float64))
            assert np.all(d <= 2.0 ** -10 * np.abs(want[name].astype(np.float64)) + 2.0 ** -24)
            assert np.mean(c != want[name]) < 1e-4
        else:
            assert np.array_equal(c, want[name])
        if scales:
            assert np.array_equal(a[name + "_scale"].cpu().numpy(), scales[name])


@pytest.mark.gpu
@pytest.mark.parametrize("pos", [131071, 999999, 2 ** 31 - 70000])
def test_append_far_positions(pos):
    """Angles far out keep 64-bit precision: the products differ from the formula's by
    the rounding of pos * inv_freq to 64 bits at most.  Earlier pages are not there."""
    page = 65536
    width = -(-(pos + 1) // page)
    bt = Batch([(1, 1)], page, 21, extra=0, kv_heads=1, dim=64)
    bt.table = np.full((1, width), -1, np.int32)
    bt.table[0, pos // page] = 0
    bt.lens[0], bt.seqs = pos + 1, [(1, pos + 1)]
    rng = np.random.default_rng(21)
    q, k, v = (rng.standard_normal((1, h, 64)).astype(np.float32) for h in (2, 1, 1))
    inv = (10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)
    got, a = run_append(bt, q, k, v, inv, "halves")
    p = np.array([pos])
    ref = rotate(q, p, inv, "halves")
    lim = EPS * np.abs(ref) + pos * 2.0 ** -52 * np.abs(q).max() + 1e-14
    assert np.all(np.abs(got.cpu().numpy() - ref) <= lim)
    c = a["k_cache"].cpu().numpy()[0, 0, pos % page].astype(np.float64)
    rk = rotate(k, p, inv, "halves")[0, 0]
    assert np.all(np.abs(c - rk) <= (2.0 ** -11 + 2 * EPS) * np.abs(rk) + 2.0 ** -25)


@pytest.mark.gpu
def test_append_int8_edges():
    """Rows of zeros, of the smallest and largest values, halves, infinities and NaN."""
    dim = 32
    rows = [np.zeros(dim), np.full(dim, 1e-45), np.full(dim, 1e-40), np.full(dim, 3e38),
            np.arange(dim) + 0.5, np.where(np.arange(dim) == 3, 127.0, np.arange(dim) / 2),
            np.where(np.arange(dim) == 5, np.inf, 1.0), np.where(np.arange(dim) == 5, np.nan, 1.0),
            -np.arange(dim) / 2.0 - 111.5, np.where(np.arange(dim) == 5, -np.inf, np.nan)]
    v = np.array(rows, np.float32)[:, None]
    n = len(rows)
    bt = Batch([(n, n)], 16, 22, kv_heads=1, dim=dim, kind="int8")
    _, a = run_append(bt, None, v.copy(), v, None, "halves")
    with np.errstate(invalid="ignore", over="ignore"):
        c, s = codes(v)
    pg, sl = bt.place(0, np.arange(n))
    for name in ("k", "v"):
        assert np.array_equal(a[name + "_scale"].cpu().numpy()[pg, :, sl], s, equal_nan=True)
        assert np.array_equal(a[name + "_cache"].cpu().numpy()[pg, :, sl], c)


@pytest.mark.gpu
def test_append_bad_places():
    """Tokens in pages that are none, past the table or at negative positions are not
    stored (nothing else of the cache changes); their q is rotated all the same."""
    bt = Batch([(2, 20), (2, 20), (3, 2), (1, 16)], 16, 23)
    bt.table[0, 1], bt.table[1, 1] = -1, bt.pages
    bt.lens[3] = 2 ** 31 - 1
    rng = np.random.default_rng(23)
    q, k, v = (rng.standard_normal((bt.tokens, h, 64)).astype(np.float32) for h in (4, 2, 2))
    inv = (10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)
    got, a = run_append(bt, q, k, v, inv, "halves")
    pos = np.array([18, 19, 18, 19, -1, 0, 1, 2 ** 31 - 2])
    ref = rotate(q, pos, inv, "halves")
    lim = EPS * np.abs(ref) + pos[:, None, None] * 2.0 ** -52 * np.abs(q).max() + 1e-14
    assert np.all(np.abs(got.cpu().numpy() - ref) <= lim)
    want = bt.v.copy()
    for t, p in ((5, 0), (6, 1)):
        pg, sl = bt.place(2, p)
        want[pg, :, sl] = v[t].astype(np.float16)
    assert np.array_equal(a["v_cache"].cpu().numpy(), want)


@pytest.mark.gpu
def test_append_in_place_and_strides():
    """q rotated in place, all three out of one fused projection at an odd offset, a
    pool of pages and layers; the same values as from tensors of their own."""
    import torch
    bt = Batch([(5, 37), (1, 100)], 16, 24)
    rng = np.random.default_rng(24)
    q, k, v = (rng.standard_normal((6, h, 64)).astype(np.float32) for h in (4, 2, 2))
    inv = (10000.0 ** (-np.arange(0, 64, 2) / 64)).astype(np.float32)
    want, wa = run_append(bt, q, k, v, inv, "halves")
    for shift in (0, 1):
        fused = torch.zeros(6, 8 * 64 + 4 + shift, device="cuda")
        part = [fused[:, shift + o * 64:shift + (o + h) * 64].view(6, h, 64)
                for o, h in ((0, 4), (4, 2), (6, 2))]
        for p, x in zip(part, (q, k, v)):
            p.copy_(torch.from_numpy(x))
        a = bt.gpu()
        pools = [torch.zeros((bt.pages, 2, *a[n].shape[1:]), dtype=torch.float16, device="cuda")
                 for n in ("k_cache", "v_cache")]
        for n, p in zip(("k_cache", "v_cache"), pools):
            p[:, 1].copy_(a[n])
            a[n] = p[:, 1]
        got = hk.append_kv(*part, inv_freq=torch.from_numpy(inv).cuda(), out=part[0], **a)
        assert torch.equal(got, want)
        for n, p in zip(("k_cache", "v_cache"), pools):
            assert torch.equal(p[:, 1], wa[n]) and not p[:, 0].any()


# --- refusals (no GPU) --------------------------------------------------------------------

def _kv(**kw):
    c = dict(dtype=0, k=1 << 40, v=2 << 40, k_scale=None, v_scale=None, pages=4, kv_heads=2,
             page_size=16, head_dim=64, k_page_stride=0, v_page_stride=0, k_scale_page_stride=0,
             v_scale_page_stride=0)
    b = dict(cu_q=3 << 40, kv_lens=4 << 40, page_table=5 << 40, batch=2, table_width=4, tokens=3)
    for k, v in kw.items():
        (c if k in c else b)[k] = v
    return _lib.KvCache(**c), _lib.KvBatch(**b)


BAD = [dict(dtype=2), dict(head_dim=0), dict(head_dim=60), dict(head_dim=264), dict(page_size=0),
       dict(page_size=24), dict(page_size=1 << 17), dict(kv_heads=0), dict(k=None), dict(v=None),
       dict(k=(1 << 40) + 8), dict(cu_q=None), dict(kv_lens=None), dict(page_table=None),
       dict(dtype=1), dict(dtype=1, k_scale=6 << 40), dict(k_page_stride=64),
       dict(v_page_stride=2 * 16 * 64 + 4), dict(pages=1 << 40), dict(batch=1 << 40),
       dict(tokens=1 << 40), dict(table_width=1 << 40), dict(table_width=1 << 28),
       dict(dtype=1, k_scale=6 << 40, v_scale=7 << 40, k_scale_page_stride=16)]
Q, K, V, F, O = ((n << 40) for n in (8, 9, 10, 11, 12))


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_c_refuses_cache_and_batch(bad):
    lib = _lib.load()
    c, b = (ctypes.byref(x) for x in _kv(**bad))
    d = bad.get("head_dim", 64)
    assert lib.hypno_hip_append_kv_dev(c, b, O, 4 * d, Q, 4 * d, 4, K, 2 * d, V, 2 * d, F, 0, 0,
                                       None) == 22
    assert b"append_kv" in lib.hypno_hip_last_error()
    assert lib.hypno_hip_paged_attention_dev(O, Q, 4 * d, 4, c, b, 0.1, 0, 0, None) == 22
    assert b"paged_attention" in lib.hypno_hip_last_error()


def test_c_refuses_arguments():
    lib = _lib.load()
    c, b = (ctypes.byref(x) for x in _kv())

    def append(o=O, os=256, q=Q, qs=256, h=4, k=K, ks=128, v=V, vs=128, f=F, rot=64, style=0,
               c=c, b=b):
        return lib.hypno_hip_append_kv_dev(c, b, o, os, q, qs, h, k, ks, v, vs, f, rot, style,
                                           None)

    def attention(o=O, q=Q, qs=256, h=4, c=c, b=b):
        return lib.hypno_hip_paged_attention_dev(o, q, qs, h, c, b, 0.1, 0, 0, None)

    for kw in (dict(o=None), dict(q=None), dict(k=None), dict(v=None), dict(f=None),
               dict(os=255), dict(qs=255), dict(ks=127), dict(vs=127), dict(rot=63),
               dict(rot=66), dict(style=2), dict(h=70000), dict(c=None), dict(b=None),
               dict(o=Q + 4), dict(o=Q, os=300), dict(o=K - 4), dict(o=V + 8), dict(o=1 << 40),
               dict(o=3 << 40), dict(q=(2 << 40) + 4), dict(k=1 << 40), dict(v=4 << 40),
               dict(f=5 << 40), dict(o=F), dict(qs=1 << 62)):
        assert append(**kw) == 22, kw
    for kw in (dict(o=None), dict(q=None), dict(qs=255), dict(h=3), dict(h=0), dict(h=70000),
               dict(c=None), dict(b=None), dict(o=Q + 4), dict(o=Q), dict(o=2 << 40),
               dict(o=5 << 40), dict(qs=1 << 62)):
        assert attention(**kw) == 22, kw
    # Nothing to do succeeds without a device.
    for kw in (dict(tokens=0), dict(batch=0)):
        c0, b0 = (ctypes.byref(x) for x in _kv(**kw))
        assert append(c=c0, b=b0) == 0 and attention(c=c0, b=b0) == 0


def test_python_refuses_host_tensors():
    import torch
    x = torch.zeros(2, 4, 64)
    c = torch.zeros(4, 4, 16, 64, dtype=torch.float16)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="GPU"):
        hk.append_kv(x, x, x, c, c, i[None], i[:1], i)
    with pytest.raises(ValueError, match="GPU"):
        hk.paged_attention(x, c, c, i[None], i[:1], i)
    with pytest.raises(ValueError, match="style"):
        hk.append_kv(x, x, x, c, c, i[None], i[:1], i, style="other")


@pytest.mark.gpu
def test_python_refusals():
    import torch
    bt = Batch([(2, 20)], 16, 30)
    a = bt.gpu()
    q, k = torch.zeros(2, 4, 64, device="cuda"), torch.zeros(2, 2, 64, device="cuda")
    f = torch.zeros(32, device="cuda")
    i8 = {**a, "k_cache": a["k_cache"].to(torch.int8), "v_cache": a["v_cache"].to(torch.int8)}
    sc = torch.zeros(bt.pages, 2, 16, device="cuda")
    for kw in (dict(k_cache=a["k_cache"].float(), v_cache=a["v_cache"].float()),
               dict(v_cache=a["v_cache"][:1]), dict(v_cache=a["v_cache"].to(torch.int8)),
               dict(k_cache=a["k_cache"].transpose(2, 3)), dict(k_cache=a["k_cache"].cpu()),
               dict(page_table=a["page_table"].long()), dict(page_table=a["page_table"][0]),
               dict(kv_lens=a["kv_lens"].repeat(2)), dict(cu_q=a["cu_q"][:1]),
               dict(cu_q=a["cu_q"].cpu()), dict(k_scale=sc), i8, {**i8, "k_scale": sc},
               {**i8, "k_scale": sc, "v_scale": sc[:, :1]},
               {**i8, "k_scale": sc, "v_scale": sc.half()}):
        with pytest.raises(ValueError):
            hk.append_kv(q, k, k, **{**a, **kw})
        with pytest.raises(ValueError):
            hk.paged_attention(q, **{**a, **kw})
    for args, kw in (((q.half(), k, k), {}), ((q[:1], k, k), {}), ((q, k[:1], k), {}),
                     ((q, k, k[..., :32]), {}), ((q, q, q), {}), ((q.transpose(0, 1), k, k), {}),
                     ((q, k, k), dict(inv_freq=f.double())), ((q, k, k), dict(inv_freq=f[::2])),
                     ((q, k, k), dict(inv_freq=torch.zeros(33, device="cuda"))),
                     ((q, k, k), dict(out=q[:1])), ((None, k, k), dict(out=q)),
                     ((q.cpu(), k, k), {})):
        with pytest.raises(ValueError):
            hk.append_kv(*args, **a, **kw)
    for x, kw in ((q[:, :3], {}), (q[..., :32], {}), (q.half(), {}), (q, dict(window=-1)),
                  (q, dict(max_kv_len=-1)), (q, dict(out=q.half())), (q, dict(out=q[:1])),
                  (q.cpu(), {})):
        with pytest.raises(ValueError):
            hk.paged_attention(x, **a, **kw)
    with pytest.raises(hk.HypnoHipError) as e:
        hk.paged_attention(q, out=q, **a)
    assert e.value.status == 22
