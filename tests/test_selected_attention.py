"""key_bounds, select_pages and selected_attention against their definitions: whole numbers
and codes bit for bit, attention within test_paged_attention's bounds; runs of them
together, and their refusals."""
import ctypes
import math
import os
import subprocess
import sys

import numpy as np
import pytest

import hypno_amd as hk
from hypno_amd import _lib, attention
from conftest import ROOT
from test_fp4_cache import Batch4
from test_paged_attention import EPS, O, Q, Batch, _kv, check, queries

KINDS = ["fp16", "int8", "fp4"]
FMAX = np.float32(3.4028234663852886e38)


def batch(kind, seqs, page, seed, **kw):
    return Batch4(seqs, page, seed, **kw) if kind == "fp4" else Batch(seqs, page, seed, kind=kind,
                                                                      **kw)


def keys(bt, b, g, p):
    """float32 keys, as key_bounds takes them."""
    if bt.kind != "int8":
        with np.errstate(over="ignore"):
            return bt.values(b, g, p)[0].astype(np.float32)
    pg, sl = bt.place(b, p)
    with np.errstate(invalid="ignore"):
        return bt.k[pg, g, sl].astype(np.float32) * bt.ks[pg, g, sl][:, None]


def codes8(x):
    """Codes and scale of float32 x by the 8-bit rule."""
    top = np.abs(x).max()
    if not np.isfinite(top):
        return np.zeros(x.shape, np.int8), np.float32(np.nan)
    s = np.float32(top) / np.float32(127)
    if s == 0:
        return np.zeros(x.shape, np.int8), s
    y = (x.astype(np.float32) / s).astype(np.float64)
    return np.clip(np.sign(y) * np.floor(np.abs(y) + 0.5), -127, 127).astype(np.int8), s


def bounds_of(bt, codes, scale):
    """What key_bounds makes of codes and scale."""
    codes, scale = codes.copy(), scale.copy()
    for b, (n, kv) in enumerate(bt.seqs):
        if n <= 0 or kv <= 0:
            continue
        for at in range(max(kv - n, 0) // bt.page, (kv - 1) // bt.page + 1):
            page = bt.table[b, at] if at < bt.table.shape[1] else -1
            if not 0 <= page < bt.pages:
                continue
            p = np.arange(at * bt.page, min(kv, (at + 1) * bt.page))
            for g in range(bt.kv_heads):
                k = keys(bt, b, g, p)
                codes[page, g], scale[page, g] = codes8(np.stack([k.min(0), k.max(0)])
                                                        if np.isfinite(k).all() else k[:2] * np.nan)
    return codes, scale


def run_bounds(bt, codes, scale, **kw):
    import torch
    a = bt.gpu()
    c, s = torch.from_numpy(codes).cuda(), torch.from_numpy(scale).cuda()
    a.update(kw)
    assert hk.key_bounds(a["k_cache"], c, s, a["page_table"], a["kv_lens"], a["cu_q"],
                         k_scale=a["k_scale"]) is None
    torch.cuda.synchronize()
    return c.cpu().numpy(), s.cpu().numpy()


def old_bounds(bt, seed=1):
    rng = np.random.default_rng(seed)
    return (rng.integers(-127, 128, (bt.pages, bt.kv_heads, 2, bt.dim)).astype(np.int8),
            rng.random((bt.pages, bt.kv_heads)).astype(np.float32))


RAGGED = [(3, 50), (1, 1), (40, 40), (0, 7), (2, 18), (1, 33), (5, 3), (2, 0), (100, 301), (1, 64)]


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kv_heads,dim,page", [(2, 64, 16), (1, 128, 64), (3, 32, 32), (1, 256, 16),
                                               (5, 160, 128)])
def test_bounds(kind, kv_heads, dim, page):
    bt = batch(kind, RAGGED, page, 40, kv_heads=kv_heads, dim=dim)
    old = old_bounds(bt)
    for got, want in zip(run_bounds(bt, *old), bounds_of(bt, *old)):
        assert np.array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("dim,page", [(8, 1), (40, 4), (80, 8), (24, 512), (200, 2)])
def test_bounds_of_odd_sizes(kind, dim, page):
    bt = batch(kind, RAGGED, page, 41, kv_heads=2, dim=dim)
    old = old_bounds(bt)
    for got, want in zip(run_bounds(bt, *old), bounds_of(bt, *old)):
        assert np.array_equal(got, want)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_bounds_of_odd_values(kind):
    """NaN past the end, NaN and infinities among the keys, zeros, keys of one sign, pages
    that are none."""
    bt = batch(kind, [(200, 200), (90, 90)], 16, 42)
    last, slots = bt.table[0, 12], slice(8, 16)
    scale = {"fp16": bt.k, "int8": bt.ks, "fp4": bt.ks}[kind]
    part = (lambda pg, g, sl: (pg, g, sl)) if kind != "fp4" else (lambda pg, g, sl: (pg, g, 1, sl))
    scale[part(last, slice(None), slots) if kind != "fp4" else (last, slice(None), slice(None),
                                                               slots)] = np.nan
    scale[part(bt.table[0, 1], 0, 3)] = np.nan
    scale[part(bt.table[0, 2], 1, 15)] = np.inf
    if kind == "fp16":
        bt.k[bt.table[0, 3]] = 0
        bt.k[bt.table[0, 4]] = np.abs(bt.k[bt.table[0, 4]])
        bt.k[bt.table[0, 5]] = -np.abs(bt.k[bt.table[0, 5]]) * np.float16(1e-4)
    bt.table[0, 6], bt.table[1, 2] = -1, bt.pages
    if kind == "fp4":  # (an infinite scale times a code of 0: NaN; no code at all: -0)
        bt.k[bt.table[0, 2], 1, 15] |= 0x11
    old = old_bounds(bt)
    got, want = run_bounds(bt, *old), bounds_of(bt, *old)
    assert np.array_equal(got[1], want[1], equal_nan=True) and np.array_equal(got[0], want[0])
    assert np.isnan(got[1][bt.table[0, 1], 0]) and np.isnan(got[1][bt.table[0, 2], 1])
    assert not np.isnan(got[1][last]).any()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 700])
def test_bounds_of_many(n):
    """More pages than work-groups; a pool of layers."""
    import torch
    bt = Batch([(n, 700 + i) for i in range(33)], 16, 43, kv_heads=3, dim=64)
    old = old_bounds(bt)
    want = bounds_of(bt, *old)
    a = bt.gpu()
    pool = [torch.zeros((x.shape[0], 2, *x.shape[1:]), dtype=x.dtype, device="cuda")
            for x in (a["k_cache"], torch.from_numpy(old[0]), torch.from_numpy(old[1]))]
    for p, x in zip(pool, (a["k_cache"], torch.from_numpy(old[0]), torch.from_numpy(old[1]))):
        p[:, 1].copy_(x)
    hk.key_bounds(pool[0][:, 1], pool[1][:, 1], pool[2][:, 1], a["page_table"], a["kv_lens"],
                  a["cu_q"])
    for got, ref in zip(pool[1:], want):
        assert np.array_equal(got[:, 1].cpu().numpy(), ref) and not got[:, 0].any()


# --- selection ----------------------------------------------------------------------------------

def scores(q, codes, scale):
    """float32 scores [P] of one token's heads q [G, D] (of one kv head) for pages' bounds."""
    best = None
    for x in q:
        c, s = codes8(x)
        if not np.isfinite(s):
            s = np.float32(0)
        c = c.astype(np.int64)
        # (by the code's sign also where a lower bound is above its upper one)
        whole = np.where(c < 0, c * codes[:, 0].astype(np.int64), c * codes[:, 1].astype(np.int64))
        whole = whole.sum(-1)
        with np.errstate(over="ignore"):
            y = whole.astype(np.float32) * s
        best = y if best is None else np.maximum(best, y)
    with np.errstate(all="ignore"):
        y = best * scale
    y[np.isnan(y)] = FMAX
    return np.clip(y, -FMAX, FMAX)


def select(bt, q, codes, scale, count, first=1, last=1, max_kv=None):
    T, H = q.shape[:2]
    G = H // bt.kv_heads
    out = np.full((T, bt.kv_heads, count), -77, np.int32)
    for b, (n, kv) in enumerate(bt.seqs):
        row = bt.table[b]
        if max_kv:
            row = row[:-(-max_kv // bt.page)]
        there = (row >= 0) & (row < bt.pages)
        ids = np.where(there, row, 0)
        for i in range(n):
            pos, t = kv - n + i, bt.cu[b] + i
            own = pos // bt.page if pos >= 0 else -1
            kept = [p for p in range(own + 1) if p < first or p > own - last]
            for g in range(bt.kv_heads):
                free = np.array([p for p in range(min(own + 1, len(row)))
                                 if p >= first and p <= own - last and there[p]], np.int64)
                pick = []
                if len(free):
                    s = scores(q[t, g * G:g * G + G], codes[ids[free], g], scale[ids[free], g])
                    pick = list(free[np.argsort(-s.astype(np.float64), kind="stable")]
                                [:count - first - last])
                pick = sorted(kept + pick)
                out[t, g] = pick + [-1] * (count - len(pick))
    return out


def run_select(bt, q, codes, scale, count, first=1, last=1, max_kv=None, **kw):
    import torch
    a = bt.gpu()
    T = q.shape[0]
    out = torch.full((T, bt.kv_heads, count), -77, dtype=torch.int32, device="cuda")
    got = hk.select_pages(torch.from_numpy(q).cuda(), torch.from_numpy(codes).cuda(),
                          torch.from_numpy(scale).cuda(), bt.page, a["page_table"], a["kv_lens"],
                          a["cu_q"], count, first=first, last=last, max_kv_len=max_kv, out=out)
    torch.cuda.synchronize()
    assert got is out
    return got.cpu().numpy()


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (8, 1, 128), (3, 3, 40), (10, 2, 80),
                                                (7, 1, 96), (2, 1, 256), (4, 4, 8), (20, 1, 64),
                                                (33, 1, 136), (5, 1, 24), (16, 1, 32)])
@pytest.mark.parametrize("count,first,last", [(1, 0, 1), (2, 1, 1), (5, 1, 2), (12, 0, 3), (64, 2, 2),
                                              (8, 4, 4)])
def test_select(heads, kv_heads, dim, count, first, last):
    bt = Batch([(1, 1), (1, 300), (3, 50), (20, 200), (0, 9), (1, 16), (2, 17), (5, 3), (1, 33)], 16,
               44, kv_heads=kv_heads, dim=dim)
    q, b = queries(bt.tokens, heads, dim, 44), old_bounds(bt)
    assert np.array_equal(run_select(bt, q, *b, count, first, last),
                          select(bt, q, *b, count, first, last))


@pytest.mark.gpu
@pytest.mark.parametrize("n,kv,page,count", [(1, 20000, 16, 64), (1, 70001, 16, 1000), (2, 5000, 1, 33),
                                             (30, 3000, 2, 20), (3, 40000, 16, 128)])
def test_select_of_many(n, kv, page, count):
    """Long contexts: several waves search one token's scores."""
    bt = Batch([(n, kv), (1, kv // 3)], page, 45, kv_heads=1, dim=32)
    q, b = queries(bt.tokens, 4, 32, 45), old_bounds(bt)
    want = select(bt, q, *b, count, 1, 2)
    assert np.array_equal(run_select(bt, q, *b, count, 1, 2), want)
    assert np.array_equal(run_select(bt, q, *b, count, 1, 2, max_kv=kv), want)


@pytest.mark.gpu
@pytest.mark.parametrize("heads,kv_heads,n,kv", [(2, 2, 40, 3000), (3, 1, 300, 8000), (4, 1, 70, 5100),
                                                 (20, 1, 33, 21000)])
def test_select_of_chunks(heads, kv_heads, n, kv):
    """Chunks over many pages: scores by one kernel and the choice by another, a wave a token."""
    bt = Batch([(n, kv), (1, kv // 2), (n // 2, kv // 3)], 2, 49, kv_heads=kv_heads, dim=16)
    q, b = queries(bt.tokens, heads, 16, 49), old_bounds(bt)
    assert np.array_equal(run_select(bt, q, *b, 40, 1, 2), select(bt, q, *b, 40, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("kv", [500, 9000])
def test_select_ties(kv):
    """Equal scores: the lower page.  Scores that are 0 with either sign are equal."""
    bt = Batch([(2, kv)], 4, 46, kv_heads=2, dim=16)
    codes, scale = old_bounds(bt)
    codes[:], scale[:] = codes[:1], 0.5
    row = bt.table[0]
    codes[row[::7]] = codes[row[0]] // 2
    scale[row[3::5]] = 0.0
    q = queries(2, 4, 16, 46)
    for count in (3, 20, 60):
        assert np.array_equal(run_select(bt, q, codes, scale, count), select(bt, q, codes, scale, count))
    q[:] = 0
    want = np.array([*range(19), (kv - 1) // 4])
    got = run_select(bt, q, codes, scale, 20)
    assert (got[1] == want).all()


@pytest.mark.gpu
def test_select_odd_values():
    """Pages that are none, bounds that are NaN or infinite, queries that hold NaN or
    infinities, or are zero; a bound of kv_lens that is too low."""
    bt = Batch([(2, 900), (1, 400)], 16, 47, kv_heads=1, dim=64)
    codes, scale = old_bounds(bt)
    bt.table[0, [3, 4, 20]] = -1, bt.pages, 2 ** 31 - 1
    bt.table[0, 56] = -1                       # the token's own: always selected
    scale[bt.table[0, 10]], scale[bt.table[0, 30]] = np.nan, np.inf
    scale[bt.table[1, 5]] = 3e38
    q = queries(3, 4, 64, 47)
    q[0, 1, 5], q[1, 2, 63], q[1, 3] = np.nan, np.inf, 0
    q[2] *= np.float32(1e30)
    for count in (2, 4, 9, 40, 100):
        want = select(bt, q, codes, scale, count)
        assert np.array_equal(run_select(bt, q, codes, scale, count), want)
    assert {10, 30} <= set(select(bt, q, codes, scale, 4)[0, 0])
    assert np.array_equal(run_select(bt, q, codes, scale, 9, max_kv=300),
                          select(bt, q, codes, scale, 9, max_kv=300))


@pytest.mark.gpu
def test_select_leaves_other_rows():
    import torch
    bt = Batch([(1, 100), (0, 50)], 16, 48, kv_heads=2, dim=64)
    q, (codes, scale) = queries(4, 4, 64, 48), old_bounds(bt)
    got = run_select(bt, q, codes, scale, 5)
    assert np.array_equal(got[:1], select(bt, q[:1], codes, scale, 5)) and (got[1:] == -77).all()
    bt.lens[0] = 2 ** 31 - 1  # longer than its table row
    got = run_select(bt, q, codes, scale, 5)
    assert list(got[0, 0]) == [0, *got[0, 0, 1:4], (2 ** 31 - 2) // 16]
    # fused queries
    fused = torch.randn(1, 700, device="cuda")
    view = fused[:, 1:257].view(1, 4, 64)
    a = bt.gpu()
    g = hk.select_pages(view, torch.from_numpy(codes).cuda(), torch.from_numpy(scale).cuda(), 16,
                        a["page_table"], a["kv_lens"], a["cu_q"][:3], 5)
    assert g.shape == (1, 2, 5) and g.dtype == torch.int32


# --- attention over them --------------------------------------------------------------------------

def attend_selected(q, bt, sel, scale=None):
    """The formula in 64 bits, and how far an fp32 computation may be from it (as
    test_paged_attention.attend: the same sums over fewer positions)."""
    T, H, D = q.shape
    scale = 1.0 / math.sqrt(D) if scale is None else scale
    out, tol = np.zeros((T, H, D)), np.zeros((T, H, D))
    per = H // bt.kv_heads
    for b, (n, kv) in enumerate(bt.seqs):
        for i in range(n):
            pos, t = kv - n + i, bt.cu[b] + i
            for g in range(bt.kv_heads):
                p = [np.arange(j * bt.page, min((j + 1) * bt.page, pos + 1))
                     for j in sel[t, g].tolist()
                     if 0 <= j and j * bt.page <= pos]
                p = np.concatenate(p) if p else np.zeros(0, int)
                if not len(p):
                    continue
                k, v = bt.values(b, g, p)
                for h in range(g * per, g * per + per):
                    x = q[t, h].astype(np.float64)
                    s = (k @ x) * scale
                    size = (np.abs(k) @ np.abs(x)).max() * abs(scale)
                    w = np.exp(s - s.max())
                    w /= w.sum()
                    out[t, h] = w @ v
                    off = 2 * size * (8 * math.sqrt(D) + 8) + 16 * math.sqrt(len(p)) + 16
                    tol[t, h] = EPS * off * (w @ np.abs(v)) + 1e-37
    return out, tol


def run_selected(bt, q, sel, **kw):
    import torch
    a = bt.gpu()
    out = torch.full(q.shape, 7.25, device="cuda")
    got = hk.selected_attention(torch.from_numpy(q).cuda(), a["k_cache"], a["v_cache"],
                                torch.from_numpy(sel).cuda(), a["page_table"], a["kv_lens"],
                                a["cu_q"], k_scale=a["k_scale"], v_scale=a["v_scale"], out=out, **kw)
    torch.cuda.synchronize()
    assert got is out
    return got.cpu().numpy()


def some_pages(bt, count, seed):
    """Random pages in no order, each at most once, with holes and pages ahead among them."""
    rng = np.random.default_rng(seed)
    sel = np.full((bt.tokens, bt.kv_heads, count), -1, np.int32)
    for b, (n, kv) in enumerate(bt.seqs):
        most = max(kv - 1, 0) // bt.page + 1
        for i in range(n):
            for g in range(bt.kv_heads):
                own = max(kv - n + i, 0) // bt.page
                p = rng.permutation(most)[:count]
                p[rng.random(len(p)) < 0.1] = -1
                if rng.random() < 0.7 and own not in p:
                    p[0] = own
                sel[bt.cu[b] + i, g, rng.permutation(count)[:len(p)]] = p
    return sel


SHAPES = [(4, 2, 64), (8, 1, 128), (3, 3, 32), (10, 2, 160), (7, 1, 96), (2, 1, 256), (20, 1, 64),
          (33, 1, 128)]
BATCHES = {"one": ([(1, 1)], 16, 1), "single": ([(1, 1), (1, 15), (1, 17), (1, 300), (1, 64)], 16, 7),
           "drafts": ([(3, 900), (2, 40), (5, 17), (0, 4), (5, 3), (1, 600)], 32, 6),
           "chunk": ([(70, 500)], 64, 5), "long": ([(1, 20000), (1, 7000)], 64, 128),
           "large pages": ([(2, 1500)], 512, 2)}


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("heads,kv_heads,dim", SHAPES)
@pytest.mark.parametrize("seqs", list(BATCHES))
def test_selected(seqs, heads, kv_heads, dim, kind):
    lens, page, count = BATCHES[seqs]
    bt = batch(kind, lens, page, 50, kv_heads=kv_heads, dim=dim)
    q, sel = queries(bt.tokens, heads, dim, 50), some_pages(bt, count, 50)
    check(run_selected(bt, q, sel), *attend_selected(q, bt, sel))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(3, 3, 40), (10, 2, 80), (4, 4, 8), (3, 1, 200)])
def test_selected_odd_dims(heads, kv_heads, dim, kind):
    bt = batch(kind, [(3, 900), (2, 40), (20, 170)], 16, 51, kv_heads=kv_heads, dim=dim)
    q, sel = queries(bt.tokens, heads, dim, 51), some_pages(bt, 9, 51)
    check(run_selected(bt, q, sel), *attend_selected(q, bt, sel))
    check(run_selected(bt, q, sel, scale=-0.05), *attend_selected(q, bt, sel, scale=-0.05))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_selected_numbers(kind):
    """Nothing but holes (zeros), a page twice (counts twice), numbers far out of range, all
    1024 places."""
    bt = batch(kind, [(6, 200)], 16, 52)
    q = queries(6, 4, 64, 52)
    sel = np.full((6, 2, 1024), -1, np.int32)
    sel[1, :, ::100] = 2 ** 31 - 1
    sel[2, :, 5], sel[2, :, 900] = 3, 3
    sel[2, 0, 77] = 4
    sel[3, :, :13] = np.arange(13)
    sel[4, :, -13:] = np.arange(13)[::-1]
    sel[4, 1, 0], sel[4, 1, 3] = -2 ** 31, 13
    sel[5, 0, 511] = 12
    ref, tol = attend_selected(q, bt, sel)
    got = run_selected(bt, q, sel)
    check(got, ref, tol)
    assert (got[:2] == 0).all() and (got[5, 2:] == 0).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("n", [1, 30])
def test_selected_hidden(kind, n):
    """Infinities and NaN in slots that are not seen and in pages that are not selected do no
    harm; in a seen one they give what the definition gives; a page that is none is NaN,
    selected or its sequence too long, and nothing where it is not selected."""
    bt = batch(kind, [(n, 75), (n, 200), (n, 75)], 16, 53)
    q = queries(bt.tokens, 4, 64, 53)
    sel = np.full((bt.tokens, 2, 4), -1, np.int32)
    for b, (_, kv) in enumerate(bt.seqs):
        for i in range(n):
            sel[bt.cu[b] + i] = [0, 2, 1, (kv - n + i) // 16]
            if (kv - n + i) // 16 < 3:
                sel[bt.cu[b] + i, :, 3] = -1
    ref, tol = attend_selected(q, bt, sel)

    def spoil(page, slots, x):
        for data, scale in ((bt.k, bt.ks), (bt.v, bt.vs)):
            if kind == "fp16":
                data[page, :, slots] = x
            elif kind == "int8":
                scale[page, :, slots] = x
            else:
                scale[page, :, :, slots] = x

    for b, (_, kv) in enumerate(bt.seqs):
        spoil(bt.table[b, kv // 16], slice(kv % 16, 16), np.nan if b else np.inf)
    spoil(bt.table[1, 7], slice(0, 16), np.nan)  # selected by nobody
    free = bt.table[1, 6]
    bt.table[1, 6] = -1
    check(run_selected(bt, q, sel), ref, tol)
    bt.table[1, 6] = free
    spoil(bt.table[1, 2], 5, np.nan)
    got = run_selected(bt, q, sel)
    assert np.isnan(got[n:2 * n]).all()
    check(got[:n], ref[:n], tol[:n])
    check(got[2 * n:], ref[2 * n:], tol[2 * n:])
    for none in (-1, bt.pages, 2 ** 31 - 1):
        bt.table[2, 1] = none
        got = run_selected(bt, q, sel)
        assert np.isnan(got[2 * n:]).all() and not np.isnan(got[:n]).any()
    bt.lens[0] = bt.table.shape[1] * 16 + 1
    assert np.isnan(run_selected(bt, q, sel)[:n]).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_selected_strides(kind):
    import torch
    bt = batch(kind, [(2, 100), (9, 61)], 16, 54)
    q, sel = queries(bt.tokens, 4, 64, 54), some_pages(bt, 4, 54)
    ref, tol = attend_selected(q, bt, sel)
    a = bt.gpu()
    fused = torch.randn(bt.tokens, 4 * 64 + 2 * 2 * 64 + 3, device="cuda")
    view = fused[:, 1:257].view(bt.tokens, 4, 64)
    view.copy_(torch.from_numpy(q))
    for name in ("k_cache", "v_cache", "k_scale", "v_scale"):
        if a[name] is not None:
            pool = torch.zeros((bt.pages, 3, *a[name].shape[1:]), dtype=a[name].dtype, device="cuda")
            pool[:, 1].copy_(a[name])
            a[name] = pool[:, 1]
    check(hk.selected_attention(view, selected=torch.from_numpy(sel).cuda(), **a).cpu().numpy(), ref,
          tol)
    # rows of no sequence
    out = torch.full((bt.tokens + 2, 4, 64), 7.25, device="cuda")
    more = torch.cat([view, view[:2]])
    hk.selected_attention(more, selected=torch.from_numpy(np.concatenate([sel, sel[:2]])).cuda(),
                          out=out, **a)
    check(out[:-2].cpu().numpy(), ref, tol)
    assert (out[-2:] == 7.25).all()


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_all_pages_are_all_of_the_context(kind):
    """With every page selected: paged_attention."""
    import torch
    bt = batch(kind, [(1, 500), (4, 333), (60, 60)], 32, 55, dim=128)
    q, a = torch.from_numpy(queries(bt.tokens, 4, 128, 55)).cuda(), bt.gpu()
    codes, scale = (torch.from_numpy(x).cuda() for x in old_bounds(bt))
    sel = hk.select_pages(q, codes, scale, 32, a["page_table"], a["kv_lens"], a["cu_q"], 16)
    got = hk.selected_attention(q, selected=sel, **a)
    ref, tol = attend_selected(q.cpu().numpy(), bt, sel.cpu().numpy())
    check(got.cpu().numpy(), ref, tol)
    check(hk.paged_attention(q, **a).cpu().numpy(), ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_together(kind):
    """A prompt in chunks and tokens one by one: append, bounds, choice, attention, each
    against its definition over what the calls before it left; then a token in a graph."""
    import torch
    bt = batch(kind, [(0, 0)], 16, 56, extra=30)
    bt.table = np.random.default_rng(56).permutation(bt.pages)[None].astype(np.int32)
    x = torch.from_numpy(np.random.default_rng(57).standard_normal((420, 8, 64)).astype(np.float32))
    x = x.cuda()
    a, done = bt.gpu(), 0
    codes, scale = (torch.from_numpy(y).cuda() for y in old_bounds(bt))
    where = {n: a[n] for n in ("page_table", "kv_lens", "cu_q")}

    def step(x):
        q, k, v = x.split([4, 2, 2], 1)
        q = hk.append_kv(q, k, v, **a)
        hk.key_bounds(a["k_cache"], codes, scale, k_scale=a["k_scale"], **where)
        sel = hk.select_pages(q, codes, scale, 16, count=6, last=2, **where)
        return q, sel, hk.selected_attention(q, selected=sel, **a)

    for n in (300, 100, 1, 1, 15, 1):
        bt.seqs, bt.cu = [(n, done + n)], np.array([0, n], np.int32)
        a["kv_lens"].fill_(done + n)
        a["cu_q"].copy_(torch.tensor([0, n], dtype=torch.int32))
        old = codes.cpu().numpy(), scale.cpu().numpy()
        q, sel, o = (y.cpu().numpy() for y in step(x[done:done + n]))
        bt.k, bt.v = a["k_cache"].cpu().numpy(), a["v_cache"].cpu().numpy()
        if kind != "fp16":
            bt.ks, bt.vs = a["k_scale"].cpu().numpy(), a["v_scale"].cpu().numpy()
        want = bounds_of(bt, *old)
        assert np.array_equal(codes.cpu().numpy(), want[0])
        assert np.array_equal(scale.cpu().numpy(), want[1])
        assert np.array_equal(sel, select(bt, q, *want, 6, 1, 2))
        check(o, *attend_selected(q, bt, sel))
        done += n
    token = x[:1].clone()
    a["cu_q"].copy_(torch.tensor([0, 1], dtype=torch.int32))
    a["kv_lens"].fill_(done + 1)
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(token)
    side.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        _, sel, o = step(token)
    for i in range(4):
        token.copy_(x[i:i + 1] * 2)
        a["kv_lens"].fill_(done + 1 + i)
        graph.replay()
        torch.cuda.synchronize()
        got = sel.clone(), o.clone()
        _, want, ref = step(token)
        assert torch.equal(got[0], want)
        # (the graph's positions may be split into other ranges)
        assert torch.allclose(got[1], ref, rtol=1e-4, atol=1e-5)


def long_step(bt, seed):
    """A function that chooses pages of a long context and attends to them and to all, and
    what it gives, checked."""
    import torch
    q, a = torch.from_numpy(queries(bt.tokens, 4, bt.dim, seed)).cuda(), bt.gpu()
    bounds = old_bounds(bt, seed)
    codes, scale = (torch.from_numpy(x).cuda() for x in bounds)
    where = {n: a[n] for n in ("page_table", "kv_lens", "cu_q")}

    def step():
        sel = hk.select_pages(q, codes, scale, bt.page, count=90, **where)
        return sel, hk.selected_attention(q, selected=sel, **a), hk.paged_attention(q, **a)

    want = [x.clone() for x in step()]
    x, sel = q.cpu().numpy(), want[0].cpu().numpy()
    assert np.array_equal(sel, select(bt, x, *bounds, 90))
    check(want[1].cpu().numpy(), *attend_selected(x, bt, sel))
    return step, want


def same(got, want):
    import torch
    assert torch.equal(got[0], want[0])
    for x, y in zip(got[1:], want[1:]):  # (other ranges of positions)
        assert torch.allclose(x, y, rtol=1e-4, atol=1e-5)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", KINDS)
def test_captured_without_a_workspace(kind):
    """On a stream that never had one: neither pages nor positions are split."""
    import torch
    step, want = long_step(batch(kind, [(1, 40000)], 16, 58, kv_heads=1), 58)
    side = torch.cuda.Stream()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        got = step()
    for _ in range(3):
        for x in got:
            x.zero_()
        graph.replay()
        torch.cuda.synchronize()
        same(got, want)
        same(step(), want)


@pytest.mark.gpu
def test_streams_side_by_side():
    """Each stream has a workspace of its own."""
    import torch
    steps = [long_step(batch(k, [(1, 30000 + 3000 * i)], 16, 59 + i, kv_heads=1), 59 + i)
             for i, k in enumerate(KINDS)]
    streams = [torch.cuda.Stream() for _ in steps]
    torch.cuda.synchronize()
    got = [[] for _ in steps]
    for _ in range(5):
        for (step, _), stream, out in zip(steps, streams, got):
            with torch.cuda.stream(stream):
                out.append(step())
    torch.cuda.synchronize()
    for (_, want), out in zip(steps, got):
        for x in out:
            assert all(torch.equal(y, z) for y, z in zip(x, want))


@pytest.mark.gpu
@pytest.mark.parametrize("args", [["--fp4"], ["--pages", "5"], ["--fp4", "--pages", "4"],
                                  ["--int8", "--pages", "3"]], ids=" ".join)
def test_example(args):
    """examples/paged_decode.py: a layer's prompt and tokens through all operators."""
    p = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "paged_decode.py"),
                        "--prompt", "70", "--tokens", "5", *args], capture_output=True, text=True,
                       timeout=100)
    assert p.returncode == 0, p.stderr
    assert ("agree" if args in (["--fp4"], ["--pages", "5"]) else "pages") in p.stdout


# --- arguments ------------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("fn", ["key_bounds", "select_pages", "selected_attention"])
def test_native_reader_answers_the_same(fn, monkeypatch):
    """Every argument in many wrong and unusual forms: the native reader and the Python
    functions raise the same or give the same."""
    import torch
    from test_attention_args import variants  # (its changes of names that a call has not: none)
    bt = Batch4([(2, 30), (1, 25)], 16, 60)
    q = torch.from_numpy(queries(3, 4, 64, 60)).cuda()
    codes, scale = (torch.from_numpy(x).cuda() for x in old_bounds(bt))
    sel = torch.from_numpy(some_pages(bt, 2, 60)).cuda()
    names = {"key_bounds": "k_cache bounds bounds_scale page_table kv_lens cu_q k_scale",
             "select_pages": "q bounds bounds_scale page_size page_table kv_lens cu_q count first "
                             "last max_kv_len out",
             "selected_attention": "q k_cache v_cache selected page_table kv_lens cu_q scale "
                                   "k_scale v_scale out"}[fn].split()

    def call(change):
        a = dict(bt.gpu(), q=q.clone(), bounds=codes.clone(), bounds_scale=scale.clone(),
                 page_size=16, count=3, first=1, last=1, max_kv_len=None, scale=None,
                 selected=sel.clone(), window=0,
                 out=torch.zeros(3, 2, 3, dtype=torch.int32, device="cuda")
                 if fn == "select_pages" else torch.zeros_like(q))
        change(a)
        try:
            got = getattr(hk, fn)(**{k: a[k] for k in names})
            torch.cuda.synchronize()
        except (ValueError, hk.HypnoHipError) as e:
            return type(e), str(e)
        return [None if t is None else t.clone() for t in (got, a["bounds"], a["bounds_scale"])]

    how = [f for n, f in variants() if n.split()[0] in names and n.split()[0] in
           ("q", "k_cache", "v_cache", "k_scale", "v_scale", "page_table", "kv_lens", "cu_q", "out",
            "max_kv_len", "scale")]
    for name in {"bounds", "bounds_scale", "selected"}.intersection(names):
        for f in (lambda t: t.int(), lambda t: t.float(), lambda t: t.cpu(), lambda t: t[:1],
                  lambda t: None, lambda t: t[..., :-1], lambda t: t[..., ::2], lambda t: t[None],
                  lambda t: t[:0], lambda t: torch.stack([t, t], 1)[:, 1], lambda t: 3,
                  lambda t: t.transpose(0, 1), lambda t: t[:, :, :0]):
            how.append(lambda a, name=name, f=f: a.update({name: f(a[name])}))
    for name in ("page_size", "count", "first", "last"):
        for x in (0, 1, 2, 3, 16, -1, 24, 1024, 1025, 2 ** 40, 2 ** 70, True, None, 2.0, np.int64(2)):
            how.append(lambda a, name=name, x=x: a.update({name: x, "out": None}))
    call(lambda a: None)
    native = attention._args
    assert native is not attention._NoArgs
    bad = []
    for i, change in enumerate(how):
        answers = []
        for reader in (native, attention._NoArgs):
            monkeypatch.setattr(attention, "_args", reader)
            try:
                answers.append(call(change))
            except (TypeError, IndexError, RuntimeError) as e:  # (the change itself)
                answers.append(type(e))
        got, want = answers
        same = got == want if not isinstance(got, list) or not isinstance(want, list) else \
            all(x is y is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
                for x, y in zip(got, want))
        if not same:
            bad.append((i, got, want))
    assert not bad, bad


def _bounds(**kw):
    o = dict(codes=13 << 40, scale=14 << 40, pages=4, kv_heads=2, page_size=16, head_dim=64,
             page_stride=0, scale_page_stride=0)
    o.update(kw)
    return _lib.KeyBounds(**o)


def test_c_refuses_bounds():
    lib = _lib.load()

    def call(o=None, c=None, b=None, kv={}, **kw):
        cc, bb = _kv(**kv)
        o = ctypes.byref(_bounds(**kw)) if o is None else o
        return lib.hypno_hip_key_bounds_dev(o, ctypes.byref(cc) if c is None else c,
                                            ctypes.byref(bb) if b is None else b, None)

    null = ctypes.c_void_p()
    for kw in (dict(o=null), dict(c=null), dict(b=null), dict(pages=3), dict(kv_heads=1),
               dict(page_size=32), dict(head_dim=128), dict(codes=None), dict(scale=None),
               dict(codes=(13 << 40) + 8), dict(page_stride=2 * 2 * 64 - 16),
               dict(page_stride=2 * 2 * 64 + 8), dict(scale_page_stride=1), dict(pages=1 << 40),
               dict(codes=1 << 40), dict(scale=3 << 40), dict(codes=14 << 40),
               dict(kv=dict(dtype=2)), dict(kv=dict(k=None)), dict(kv=dict(dtype=1)),
               dict(kv=dict(page_table=None))):
        assert call(**kw) == 22, kw
        assert b"key_bounds" in lib.hypno_hip_last_error()
    # V is not looked at; nothing to do succeeds without a device.
    for kv in (dict(tokens=0, v=None), dict(batch=0, v=None)):
        assert call(kv=kv) == 0
    assert call(kv=dict(pages=0, v=None), pages=0) == 0


def test_c_refuses_selection():
    lib = _lib.load()

    def call(sel=O, count=4, first=1, last=1, q=Q, qs=256, h=4, o=None, most=0, kv={}, **kw):
        b = ctypes.byref(_kv(**kv)[1])
        o = ctypes.byref(_bounds(**kw)) if o is None else o
        return lib.hypno_hip_select_pages_dev(sel, count, first, last, q, qs, h, o, b, most, None)

    for kw in (dict(sel=None), dict(q=None), dict(o=ctypes.c_void_p()), dict(count=0),
               dict(count=1025), dict(last=0), dict(first=4), dict(first=2 ** 63, last=2 ** 63),
               dict(last=5), dict(qs=255), dict(h=0), dict(h=3), dict(h=70000), dict(head_dim=60),
               dict(page_size=24), dict(codes=None), dict(scale=None), dict(sel=Q), dict(sel=Q - 4),
               dict(sel=13 << 40), dict(sel=14 << 40), dict(sel=4 << 40), dict(sel=3 << 40),
               dict(sel=5 << 40), dict(kv=dict(table_width=1 << 20)),
               dict(kv=dict(table_width=1 << 20), most=32768 * 16 + 1), dict(kv=dict(kv_lens=None))):
        assert call(**kw) == 22, kw
        assert b"select_pages" in lib.hypno_hip_last_error()
    for kv in (dict(tokens=0), dict(batch=0)):
        assert call(kv=kv) == 0


def test_c_refuses_selected_attention():
    lib = _lib.load()

    def call(o=O, q=Q, qs=256, h=4, sel=15 << 40, count=4, c=None, b=None, kv={}):
        cc, bb = _kv(**kv)
        return lib.hypno_hip_selected_attention_dev(
            o, q, qs, h, ctypes.byref(cc) if c is None else c, ctypes.byref(bb) if b is None else b,
            0.1, sel, count, None)

    null = ctypes.c_void_p()
    for kw in (dict(o=None), dict(q=None), dict(sel=None), dict(qs=255), dict(h=0), dict(h=3),
               dict(c=null), dict(b=null), dict(count=0), dict(count=1025), dict(o=Q), dict(o=15 << 40),
               dict(o=(15 << 40) - 4), dict(o=2 << 40), dict(o=5 << 40), dict(kv=dict(page_size=8)),
               dict(kv=dict(head_dim=60)), dict(kv=dict(dtype=3)), dict(kv=dict(dtype=2))):
        assert call(**kw) == 22, kw
        assert b"selected_attention" in lib.hypno_hip_last_error()
    for kv in (dict(tokens=0), dict(batch=0)):
        assert call(kv=kv) == 0


def test_python_refuses_host_tensors():
    import torch
    x, i = torch.zeros(2, 4, 64), torch.zeros(3, dtype=torch.int32)
    c, o, s = torch.zeros(4, 4, 16, 64).half(), torch.zeros(4, 4, 2, 64).char(), torch.zeros(4, 4)
    with pytest.raises(ValueError, match="GPU"):
        hk.key_bounds(c, o, s, i[None], i[:1], i[:2])
    with pytest.raises(ValueError, match="GPU"):
        hk.select_pages(x, o, s, 16, i[None], i[:1], i[:2], 4)
    with pytest.raises(ValueError, match="GPU"):
        hk.selected_attention(x, c, c, i[None, None], i[None], i[:1], i[:2])
