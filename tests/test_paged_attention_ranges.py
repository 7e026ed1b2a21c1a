"""paged_attention where its two kernels, their ranges of positions and the rows that
are computed again meet: against the formula in 64 bits, with the bounds of
test_paged_attention.attend."""
import ctypes
import os
import subprocess
import sys

import numpy as np
import pytest

import hypno_amd as hk
from hypno_amd import _lib
from test_paged_attention import Batch, attend, check, queries, run_attend

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("page", [8, 16, 64])
@pytest.mark.parametrize("seqs", [
    [(1, 1024)], [(1, 1025)], [(1, 1030), (1, 2049), (1, 3)],           # whole, then ranges
    [(3, 1500)], [(1, 140)], [(2, 1100), (5, 1300)],
    [(40, 2500)], [(70, 2100), (1, 1900), (1, 1)],                       # tiles in ranges
    [(1, 90), (30, 90), (1, 700), (17, 17)] * 3,                         # both kernels
], ids=str)
def test_ranges(seqs, page, kind):
    bt = Batch(seqs, page, 40, kind=kind)
    q = queries(bt.tokens, 4, 64, 40)
    check(run_attend(bt, q), *attend(q, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(20, 1, 64), (34, 2, 40), (3, 1, 256), (6, 2, 256),
                                                (5, 5, 128), (6, 3, 72)])
def test_groups(heads, kv_heads, dim, kind):
    """Groups above 16, odd ones, head_dim 256: single tokens, drafts and chunks."""
    bt = Batch([(1, 1300), (7, 200), (50, 90), (1, 5)], 16, 41, kv_heads=kv_heads, dim=dim,
               kind=kind)
    q = queries(bt.tokens, heads, dim, 41)
    check(run_attend(bt, q), *attend(q, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("page", [4, 16, 32, 128])
@pytest.mark.parametrize("window", [5, 17, 1000, 1400])
def test_windows_and_freed_pages(window, page, kind):
    """Windows that begin anywhere in a page, pages before them not in the table."""
    bt = Batch([(1, 1999), (60, 1777), (1, 30), (3, 1601)], page, 42, kind=kind)
    q = queries(bt.tokens, 4, 64, 42)
    ref, tol = attend(q, bt, window=window)
    for b, (n, kv) in enumerate(bt.seqs):
        bt.table[b, :max(0, kv - n - window + 1) // page] = -1
    check(run_attend(bt, q, window=window), ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("what", [float("nan"), float("inf")])
@pytest.mark.parametrize("seqs", [[(1, 2500)], [(40, 2500)], [(2, 1800), (33, 40), (1, 10)]])
def test_again_in_ranges(seqs, what, kind):
    """One spoilt value in one range, seen by the last token only: that token's rows of the
    kv head are not finite, all others as they were."""
    bt = Batch(seqs, 16, 43, kind=kind)
    q = queries(bt.tokens, 4, 64, 43)
    ref, tol = attend(q, bt)
    n, kv = seqs[0]
    pg, sl = bt.place(0, kv - 1)
    (bt.v if kind == "fp16" else bt.vs)[pg, 1, sl] = what
    got = run_attend(bt, q)
    hit = np.zeros(q.shape[:2], bool)
    hit[n - 1, 2:] = True
    assert not np.isfinite(got[hit]).any()
    check(got[~hit], ref[~hit], tol[~hit])


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 60])
def test_scales_of_all_sizes(n):
    """8-bit values' scales over all of fp32 within one tile, a code of 0 beside the
    largest weight: what is left is the smallest ones' sum."""
    bt = Batch([(n, 900)], 32, 44, kv_heads=1, kind="int8")
    rng = np.random.default_rng(44)
    bt.vs[:] = 10.0 ** rng.uniform(-34, 34, bt.vs.shape)
    bt.v[:, :, :, 7] = 0
    pg, sl = bt.place(0, np.arange(0, 900, 3))
    bt.v[pg, 0, sl, 7] = 1
    bt.vs[pg, 0, sl] = 1e-30
    q = queries(bt.tokens, 2, 64, 44)
    check(run_attend(bt, q), *attend(q, bt))


@pytest.mark.gpu
def test_no_pages():
    """A cache of no pages: what is seen is in no page of it, what sees nothing is zero."""
    import torch
    q = torch.randn(3, 4, 64, device="cuda")
    c = torch.zeros(0, 2, 16, 64, dtype=torch.float16, device="cuda")
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = hk.paged_attention(q, c, c, i(0, 0)[:, None].contiguous(), i(1, 0), i(0, 1, 3))
    assert got[0].isnan().all() and not got[1:].any()


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 90])
def test_any_alignment(n):
    """q and out at any float (through the C entry)."""
    import torch
    bt = Batch([(n, 300)], 16, 45)
    q = queries(n, 4, 64, 45)
    a = bt.gpu()
    src, dst = torch.zeros(n * 256 + 3, device="cuda"), torch.zeros(n * 256 + 3, device="cuda")
    src[3:] = torch.from_numpy(q.ravel()).cuda()
    c = _lib.KvCache(0, a["k_cache"].data_ptr(), a["v_cache"].data_ptr(), None, None,
                     bt.pages, 2, 16, 64, 0, 0, 0, 0)
    b = _lib.KvBatch(a["cu_q"].data_ptr(), a["kv_lens"].data_ptr(), a["page_table"].data_ptr(), 1,
                     bt.table.shape[1], n)
    torch.cuda.synchronize()
    for off in (1, 2, 3):
        src[off:off + n * 256] = torch.from_numpy(q.ravel()).cuda()
        torch.cuda.synchronize()
        assert _lib.load().hypno_hip_paged_attention_dev(
            dst.data_ptr() + 4 * off, src.data_ptr() + 4 * off, 256, 4, ctypes.byref(c),
            ctypes.byref(b), 0.125, 0, 300, None) == 0
        torch.cuda.synchronize()
        check(dst[off:off + n * 256].cpu().numpy().reshape(q.shape), *attend(q, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("seqs", [[(1, 3000)], [(60, 2800)]])
def test_capture_without_workspace(seqs):
    """Captured on a stream that has no workspace yet, ranges are not taken; replays are
    right and the same."""
    import torch
    bt = Batch(seqs, 16, 46)
    q = queries(bt.tokens, 4, 64, 46)
    ref, tol = attend(q, bt)
    a, x = bt.gpu(), torch.from_numpy(q).cuda()
    hk.paged_attention(x, **a)  # (loads the library)
    torch.cuda.synchronize()
    side, g = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = hk.paged_attention(x, **a)
    for _ in range(3):
        out.zero_()
        torch.cuda.synchronize()
        g.replay()
        torch.cuda.synchronize()
        check(out.cpu().numpy(), ref, tol)
        hk.paged_attention(x, **a)


@pytest.mark.gpu
def test_same_bits():
    """Sums go in one order: two calls, and calls on two streams at once, are equal."""
    import torch
    bt = Batch([(1, 4000), (1, 2200), (90, 1500)] * 3, 16, 47)
    a, x = bt.gpu(), torch.from_numpy(queries(bt.tokens, 4, 64, 47)).cuda()
    want = hk.paged_attention(x, **a)
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], []
    for _ in range(3):
        for s in streams:
            with torch.cuda.stream(s):
                got.append(hk.paged_attention(x, **a))
    torch.cuda.synchronize()
    assert all(torch.equal(want, g) for g in got)


@pytest.mark.gpu
def test_arguments_both_ways():
    """Calls that the native reader of tensors leaves to the Python functions (numbers of
    other types, empty batches) give the same."""
    import torch
    bt = Batch([(2, 300)], 16, 48)
    a, x = bt.gpu(), torch.from_numpy(queries(2, 4, 64, 48)).cuda()
    want = hk.paged_attention(x, scale=1.0, window=7, max_kv_len=300, **a)
    got = hk.paged_attention(x, scale=1, window=np.int64(7), max_kv_len=np.int32(300), **a)
    assert torch.equal(want, got)
    none = Batch([(0, 20)], 16, 48).gpu()
    assert hk.paged_attention(x[:0], **none).shape == (0, 4, 64)
    k = torch.zeros(0, 2, 64, device="cuda")
    assert hk.append_kv(x[:0], k, k, **none).shape == (0, 4, 64)


@pytest.mark.gpu
def test_example():
    """examples/paged_decode.py: a layer's prompt and tokens through both operators."""
    p = subprocess.run([sys.executable, os.path.join(ROOT, "examples", "paged_decode.py"),
                        "--prompt", "70", "--tokens", "5"], capture_output=True, text=True,
                       timeout=100)
    assert p.returncode == 0, p.stderr
    assert "agree" in p.stdout
