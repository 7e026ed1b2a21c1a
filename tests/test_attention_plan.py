"""How paged_attention splits positions into ranges (attn_plan, on the CPU), and calls
chosen from that plan against the formula in 64 bits, with the bounds of
test_paged_attention.attend."""
import ctypes

import numpy as np
import pytest

from hypno_amd import _lib
from test_paged_attention import O, Q, Batch, _kv, attend, check, queries, run_attend

RUN = 16  # positions that attn_few_kernel takes to lie in one page (pages of as many or more)


class Cache(ctypes.Structure):
    """KvCache of csrc/kv_cache.hpp."""
    _fields_ = [("dtype", ctypes.c_int), ("pointers", ctypes.c_void_p * 4),
                ("strides", ctypes.c_size_t * 4), ("pages", ctypes.c_int),
                ("kv_heads", ctypes.c_int), ("page_shift", ctypes.c_int),
                ("head_dim", ctypes.c_int)]


class Sequences(ctypes.Structure):
    """KvBatch of csrc/kv_cache.hpp."""
    _fields_ = [("pointers", ctypes.c_void_p * 3), ("batch", ctypes.c_int),
                ("width", ctypes.c_int), ("tokens", ctypes.c_int)]


class Split(ctypes.Structure):
    _fields_ = [("splits", ctypes.c_int), ("chunk", ctypes.c_int)]


class Plan(ctypes.Structure):
    """The first members of AttnPlan, and room for the rest."""
    _fields_ = [("few", ctypes.c_int), ("few_waves", ctypes.c_int), ("tile_rows", ctypes.c_int),
                ("cus", ctypes.c_int), ("fs", Split), ("ts", Split), ("bytes", ctypes.c_size_t),
                ("rest", ctypes.c_byte * 256)]


def plan(batch, tokens, heads, kv_heads, dim, kv, kind="fp16", page=16, window=0, max_kv=0,
         cus=256):
    import torch  # noqa: F401  (before the library: both take one HIP runtime then)
    fn = getattr(_lib.load(), "_ZN5hypno9attn_planERKNS_7KvCacheERKNS_7KvBatchEiili")
    fn.restype = Plan
    fn.argtypes = [ctypes.POINTER(Cache), ctypes.POINTER(Sequences), ctypes.c_int, ctypes.c_int,
                   ctypes.c_int64, ctypes.c_int]
    c = Cache(dtype=int(kind == "int8"), pages=1, kv_heads=kv_heads,
              page_shift=page.bit_length() - 1, head_dim=dim)
    b = Sequences(batch=batch, width=-(-kv // page), tokens=tokens)
    return fn(c, b, heads, window, max_kv, cus)


# --- ranges -----------------------------------------------------------------------------

def test_ranges_are_whole_runs():
    """A range that another one follows ends where a run of positions does: its kernel
    takes a run's keys from the page of the first."""
    seen = set()
    for batch in [*range(1, 71), 100, 255, 256]:
        for kv_heads in (1, 2, 3, 4, 5, 6, 7, 8, 11, 33):
            for kv in (1025, 1500, 2049, 3000, 5003, 9001, 40000, 131072, 1000003):
                for tokens in (batch, 3 * batch):
                    for window in (0, 2500):
                        p = plan(batch, tokens, 4 * kv_heads, kv_heads, 64, kv, window=window)
                        for s in (p.fs, p.ts):
                            if s.splits > 1:
                                assert s.chunk % RUN == 0, (batch, kv_heads, kv, tokens, s.chunk)
                                seen.add(s.chunk)
    assert len(seen) > 10


def places(p, dim):
    return p.bytes // (4 * dim + 8)


def test_workspace_goes_by_the_rows_that_take_ranges():
    """Ranges of a long context beside a prompt take room for the few rows that have them,
    and no call more than 512 MB a kernel."""
    # One sequence of 8192 new tokens and eight of one, 131072 positions at most.
    p = plan(9, 8200, 32, 8, 128, 131072)
    assert p.few == 16 and p.fs.splits > 50 and 1 < p.ts.splits < 5
    assert places(p, 128) == p.fs.splits * 9 * 8 * 16 + p.ts.splits * 8200 * 32
    p = plan(16, 2063, 32, 8, 128, 131072)
    assert p.fs.splits > 30 and p.bytes < 512 << 20
    for batch in (1, 2, 8, 9, 17, 64, 256, 1000):
        for new in (1, 2, 7, 40, 300, 2400, 10000):
            for heads, kv_heads, dim in ((32, 8, 128), (12, 12, 64), (64, 1, 256), (7, 7, 40)):
                for kv in (1500, 9000, 131072, 1 << 24):
                    tokens = batch - 1 + new
                    if tokens * heads > 2 ** 31 or batch * kv > 2 ** 31:
                        continue
                    p = plan(batch, tokens, heads, kv_heads, dim, kv)
                    assert p.bytes <= (512 << 20) * (2 if p.few == 16 else 1) + 256
                    if batch == 1 and new * heads // kv_heads <= 16 and kv > 1500:
                        assert p.fs.splits > 1


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("heads,kv_heads,dim", [(4, 2, 64), (8, 8, 40), (16, 1, 128)])
@pytest.mark.parametrize("tokens", [20, 300])
def test_ranges_of_both_kernels(tokens, heads, kv_heads, dim, kind):
    """Chunks and single tokens in one call, both in ranges; rows counted by token and by
    sequence."""
    seqs = [(1, 3100), (tokens, 2600), (1, 2), (2, 1500), (0, 900), (1, 2100), (30, 3000), (1, 1111),
            (16 * kv_heads // heads, 1900), (1, 3090)]
    bt = Batch(seqs, 16, 66, kv_heads=kv_heads, dim=dim, kind=kind)
    p = plan(len(seqs), bt.tokens, heads, kv_heads, dim, 3100, kind)
    assert p.few == 16 and p.fs.splits > 1 and p.ts.splits > 1
    q = queries(bt.tokens, heads, dim, 66)
    rows = np.r_[0:bt.cu[1] + 2, bt.cu[2] - 2:bt.cu[6] + 2, bt.cu[7] - 2:bt.tokens]
    ref, tol = attend(q, bt)
    check(run_attend(bt, q)[rows], ref[rows], tol[rows])


# Batches times kv heads whose ranges' least length (8 positions for each) is no multiple
# of a run.
@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("page", [4, 16, 64, 8192])
@pytest.mark.parametrize("batch,heads,kv_heads,kv", [(7, 10, 5, 5003), (33, 2, 1, 3000),
                                                     (3, 14, 7, 4100), (1, 42, 21, 3000)])
def test_odd_batches_times_heads(batch, heads, kv_heads, kv, page, kind):
    seqs = [(1, kv)] + [(1, kv // 8 + 251 * b) for b in range(1, min(batch, 5))]
    seqs += [(1, 40 + b) for b in range(len(seqs), batch)]
    bt = Batch(seqs, page, 60, kv_heads=kv_heads, dim=64, kind=kind)
    assert plan(batch, batch, heads, kv_heads, 64, kv, kind, page).fs.splits > 1
    q = queries(bt.tokens, heads, 64, 60)
    check(run_attend(bt, q), *attend(q, bt))


# --- the parts' sum ------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 64, 128, 256])
@pytest.mark.parametrize("ranges", [9, 10, 32, 33, 34, 35, 48, 49, 50, 64, 65, 66, 129, 131, 134,
                                    138, 196, 200, 258, 262])
def test_join_by_four_waves(ranges, dim):
    """Ranges in all numbers that leave some of a wave's lanes without one, split over
    four waves."""
    kv = 128 * ranges - 50
    bt = Batch([(1, kv)], 16, 61, kv_heads=1, dim=dim)
    p = plan(1, 1, 2, 1, dim, kv)
    assert (p.fs.splits, p.fs.chunk) == (ranges, 128)
    q = queries(1, 2, dim, 61)
    check(run_attend(bt, q), *attend(q, bt))


@pytest.mark.gpu
@pytest.mark.parametrize("dim", [40, 64, 128, 256])
@pytest.mark.parametrize("ranges", [9, 17, 31, 32, 33, 34, 35, 48, 49, 50, 63, 64, 65, 98])
def test_join_by_one_wave(ranges, dim):
    """The same with a wave a row: 1024 rows and more."""
    kv = 128 * ranges - 50
    bt = Batch([(1, kv)], 16, 62, kv_heads=1, dim=dim)
    p = plan(1, 1, 1024, 1, dim, kv)
    assert (p.fs.splits, p.fs.chunk) == (ranges, 128)
    q = queries(1, 1024, dim, 62)
    ref, tol = attend(q[:, ::73], bt)  # (all read one kv head)
    check(run_attend(bt, q)[:, ::73], ref, tol)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("ranges", [33, 34, 49])
@pytest.mark.parametrize("tokens,heads,dim", [(20, 4, 64), (20, 4, 128), (70, 16, 64)])
def test_join_of_tiles(tokens, heads, dim, ranges, kind):
    """Tiles' ranges, of a sequence shorter than max_kv_len says."""
    p = plan(1, tokens, heads, 1, dim, 60000, kind)
    assert p.few == 0 and p.ts.splits >= ranges
    kv = p.ts.chunk * ranges - 40
    bt = Batch([(tokens, kv)], 16, 63, kv_heads=1, dim=dim, kind=kind)
    bt.table = np.concatenate([bt.table, np.full((1, 60000 // 16 - bt.table.shape[1]), -1,
                                                 np.int32)], 1)
    q = queries(tokens, heads, dim, 63)
    got = run_attend(bt, q, max_kv_len=60000)
    # (the last tokens' rows are in the tile that sees all ranges)
    last = Batch([(3, kv)], 16, 63, kv_heads=1, dim=dim, kind=kind)
    last.table, last.k, last.v, last.ks, last.vs = bt.table, bt.k, bt.v, bt.ks, bt.vs
    ref, tol = attend(q[-3:, ::5], last)
    check(got[-3:, ::5], ref, tol)


# --- the last positions ----------------------------------------------------------------------

@pytest.mark.parametrize("page,width", [(128, (1 << 24) - 1), (1, (1 << 31) - 1), (4096, 1 << 19),
                                        (1, (1 << 31) - 4095), (16, (1 << 27) - 255)])
def test_refuses_positions_that_the_kernels_cannot_count(page, width):
    """The kernels add some tiles to a position in 32 bits before they clamp it."""
    lib = _lib.load()
    for tokens in (0, 3):
        c, b = (ctypes.byref(x) for x in _kv(page_size=page, table_width=width, tokens=tokens))
        assert lib.hypno_hip_paged_attention_dev(O, Q, 256, 4, c, b, 0.1, 1, 0, None) == 22
        assert b"paged_attention" in lib.hypno_hip_last_error()
    # One page less is taken.
    c, b = (ctypes.byref(x) for x in _kv(page_size=page, tokens=0,
                                         table_width=((1 << 31) - 4096) // page))
    assert lib.hypno_hip_paged_attention_dev(O, Q, 256, 4, c, b, 0.1, 1, 0, None) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("window,page", [(1, 64), (70, 8), (70, 4096), (700, 64), (700, 4096)])
@pytest.mark.parametrize("n", [1, 40])
def test_last_positions(n, window, page, kind):
    """A sequence that ends where the longest table does (earlier pages are not there)."""
    kv = (1 << 31) - 4096
    bt = Batch([(n, 6 * 4096)], page, 64, kind=kind)
    held = bt.table[0]
    bt.table = np.full((1, kv // page), -1, np.int32)
    bt.table[0, -len(held):] = held
    bt.seqs, bt.lens = [(n, kv)], np.array([kv], np.int32)
    q = queries(n, 4, 64, 64)
    check(run_attend(bt, q, window=window), *attend(q, bt, window=window))


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 20])
def test_pages_of_more_than_2e31_places(n):
    """One page of 65536 tokens and 32769 kv heads: its last head's scales are 2^31 of them
    from its first (52 GB)."""
    import torch

    import hypno_amd as hk
    if torch.cuda.mem_get_info()[0] < 60 << 30:
        pytest.skip("needs 60 GB of device memory")
    kv_heads, page, kv = 32769, 65536, 150
    at = torch.tensor([0, 1, 77, 32766, 32767, 32768], device="cuda")
    bt = Batch([(n, kv)], 256, 65, extra=0, kv_heads=len(at), dim=8, kind="int8")
    q = queries(n, len(at), 8, 65)
    ref, tol = attend(q, bt)
    big = {}
    for name, x in (("k_cache", bt.k), ("v_cache", bt.v), ("k_scale", bt.ks), ("v_scale", bt.vs)):
        x = torch.from_numpy(x[0, :, :kv]).cuda()
        t = big[name] = torch.empty((1, kv_heads, page, *x.shape[2:]), dtype=x.dtype,
                                    device="cuda")
        t[:, :, :kv] = 1
        t[0, at, :kv] = x
    x = torch.ones(n, kv_heads, 8, device="cuda")
    x[:, at] = torch.from_numpy(q).cuda()
    i = lambda *x: torch.tensor(x, dtype=torch.int32, device="cuda")  # noqa: E731
    got = hk.paged_attention(x, page_table=i(0)[None], kv_lens=i(kv), cu_q=i(0, n), **big)
    got = got[:, at].cpu().numpy()
    del big, t, x
    torch.cuda.empty_cache()
    check(got, ref, tol)


# --- small weights ----------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("n", [1, 40])
@pytest.mark.parametrize("score", [9, 12, 15, 18, 20, 22, 24, 26, 30, 60])
def test_small_weights(score, n, kind):
    """A first key whose value is 0 beside 3000 of weight e^-score: fp32's bits beside 8-bit
    codes; beside fp16 values each weight is off by 2^-37 of the largest at most."""
    kv = 3000
    bt = Batch([(n, kv)], 64, 67, kv_heads=1, kind=kind)
    pg, sl = bt.place(0, np.arange(kv))
    q = np.zeros((n, 2, 64), np.float32)
    q[:, :, 0] = 8.0
    bt.k[pg, 0, sl, 0] = 0
    bt.v[pg, 0, sl] = np.abs(bt.v[pg, 0, sl].astype(np.float32)).astype(bt.v.dtype)
    bt.v[pg[0], 0, sl[0]] = 0
    if kind == "fp16":
        bt.k[pg[0], 0, sl[0], 0] = score
    else:
        bt.k[pg[0], 0, sl[0], 0] = 120
        bt.ks[:] = score / 120
    ref, tol = attend(q, bt)
    if kind == "fp16":
        v = np.abs(bt.v[pg, 0, sl].astype(np.float64))
        tol += 2.0 ** -37 * v.sum(0)
    check(run_attend(bt, q), ref, tol)
