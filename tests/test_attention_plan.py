"""How paged_attention splits positions into ranges (attn_plan, on the CPU), and calls
chosen from that plan against the formula in 64 bits, with the bounds of
test_paged_attention.attend."""
import ctypes

import numpy as np
import pytest

from hypno_amd import _lib
from test_paged_attention import Batch, attend, check, queries, run_attend

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
                ("cus", ctypes.c_int), ("fs", Split), ("ts", Split), ("rest", ctypes.c_byte * 256)]


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
