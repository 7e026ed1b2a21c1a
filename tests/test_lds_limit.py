"""Kernels whose LDS grows with a call's sizes: a later, larger call launches as the first did
(on a HIP runtime that runs nothing), and selections in more than 64 KB on the GPU."""
import json
import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT
from test_paged_attention import Batch, queries
from test_selected_attention import old_bounds, run_select, select

HERE = os.path.dirname(os.path.abspath(__file__))

CALLS = r"""
import ctypes, json, sys
sys.path.insert(0, sys.argv[1])
limit = ctypes.CDLL(sys.argv[2], mode=ctypes.RTLD_GLOBAL)
fake = ctypes.CDLL(sys.argv[3], mode=ctypes.RTLD_GLOBAL)
limit.lds_most.restype = ctypes.c_size_t
from hypno_amd import _lib
lib = _lib.load()

def at(n):  # (addresses of nothing)
    return n << 40

def batch(batch, tokens, pages):
    return ctypes.byref(_lib.KvBatch(cu_q=at(3), kv_lens=at(4), page_table=at(5), batch=batch,
                                     table_width=pages, tokens=tokens))

out = []
for kind, captured, c in json.loads(sys.argv[4]):
    fake.fake_set_capturing(captured)
    kv, dim, heads, tokens, pages = c["kv_heads"], c["dim"], c["heads"], c["tokens"], c["pages"]
    b = batch(c["batch"], tokens, pages)
    if kind == "select":
        o = _lib.KeyBounds(codes=at(13), scale=at(14), pages=4, kv_heads=kv, page_size=16, head_dim=dim)
        st = lib.hypno_hip_select_pages_dev(at(12), 4, 1, 1, at(8), heads * dim, heads,
                                            ctypes.byref(o), b, 0, None)
    else:
        scale = (at(6), at(7)) if kind != "fp16" else (None, None)
        o = _lib.KvCache(dtype=["fp16", "int8", "fp4"].index(kind), k=at(1), v=at(2),
                         k_scale=scale[0], v_scale=scale[1], pages=4, kv_heads=kv, page_size=16,
                         head_dim=dim)
        st = lib.hypno_hip_selected_attention_dev(at(12), at(8), heads * dim, heads, ctypes.byref(o),
                                                  b, 0.1, at(15), c["count"], None)
    out.append([st, limit.lds_refused(), limit.lds_launches(), limit.lds_most()])
print(json.dumps(out))
"""


@pytest.fixture(scope="module")
def calls(tmp_path_factory):
    from hypno_amd import _lib
    assert os.path.exists(_lib.LIB_PATH)
    libs = []
    for name in ("lds_limit", "fake_hip"):
        libs.append(str(tmp_path_factory.mktemp("fake") / f"lib{name}.so"))
        subprocess.run(["g++", "-O1", "-std=c++17", "-shared", "-fPIC", "-o", libs[-1],
                        os.path.join(HERE, "fake_hip", f"{name}.cpp")], check=True)

    def run(*steps):
        p = subprocess.run([sys.executable, "-c", CALLS, ROOT, *libs, json.dumps(steps)],
                           capture_output=True, text=True, timeout=100)
        assert p.returncode == 0, p.stderr
        return json.loads(p.stdout)

    return run


def _case(kind, captured=0, **kw):
    c = dict(heads=4, kv_heads=4, dim=64, batch=1, tokens=1, pages=1000, count=4)
    c.update(kw)
    return kind, captured, c


@pytest.mark.parametrize("dim", [64, 128, 256])
@pytest.mark.parametrize("captured", [0, 1])
@pytest.mark.parametrize("batch,tokens", [(1, 1), (200, 200), (1, 20), (3, 300)])
def test_selection_of_more_pages_after_fewer(calls, batch, tokens, captured, dim):
    """Up to the 32768 pages of a sequence that a call may have, in 128 KB."""
    for most in (20000, 32768):
        got = calls(*(_case("select", captured, batch=batch, tokens=tokens, dim=dim, pages=n)
                      for n in (4, 300, 5000, most, 4)))
        assert [x[:2] for x in got] == [[0, 0]] * 5 and got[-1][2] >= 5
        if captured or tokens == batch:  # (in one kernel, or chosen from one token's scores)
            assert got[-1][3] >= 4 * most


@pytest.mark.parametrize("kind", ["fp16", "int8", "fp4"])
@pytest.mark.parametrize("dim", [64, 128, 256])
def test_longer_lists_after_shorter(calls, kind, dim):
    counts = (1, 10, 60, 64, 1024, 1)
    for tokens in (1, 300):
        got = calls(*(_case(kind, batch=tokens, tokens=tokens, dim=dim, count=n) for n in counts))
        assert [x[:2] for x in got] == [[0, 0]] * len(counts)


# --- on the GPU -------------------------------------------------------------------------------

@pytest.mark.gpu
@pytest.mark.parametrize("heads,seqs", [(4, [(1, 33), (1, 20000), *[(1, 40 + i) for i in range(37)],
                                             (1, 32768)]),
                                        (16, [(1, 2048 - 100 * i) for i in range(16)])],
                         ids=["long", "16 heads"])
def test_single_tokens(heads, seqs):
    """One kernel with as many tokens' scores as there is room for."""
    bt = Batch(seqs, 1, 81, kv_heads=heads, dim=16)
    q, b = queries(bt.tokens, heads, 16, 81), old_bounds(bt)
    for count in (3, 200):
        assert np.array_equal(run_select(bt, q, *b, count, 1, 2), select(bt, q, *b, count, 1, 2))


@pytest.mark.gpu
@pytest.mark.parametrize("heads,dim,seqs", [(1, 64, [(1, 32768)]), (2, 256, [(1, 30000)]),
                                            (3, 32, [(20, 2048)]), (1, 136, [(17, 2000), (3, 90)])],
                         ids=str)
def test_without_a_workspace(heads, dim, seqs):
    """Under capture on a stream that never had one: all scores in LDS."""
    import torch
    import hypno_amd as hk
    bt = Batch(seqs, 1, 82, kv_heads=heads, dim=dim)
    x, bounds = queries(bt.tokens, heads, dim, 82), old_bounds(bt)
    a, q = bt.gpu(), torch.from_numpy(x).cuda()
    codes, scale = (torch.from_numpy(y).cuda() for y in bounds)
    out = torch.zeros(bt.tokens, heads, 100, dtype=torch.int32, device="cuda")
    side, graph = torch.cuda.Stream(), torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        hk.select_pages(q, codes, scale, 1, a["page_table"], a["kv_lens"], a["cu_q"], 100, out=out)
    want = select(bt, x, *bounds, 100)
    for i in range(3):
        out.zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert np.array_equal(out.cpu().numpy(), want)
        assert np.array_equal(run_select(bt, x, *bounds, 100), want)
