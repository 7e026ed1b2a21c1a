"""examples/paged_decode.py with selected pages: what it compares its tokens with, on the CPU,
and that it compares them."""
import importlib.util
import os
import subprocess
import sys

import numpy as np
import pytest

from conftest import ROOT
from test_paged_attention import queries
from test_selected_attention import KINDS, attend_selected, batch

PATH = os.path.join(ROOT, "examples", "paged_decode.py")


@pytest.fixture(scope="module")
def example():
    spec = importlib.util.spec_from_file_location("paged_decode", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    return module


def state(kind, kv=75, chosen=(0, 2, 3, 4)):
    """One token's queries, cache and pages; attention over them by the tests' own formula."""
    import torch
    bt = batch(kind, [(1, kv)], 16, 90, kv_heads=2, dim=64)
    q = queries(1, 4, 64, 90, std=1.0)
    sel = np.tile(np.array(chosen, np.int32), (1, 2, 1))
    want = attend_selected(q, bt, sel)[0]
    names = {"k_cache": bt.k, "v_cache": bt.v, "k_scale": bt.ks, "v_scale": bt.vs}
    cache = {n: torch.from_numpy(x) for n, x in names.items() if x is not None}
    return torch.from_numpy(q[0]), cache, torch.from_numpy(bt.table[0]), sel[0].tolist(), kv, want[0]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("kv,chosen", [(75, (0, 2, 3, 4)), (80, (0, 3, 4, -1)), (3, (0, -1))])
def test_plain_computation(example, kind, kv, chosen):
    *args, want = state(kind, kv, chosen)
    got, size = example.over_pages(*args).numpy()
    assert np.abs(got - want).max() <= 1e-12 * max(1.0, np.abs(want).max())
    assert (size >= np.abs(got)).all()


def test_check_finds_mistakes(example):
    import torch
    *args, want = state("fp16")
    q, cache, table, chosen, kv = args
    a = torch.from_numpy(want).float()
    example.check(a, *args)
    for wrong in (a * 0, a * float("nan"), a.roll(1, 0), a * 1.01):
        with pytest.raises(SystemExit, match="differs"):
            example.check(wrong, *args)
    for pages in ([0, 1, 2, 3], [0, 3, 2, 4], [0, 3, 4, -1], [1, 2, 3, 4], [0, 3, 4, 4], [0, 1, 2, 4]):
        with pytest.raises(SystemExit, match="pages"):
            example.check(a, q, cache, table, [pages, chosen[1]], kv)


@pytest.mark.gpu
@pytest.mark.parametrize("args", [["--fp4", "--pages", "4"], ["--int8", "--pages", "3"],
                                  ["--pages", "4"], ["--int8", "--pages", "9"]], ids=" ".join)
def test_selected_pages_are_compared(args):
    p = subprocess.run([sys.executable, PATH, "--prompt", "70", "--tokens", "5", *args],
                       capture_output=True, text=True, timeout=100)
    assert p.returncode == 0 and p.stdout.rstrip().endswith("agree"), p.stdout + p.stderr
