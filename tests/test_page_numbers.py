"""Which pages key_bounds works on: the numbers of csrc/kv_cache.hpp that its work-groups
count through, on the CPU for any cu_q, and the operators that count so on the GPU."""
import ctypes
import os
import subprocess

import numpy as np
import pytest

import hypno_amd as hk
from hypno_amd import build

HARNESS = r"""
#include "kv_cache.hpp"
using namespace hypno;
// (sequence, page) of every number, as key_bounds_kernel finds them; how many there are.
extern "C" int numbers(const int* cu_q, const int* lens, int batch, int tokens, int shift, int width,
                       int* out) {
  auto cu = [&](int i) { return std::min(std::max(cu_q[i], 0), tokens); };
  const int n = (int)first_number(cu(batch), batch, shift);
  for (int number = 0; number < n; number++) {
    int b = -1;
    for (int i = 0; i <= batch; i++) b += first_number(cu(i), i, shift) <= number;
    const bool in = b >= 0 && b < batch;
    out[2 * number] = b;
    out[2 * number + 1] =
        in ? page_of_number(number, b, cu(b), cu(b + 1), lens[b], shift, width) : -1;
  }
  return n;
}
"""


@pytest.fixture(scope="module")
def numbers(tmp_path_factory):
    path = tmp_path_factory.mktemp("numbers")
    src, so = str(path / "numbers.cpp"), str(path / "numbers.so")
    with open(src, "w") as f:
        f.write(HARNESS)
    subprocess.run([build.hipcc(), "-x", "hip", "--offload-host-only", "-O1", "-std=c++17", "-fPIC",
                    "-shared", f"-I{build.CSRC}", src, "-o", so], check=True, capture_output=True,
                   timeout=100)
    fn = ctypes.CDLL(so).numbers

    def run(cu, lens, page, width, tokens=2 ** 31 - 1):
        cu, lens = np.array(cu, np.int32), np.array(lens, np.int32)
        out = np.full((1 << 16, 2), -7, np.int32)
        n = fn(cu.ctypes.data_as(ctypes.c_void_p), lens.ctypes.data_as(ctypes.c_void_p), len(lens),
               tokens, page.bit_length() - 1, width, out.ctypes.data_as(ctypes.c_void_p))
        assert n <= len(out)
        return [tuple(x) for x in out[:n].tolist() if x[1] != -1]

    return run


def pages_of_new_tokens(b, n, kv, page, width):
    return [(b, at) for at in range(max(kv - n, 0) // page, (kv - 1) // page + 1)
            if at < width] if n > 0 and kv > 0 else []


def test_every_page_once(numbers):
    rng = np.random.default_rng(0)
    for _ in range(300):
        page, batch = 1 << int(rng.integers(0, 8)), int(rng.integers(1, 9))
        n = rng.integers(0, rng.choice([2, 5, 60, 900]), batch)
        lens = np.where(rng.random(batch) < 0.2, rng.integers(0, 40, batch),
                        n + rng.integers(0, 500, batch))
        cu, width = np.cumsum([0, *n]), int(rng.integers(1, 1 + max(1, lens.max() // page + 2)))
        want = [x for b in range(batch) for x in pages_of_new_tokens(b, n[b], lens[b], page, width)]
        assert numbers(cu, lens, page, width) == want


def test_no_place_out_of_the_table(numbers):
    """cu_q that does not ascend: pages with new tokens of their sequence, or none."""
    rng = np.random.default_rng(1)
    cases = [([90, 95, 0, 95], [5, 5, 5], 16, 8), ([0, 100, 200, 0, 0], [50, 100, 50, 50], 16, 8)]
    for _ in range(300):
        batch = int(rng.integers(1, 9))
        cases.append((rng.integers(-50, 3000, batch + 1), rng.integers(-3, 3000, batch),
                      1 << int(rng.integers(0, 8)), int(rng.integers(1, 3000))))
    for cu, lens, page, width in cases:
        for tokens in (2 ** 31 - 1, 1000):
            c = np.clip(cu, 0, tokens)
            for b, at in numbers(cu, lens, page, width, tokens):
                assert (b, at) in pages_of_new_tokens(b, c[b + 1] - c[b], lens[b], page, width), \
                    (cu, lens, page, width, b, at)


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8", "fp4"])
@pytest.mark.parametrize("cu", [[90, 95, 0, 95], [0, 100, 20, 0], [400, 0, 399, 380],
                                [0, 300, 5, 9000], [7, -90, 500, 64]], ids=str)
def test_cu_q_that_does_not_ascend(cu, kind):
    """Places many pages apart: bounds of pages in no row of the table stay as they are, and
    selections stay in their rows."""
    import torch
    from test_selected_attention import batch, old_bounds
    bt = batch(kind, [(3, 90), (2, 200), (1, 5)], 16, 80, kv_heads=2, dim=64, extra=40)
    a = bt.gpu()
    a["cu_q"] = torch.tensor(cu, dtype=torch.int32, device="cuda")
    codes, scale = (torch.from_numpy(x).cuda() for x in old_bounds(bt))
    old = codes.clone(), scale.clone()
    where = {n: a[n] for n in ("page_table", "kv_lens", "cu_q")}
    q = torch.randn(400, 4, 64, device="cuda")
    rows = torch.full((402, 2, 5), -77, dtype=torch.int32, device="cuda")
    hk.key_bounds(a["k_cache"], codes, scale, k_scale=a["k_scale"], **where)
    hk.select_pages(q, *old, 16, count=5, out=rows[1:-1], **where)
    torch.cuda.synchronize()
    free = torch.ones(bt.pages, dtype=torch.bool, device="cuda")
    free[a["page_table"][a["page_table"] >= 0].long()] = False
    assert free.sum() >= 40
    assert torch.equal(codes[free], old[0][free]) and torch.equal(scale[free], old[1][free])
    assert (rows[[0, -1]] == -77).all()
