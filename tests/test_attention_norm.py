"""paged_attention's error in the L2 norm over all rows of a call, against what an fp32
computation loses on average: twenty times closer than the elements' worst case of
test_paged_attention.attend."""
import math

import numpy as np
import pytest

from test_paged_attention import EPS, Batch, queries, run_attend


def rows_of(q, bt, scale):
    """The formula in 64 bits, and each row's root mean square error in fp32.

    A score's 2 D products (q is two parts) are added up in as many roundings of partial
    sums of the size sqrt(sum (q k)^2); q's parts leave 2^-22 of its largest element.  The
    exponent takes one rounding of its argument, a weight 2^-22 and some; numerator and
    denominator are sums over the n positions.  All of it goes to the output in proportion
    to sqrt(sum (w v)^2)."""
    T, H, D = q.shape
    out, err = np.zeros((T, H, D)), np.zeros((T, H))
    for b, (n, kv) in enumerate(bt.seqs):
        for h in range(H):
            k, v = bt.values(b, h // (H // bt.kv_heads), np.arange(kv))
            for i in range(n):
                t, p = bt.cu[b] + i, kv - n + i + 1
                x = q[t, h].astype(np.float64)
                s = (k[:p] @ x) * scale
                w = np.exp(s - s.max())
                w /= w.sum()
                out[t, h] = w @ v[:p]
                score = scale * (math.sqrt(2 * D) * np.sqrt((k[:p] ** 2) @ (x ** 2)) +
                                 4 * np.abs(x).max() * np.sqrt((k[:p] ** 2).sum(1)))
                each = EPS * (score + np.abs(s - s.max()) + 8 + 2 * math.sqrt(p))
                err[t, h] = np.sqrt((((w * each)[:, None] * v[:p]) ** 2).sum())
    return out, err


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("dim", [40, 64, 128, 256])
@pytest.mark.parametrize("seqs", [[(1, 40)] * 9, [(1, 900)] * 4, [(1, 5000), (1, 3000)], [(100, 100)],
                                  [(30, 3000)]], ids=str)
def test_error_in_the_norm(seqs, dim, kind):
    bt = Batch(seqs, 16, 80, dim=dim, kind=kind)
    if kind == "int8":
        bt.ks *= 0.7  # (scores of the size that fp16's have)
    q = queries(bt.tokens, 4, dim, 80)
    ref, err = rows_of(q, bt, 1 / math.sqrt(dim))
    got = np.linalg.norm(run_attend(bt, q) - ref)
    lim = np.linalg.norm(err)
    print(f"[norm] {got / np.linalg.norm(ref):.2e} of {lim / np.linalg.norm(ref):.2e}")
    assert got <= lim
