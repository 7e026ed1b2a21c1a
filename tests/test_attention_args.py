"""The native reader of torch's tensors (csrc/attention_args.cpp): the package builds and
works without it, and where it answers it takes and refuses what the Python functions do."""
import sys

import numpy as np
import pytest

import hypno_amd as hk
from hypno_amd import attention
from hypno_amd import build as hb
from test_paged_attention import Batch, queries


@pytest.fixture
def without(monkeypatch):
    """No _attention_args.so."""
    monkeypatch.setattr(attention, "_args", None)
    monkeypatch.delattr(hk, "_attention_args", raising=False)
    monkeypatch.setitem(sys.modules, "hypno_amd._attention_args", None)


def test_builds_without_a_compiler_for_it(tmp_path, monkeypatch, capfd):
    monkeypatch.setattr(hb, "HERE", str(tmp_path))
    (tmp_path / "_attention_args.so").write_bytes(b"of older sources")
    monkeypatch.setenv("PATH", str(tmp_path))
    hb._build_args()
    assert not (tmp_path / "_attention_args.so").exists()
    assert "optional" in capfd.readouterr().err
    bad = tmp_path / "g++"  # (one that finds no headers)
    bad.write_text("#!/bin/sh\necho no such file >&2\nexit 1\n")
    bad.chmod(0o755)
    hb._build_args()
    assert "no such file" in capfd.readouterr().err


def test_refusals_without_it(without):
    import torch
    x, i = torch.zeros(2, 4, 64), torch.zeros(2, dtype=torch.int32)
    c = torch.zeros(4, 4, 16, 64, dtype=torch.float16)
    with pytest.raises(ValueError, match="GPU"):
        hk.append_kv(x, x, x, c, c, i[None], i[:1], i)
    with pytest.raises(ValueError, match="GPU"):
        hk.paged_attention(x, c, c, i[None], i[:1], i)


def variants():
    """Names and changes of the arguments (a: all of them by name, fresh for each)."""
    import torch
    up = lambda *x, **k: torch.zeros(*x, device="cuda", **k)  # noqa: E731

    def strided(t):
        pool = torch.zeros((t.shape[0], 2, *t.shape[1:]), dtype=t.dtype, device="cuda")
        pool[:, 1] = t
        return pool[:, 1]

    tensors = dict(
        half=lambda t: t.half(), double=lambda t: t.double(), int32=lambda t: t.int(),
        cpu=lambda t: t.cpu(), flat=lambda t: t.flatten(), first=lambda t: t[:1],
        none=lambda t: None, last=lambda t: t[..., :-1], step=lambda t: t[..., ::2],
        turned=lambda t: t.transpose(0, -1), more=lambda t: t[None], empty=lambda t: t[:0],
        strided=strided, twice=lambda t: torch.cat([t, t]), number=lambda t: 3,
        array=lambda t: t.cpu().numpy(), same=lambda t: t[:1].expand_as(t),
        gap=lambda t: torch.cat([t, t], -1)[..., :t.shape[-1]])
    for name in ("q", "k", "v", "k_cache", "v_cache", "k_scale", "v_scale", "page_table", "kv_lens",
                 "cu_q", "inv_freq", "out"):
        for how, f in tensors.items():
            yield f"{name} {how}", lambda a, name=name, f=f: (
                None if a.get(name) is None else a.update({name: f(a[name])}))
    yield "scales of fp16", lambda a: a.update(k_scale=up(4, 2, 16), v_scale=up(4, 2, 16))
    for window in (0, 7, -1, np.int64(7), 2 ** 40, True):
        yield f"window {window!r}", lambda a, w=window: a.update(window=w)
    for most in (None, 0, 300, -1, np.int32(300), 2 ** 40):
        yield f"max_kv_len {most!r}", lambda a, m=most: a.update(max_kv_len=m)
    for scale in (None, 0.5, 1, 0, -0.25, np.float32(0.5), float("nan")):
        yield f"scale {scale!r}", lambda a, s=scale: a.update(scale=s)
    yield "one head", lambda a: a.update(q=a["q"][:, :1], out=a["out"][:, :1])
    yield "three heads", lambda a: a.update(q=a["q"][:, :3], out=a["out"][:, :3])
    yield "rotation of a part", lambda a: a.update(inv_freq=a["inv_freq"][:9])
    yield "rotation of none", lambda a: a.update(inv_freq=a["inv_freq"][:0])
    yield "in place", lambda a: a.update(out=a["q"])
    yield "new output", lambda a: a.update(out=None)


ATTEND = ("q", "k_cache", "v_cache", "page_table", "kv_lens", "cu_q", "scale", "window", "k_scale",
          "v_scale", "max_kv_len", "out")
APPEND = ("q", "k", "v", "k_cache", "v_cache", "page_table", "kv_lens", "cu_q", "inv_freq",
          "k_scale", "v_scale", "out")


@pytest.mark.gpu
@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("fn,names", [("paged_attention", ATTEND), ("append_kv", APPEND)],
                         ids=["paged_attention", "append_kv"])
def test_same_answers(fn, names, kind, monkeypatch):
    """Every argument in many wrong and unusual forms: both ways raise the same or give
    the same."""
    import torch
    bt = Batch([(2, 30), (1, 25)], 16, 70, kind=kind)
    q = torch.from_numpy(queries(3, 4, 64, 70)).cuda()

    def call(change):
        a = {"scale": None, "window": 0, "max_kv_len": None, **bt.gpu()}
        a.update(q=q.clone(), k=q[:, :2].clone(), v=q[:, 1:3].clone(), out=torch.zeros_like(q),
                 inv_freq=torch.linspace(1, 0.01, 32, device="cuda"))
        change(a)
        try:
            got = getattr(hk, fn)(**{k: a[k] for k in names})
            torch.cuda.synchronize()
        except (ValueError, hk.HypnoHipError) as e:
            return type(e), str(e)
        return [None if t is None else t.clone() for t in
                (got, a["k_cache"], a["v_cache"], a["k_scale"], a["v_scale"])]

    call(lambda a: None)
    native = attention._args
    assert native is not attention._NoArgs
    bad = []
    for name, change in variants():
        monkeypatch.setattr(attention, "_args", native)
        got = call(change)
        monkeypatch.setattr(attention, "_args", attention._NoArgs)
        want = call(change)
        if isinstance(want, tuple) or isinstance(got, tuple):
            same = got == want
        else:
            same = all(x is y is None or torch.equal(x.view(torch.uint8), y.view(torch.uint8))
                       for x, y in zip(got, want))
        if not same:
            bad.append((name, got, want))
    assert not bad, bad


@pytest.mark.gpu
def test_results_without_it(without):
    import torch
    bt = Batch([(2, 300)], 16, 48)
    a, x = bt.gpu(), torch.from_numpy(queries(2, 4, 64, 48)).cuda()
    got = hk.paged_attention(x, **a)
    assert attention._args is attention._NoArgs
    attention._args = None
    sys.modules.pop("hypno_amd._attention_args")
    assert torch.equal(got, hk.paged_attention(x, **a))
