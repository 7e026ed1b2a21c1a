"""The step between a layer's q/k/v projections and its output projection: rotated
keys and values appended to a paged cache, and attention of the new tokens over it.
In hypno this is a flat fp32 cache per layer with its rotation and its attention
loop (transformer.rs:92-184,281-462, turbo.rs:145-185).

    q = append_kv(q, k, v, k_cache, v_cache, page_table, kv_lens, cu_q, inv_freq)
    o = paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_q)

All arguments are GPU tensors of one device; calls are asynchronous on torch's
current stream.  A batch of sequences brings new tokens, the rows of q, k and v
([tokens, heads, head_dim] float32; views of one fused projection will do): those of
sequence b are rows cu_q[b] to cu_q[b + 1].  kv_lens[b] counts what it holds with
them, so its i-th new token of n has position kv_lens[b] - n + i.  Position p is in
slot p % page_size of page page_table[b, p // page_size].  cu_q, kv_lens and
page_table are int32 and are read on the GPU: a page id that is none of the cache's
(-1 for a freed one, say) is not written, and what reads it is NaN.  A table has room
for less than 2^31 positions a sequence, for attention 2^31 - 4096 at most.  Rows of q,
k and v of no sequence (past cu_q's last, for padding) are left alone: so are the outputs'
rows in `out`, which in a new tensor hold anything.

The caches are [pages, kv_heads, page_size, head_dim], float16, or int8 with
float32 k_scale and v_scale [pages, kv_heads, page_size]: one scale a token and kv
head.  Pages may be strided (a pool of [pages, layers, ...]); the rest is contiguous.

Arguments that cannot be right raise ValueError; a library failure raises
HypnoHipError.
"""
from __future__ import annotations

import ctypes
import math
import struct

from ._lib import check, load

__all__ = ["append_kv", "paged_attention"]

_STYLES = {"halves": 0, "pairs": 1}  # HYPNO_HIP_ROPE_*

# The structs of include/hypno_hip.h (_lib.KvCache and _lib.KvBatch), packed at once.
_CACHE = struct.Struct("=I4x12Q")
_BATCH = struct.Struct("=6Q")

torch = None
_args = None  # csrc/attention_args.cpp: the same checks and packing, where all is right


class _NoArgs:
    """Stands for it where it was not built."""

    @staticmethod
    def append_kv(*_):
        return NotImplemented

    paged_attention = append_kv


def _torch():
    """(imported by the first call: the rest of the package works without it)"""
    global torch, _args
    import torch
    lib = load()
    try:
        from . import _attention_args
    except ImportError:
        _args = _NoArgs
        return
    _attention_args.bind(
        *(ctypes.cast(f, ctypes.c_void_p).value
          for f in (lib.hypno_hip_append_kv_dev, lib.hypno_hip_paged_attention_dev)),
        torch._C._cuda_getDevice, torch._C._cuda_getCurrentRawStream)
    _args = _attention_args


def _rows(t, what: str):
    """A [tokens, heads, head_dim] float32 tensor whose heads are contiguous: its shape,
    the floats from one token to the next and its device's index."""
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a GPU tensor")
    shape = t.shape
    if t.dtype is not torch.float32 or len(shape) != 3:
        raise ValueError(f"{what} must be float32 [tokens, heads, head_dim], got {t.dtype} "
                         f"{list(shape)}")
    n, h, d = shape
    s, sh, sd = t.stride()
    if n and h and d:
        if (sd != 1 and d > 1) or (sh != d and h > 1):
            raise ValueError(f"{what}: the heads of a token must be contiguous")
        if n == 1:
            s = h * d
        elif s < h * d:
            raise ValueError(f"{what}: tokens overlap")
    else:
        s = h * d
    return n, h, d, s, t.get_device()


def _empty(q):
    """(contiguous, whatever q's strides are)"""
    return torch.empty_like(q) if q.is_contiguous() else q.new_empty(q.shape)


def _page_stride(t, what: str) -> int:
    """Elements from one page to the next, 0 if there is one page or none."""
    inner = 1
    shape, stride = t.shape, t.stride()
    for i in range(len(shape) - 1, 0, -1):
        if shape[i] > 1 and stride[i] != inner:
            raise ValueError(f"{what}: the elements of a page must be contiguous")
        inner *= shape[i]
    if shape[0] <= 1 or stride[0] == inner:
        return 0
    if stride[0] < inner:
        raise ValueError(f"{what}: pages overlap")
    return stride[0]


def _cache(k_cache, v_cache, k_scale, v_scale, dev: int):
    """The packed cache, its kv heads and head_dim."""
    if not isinstance(k_cache, torch.Tensor) or not isinstance(v_cache, torch.Tensor) or \
            k_cache.get_device() != dev or v_cache.get_device() != dev:
        raise ValueError(f"k_cache and v_cache must be tensors on GPU {dev}")
    dtype, shape = k_cache.dtype, k_cache.shape
    int8 = dtype is torch.int8
    if not int8 and dtype is not torch.float16:
        raise ValueError(f"k_cache must be float16 or int8, got {dtype}")
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype is not dtype:
        raise ValueError("k_cache and v_cache must be [pages, kv_heads, page_size, head_dim] of "
                         "one type")
    pages, heads, size, dim = shape
    ks = vs = kss = vss = 0
    if int8:
        for t, what in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if not isinstance(t, torch.Tensor) or t.get_device() != dev or \
                    t.dtype is not torch.float32 or t.shape != shape[:3]:
                raise ValueError(f"{what} must be float32 [pages, kv_heads, page_size] on "
                                 f"GPU {dev} beside an int8 cache")
        ks, kss = k_scale.data_ptr(), _page_stride(k_scale, "k_scale")
        vs, vss = v_scale.data_ptr(), _page_stride(v_scale, "v_scale")
    elif k_scale is not None or v_scale is not None:
        raise ValueError("a float16 cache has no scales")
    return _CACHE.pack(int8, k_cache.data_ptr(), v_cache.data_ptr(), ks, vs, pages, heads,
                       size, dim,
                       0 if k_cache.is_contiguous() else _page_stride(k_cache, "k_cache"),
                       0 if v_cache.is_contiguous() else _page_stride(v_cache, "v_cache"),
                       kss, vss), heads, dim


def _batch(page_table, kv_lens, cu_q, tokens: int, dev: int):
    try:
        n, width = page_table.shape
        (lens,), (cus,) = kv_lens.shape, cu_q.shape
        int32 = torch.int32
        if page_table.dtype is int32 and kv_lens.dtype is int32 and cu_q.dtype is int32 and \
                page_table.get_device() == dev and kv_lens.get_device() == dev and \
                cu_q.get_device() == dev and page_table.is_contiguous() and \
                kv_lens.is_contiguous() and cu_q.is_contiguous() and lens == n and cus == n + 1:
            return _BATCH.pack(cu_q.data_ptr(), kv_lens.data_ptr(), page_table.data_ptr(), n,
                               width, tokens)
    except (AttributeError, TypeError, ValueError):
        pass
    raise ValueError("page_table [sequences, width], kv_lens [sequences] and cu_q [sequences + 1] "
                     f"must be contiguous int32 tensors on GPU {dev}")


def _call(fn, where: str, dev: int, *args) -> None:
    if torch.cuda.current_device() == dev:
        status = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    else:
        with torch.cuda.device(dev):
            status = fn(*args, torch._C._cuda_getCurrentRawStream(dev))
    if status:
        check(status, where)


def _done(result, where: str):
    if type(result) is int:
        check(result, where)
    return result


def append_kv(q, k, v, k_cache, v_cache, page_table, kv_lens, cu_q, inv_freq=None,
              style: str = "halves", k_scale=None, v_scale=None, out=None):
    """Rotates the new tokens' q and k to their positions, writes k and v to their
    places in the cache, and returns the rotated q (a new tensor, or `out`, which may
    be q).  inv_freq: float32 [rot_dim / 2], pair j turns by position * inv_freq[j];
    None: no rotation.  style "halves": pair j is elements j and j + rot_dim / 2;
    "pairs": 2j and 2j + 1.  q may be None (k and v only).  int8 caches: see
    include/hypno_hip.h for the codes."""
    if _args is None:
        _torch()
    if style not in _STYLES:
        raise ValueError(f"style must be 'halves' or 'pairs', got {style!r}")
    done = _args.append_kv(q, k, v, k_cache, v_cache, page_table, kv_lens, cu_q, inv_freq,
                           _STYLES[style], k_scale, v_scale, out)
    if done is not NotImplemented:
        return _done(done, "append_kv")
    tokens, kv_heads, dim, k_stride, dev = _rows(k, "k")
    n, vh, vd, v_stride, vdev = _rows(v, "v")
    if n != tokens or vh != kv_heads or vd != dim or vdev != dev:
        raise ValueError("k and v differ in shape or device")
    heads = q_stride = o_stride = rot = 0
    qp = op = fp = None
    if q is not None:
        n, heads, qd, q_stride, qdev = _rows(q, "q")
        if n != tokens or qd != dim or qdev != dev:
            raise ValueError("q and k differ in tokens, head_dim or device")
        if out is None:
            out = _empty(q)
            o_stride = heads * dim
        else:
            n, oh, od, o_stride, odev = _rows(out, "out")
            if n != tokens or oh != heads or od != dim or odev != dev:
                raise ValueError("q and out differ in shape or device")
        qp, op = q.data_ptr(), out.data_ptr()
    elif out is not None:
        raise ValueError("out without q")
    if inv_freq is not None:
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.get_device() != dev or \
                inv_freq.dtype is not torch.float32 or inv_freq.dim() != 1 or \
                not inv_freq.is_contiguous():
            raise ValueError(f"inv_freq must be a contiguous float32 [rot_dim / 2] on GPU {dev}")
        rot, fp = 2 * inv_freq.shape[0], inv_freq.data_ptr()
        if rot > dim:
            raise ValueError(f"inv_freq has {rot // 2} values for a head_dim of {dim}")
    cache, ch, cd = _cache(k_cache, v_cache, k_scale, v_scale, dev)
    if ch != kv_heads or cd != dim:
        raise ValueError(f"k is {list(k.shape)} for a cache of {ch} kv heads of {cd}")
    _call(load().hypno_hip_append_kv_dev, "append_kv", dev, cache,
          _batch(page_table, kv_lens, cu_q, tokens, dev), op, o_stride, qp, q_stride, heads,
          k.data_ptr(), k_stride, v.data_ptr(), v_stride, fp, rot, _STYLES[style])
    return out


def paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_q, scale=None, window: int = 0,
                    k_scale=None, v_scale=None, max_kv_len=None, out=None):
    """Attention of the new tokens over their sequences' pages, [tokens, heads,
    head_dim] float32 (a new tensor, or the contiguous `out`).  A token sees the
    positions up to its own, with window > 0 the last `window` of them; one that sees
    nothing gets zeros.  Head h reads kv head h // (heads / kv_heads).  scale: of the
    scores, by default head_dim ** -0.5.  max_kv_len: an upper bound of kv_lens, if the
    host knows one (default: what page_table has room for); it decides how many
    work-groups share a sequence."""
    if _args is None:
        _torch()
    done = _args.paged_attention(q, k_cache, v_cache, page_table, kv_lens, cu_q, scale, window,
                                 k_scale, v_scale, max_kv_len, out)
    if done is not NotImplemented:
        return _done(done, "paged_attention")
    tokens, heads, dim, q_stride, dev = _rows(q, "q")
    cache, kv_heads, cd = _cache(k_cache, v_cache, k_scale, v_scale, dev)
    if cd != dim or not kv_heads or heads % kv_heads:
        raise ValueError(f"q is {list(q.shape)} for a cache of {kv_heads} kv heads of {cd}")
    if window < 0:
        raise ValueError("window must not be negative")
    if max_kv_len is None:
        max_kv_len = 0
    elif max_kv_len < 0:
        raise ValueError("max_kv_len must not be negative")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    if out is None:
        out = _empty(q)
    elif not isinstance(out, torch.Tensor) or out.get_device() != dev or \
            out.dtype is not torch.float32 or out.shape != q.shape or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous float32 {list(q.shape)} on GPU {dev}")
    _call(load().hypno_hip_paged_attention_dev, "paged_attention", dev, out.data_ptr(),
          q.data_ptr(), q_stride, heads, cache, _batch(page_table, kv_lens, cu_q, tokens, dev),
          scale, window, max_kv_len)
    return out
