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
head.  In 4 bits they are uint8 [pages, kv_heads, page_size, head_dim / 2] with
float16 k_scale and v_scale [pages, kv_heads, head_dim / 32, page_size]: one scale
for 32 elements (head_dim: a multiple of 32, page_size: 16 or more).  Pages may be
strided (a pool of [pages, layers, ...]); the rest is contiguous.

Of a long context a token may read some pages only, chosen by a cheap score of each:

    key_bounds(k_cache, bounds, bounds_scale, page_table, kv_lens, cu_q)
    pages = select_pages(q, bounds, bounds_scale, page_size, page_table, kv_lens, cu_q, count)
    o = selected_attention(q, k_cache, v_cache, pages, page_table, kv_lens, cu_q)

after append_kv and in place of paged_attention.  The bounds (int8 [pages, kv_heads, 2,
head_dim] and float32 [pages, kv_heads], kept beside the cache, any type of it) hold
each page's smallest and largest key in every channel.

Arguments that cannot be right raise ValueError; a library failure raises
HypnoHipError.
"""
from __future__ import annotations

import ctypes
import math
import struct

from ._lib import check, load

__all__ = ["append_kv", "paged_attention", "key_bounds", "select_pages", "selected_attention"]

_STYLES = {"halves": 0, "pairs": 1}  # HYPNO_HIP_ROPE_*

# The structs of include/hypno_hip.h (_lib.KvCache, KvBatch and KeyBounds), packed at once.
_CACHE = struct.Struct("=I4x12Q")
_BATCH = struct.Struct("=6Q")
_BOUNDS = struct.Struct("=8Q")

_ANY = 0x7FFFFFFF  # tokens of a batch whose rows are in no tensor of the call

torch = None
_args = None  # csrc/attention_args.cpp: the same checks and packing, where all is right


class _NoArgs:
    """Stands for it where it was not built."""

    @staticmethod
    def append_kv(*_):
        return NotImplemented

    paged_attention = key_bounds = select_pages = selected_attention = append_kv


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
          for f in (lib.hypno_hip_append_kv_dev, lib.hypno_hip_paged_attention_dev,
                    lib.hypno_hip_key_bounds_dev, lib.hypno_hip_select_pages_dev,
                    lib.hypno_hip_selected_attention_dev)),
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
    int8, fp4 = dtype is torch.int8, dtype is torch.uint8
    if not int8 and not fp4 and dtype is not torch.float16:
        raise ValueError(f"k_cache must be float16, int8 or uint8 (two 4-bit codes), got {dtype}")
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype is not dtype:
        raise ValueError("k_cache and v_cache must be [pages, kv_heads, page_size, head_dim] of "
                         "one type")
    pages, heads, size, dim = shape
    ks = vs = kss = vss = 0
    if fp4:
        dim *= 2
        want = (pages, heads, dim // 32, size)
        for t, what in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if not isinstance(t, torch.Tensor) or t.get_device() != dev or \
                    t.dtype is not torch.float16 or t.shape != want:
                raise ValueError(f"{what} must be float16 [pages, kv_heads, head_dim / 32, "
                                 f"page_size] on GPU {dev} beside a 4-bit cache")
        ks, kss = k_scale.data_ptr(), _page_stride(k_scale, "k_scale")
        vs, vss = v_scale.data_ptr(), _page_stride(v_scale, "v_scale")
    elif int8:
        for t, what in ((k_scale, "k_scale"), (v_scale, "v_scale")):
            if not isinstance(t, torch.Tensor) or t.get_device() != dev or \
                    t.dtype is not torch.float32 or t.shape != shape[:3]:
                raise ValueError(f"{what} must be float32 [pages, kv_heads, page_size] on "
                                 f"GPU {dev} beside an int8 cache")
        ks, kss = k_scale.data_ptr(), _page_stride(k_scale, "k_scale")
        vs, vss = v_scale.data_ptr(), _page_stride(v_scale, "v_scale")
    elif k_scale is not None or v_scale is not None:
        raise ValueError("a float16 cache has no scales")
    return _CACHE.pack(2 if fp4 else int8, k_cache.data_ptr(), v_cache.data_ptr(), ks, vs, pages, heads,
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


def _bounds(bounds, scale, page_size: int, dev: int):
    """The packed bounds, their kv heads and head_dim."""
    if not isinstance(bounds, torch.Tensor) or bounds.get_device() != dev or \
            bounds.dtype is not torch.int8 or bounds.dim() != 4 or bounds.shape[2] != 2:
        raise ValueError(f"bounds must be int8 [pages, kv_heads, 2, head_dim] on GPU {dev}")
    if not isinstance(scale, torch.Tensor) or scale.get_device() != dev or \
            scale.dtype is not torch.float32 or scale.shape != bounds.shape[:2]:
        raise ValueError(f"bounds_scale must be float32 [pages, kv_heads] on GPU {dev}")
    pages, heads, _, dim = bounds.shape
    return _BOUNDS.pack(bounds.data_ptr(), scale.data_ptr(), pages, heads, page_size, dim,
                        _page_stride(bounds, "bounds"),
                        _page_stride(scale, "bounds_scale")), heads, dim


def _whole(x, what: str, least: int) -> int:
    if not isinstance(x, int) or x < least:
        raise ValueError(f"{what} must be a whole number from {least} on, got {x!r}")
    return min(x, 1 << 62)


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


def key_bounds(k_cache, bounds, bounds_scale, page_table, kv_lens, cu_q, k_scale=None):
    """Computes the bounds (see above) of every page that holds a new token of the batch,
    from all of the page's tokens below kv_lens; other pages' are left alone.  Called
    after append_kv; with cu_q counting all tokens of a sequence, for all of its pages.
    include/hypno_hip.h has the codes."""
    if _args is None:
        _torch()
    done = _args.key_bounds(k_cache, bounds, bounds_scale, page_table, kv_lens, cu_q, k_scale)
    if done is not NotImplemented:
        return _done(done, "key_bounds")
    if not isinstance(k_cache, torch.Tensor) or not k_cache.is_cuda:
        raise ValueError("k_cache must be a GPU tensor")
    dev = k_cache.get_device()
    cache, heads, dim = _cache(k_cache, k_cache, k_scale, k_scale, dev)
    packed, bh, bd = _bounds(bounds, bounds_scale, k_cache.shape[2], dev)
    if bh != heads or bd != dim or bounds.shape[0] != k_cache.shape[0]:
        raise ValueError(f"bounds of {list(bounds.shape)} for a cache of {k_cache.shape[0]} pages, "
                         f"{heads} kv heads of {dim}")
    _call(load().hypno_hip_key_bounds_dev, "key_bounds", dev, packed, cache,
          _batch(page_table, kv_lens, cu_q, _ANY, dev))


def select_pages(q, bounds, bounds_scale, page_size: int, page_table, kv_lens, cu_q, count: int,
                 first: int = 1, last: int = 1, max_kv_len=None, out=None):
    """The pages that each token is to read for each kv head: int32 [tokens, kv_heads,
    count] (a new tensor, or the contiguous `out`), numbers of the sequence's pages,
    ascending, -1 behind them.  The sequence's first `first` pages and the last `last` up to
    the token's own are always among them, then those with the largest score: the most
    that q . k can be for a key within the page's bounds, in 8-bit codes, the largest over
    the kv head's query heads; the lower page first among equal ones.  max_kv_len: an upper
    bound of kv_lens, if the host knows one (default: what page_table has room for, which
    may be 32768 pages at most); pages past it have no score."""
    if _args is None:
        _torch()
    done = _args.select_pages(q, bounds, bounds_scale, page_size, page_table, kv_lens, cu_q, count,
                              first, last, max_kv_len, out)
    if done is not NotImplemented:
        return _done(done, "select_pages")
    tokens, heads, dim, q_stride, dev = _rows(q, "q")
    packed, kv_heads, bd = _bounds(bounds, bounds_scale, _whole(page_size, "page_size", 1), dev)
    if bd != dim or not kv_heads or heads % kv_heads:
        raise ValueError(f"q is {list(q.shape)} for bounds of {kv_heads} kv heads of {bd}")
    count, first, last = _whole(count, "count", 1), _whole(first, "first", 0), \
        _whole(last, "last", 1)
    if first + last > count or count > 1024:
        raise ValueError(f"count {count} is above 1024, or below first {first} and last {last}")
    most = 0 if max_kv_len is None else _whole(max_kv_len, "max_kv_len", 0)
    shape = (tokens, kv_heads, count)
    if out is None:
        out = torch.empty(shape, dtype=torch.int32, device=q.device)
    elif not isinstance(out, torch.Tensor) or out.get_device() != dev or \
            out.dtype is not torch.int32 or out.shape != shape or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous int32 {list(shape)} on GPU {dev}")
    _call(load().hypno_hip_select_pages_dev, "select_pages", dev, out.data_ptr(), count, first,
          last, q.data_ptr(), q_stride, heads, packed,
          _batch(page_table, kv_lens, cu_q, tokens, dev), most)
    return out


def selected_attention(q, k_cache, v_cache, selected, page_table, kv_lens, cu_q, scale=None,
                       k_scale=None, v_scale=None, out=None):
    """paged_attention over the positions up to a token's own that are in its selected
    pages: `selected` is what select_pages gives, or any contiguous int32 [tokens, kv_heads,
    count].  Numbers below 0 or past the token's own page are passed over, a page that is
    named twice counts twice; a token without any gets zeros.  Pages of 16 tokens at
    least."""
    if _args is None:
        _torch()
    done = _args.selected_attention(q, k_cache, v_cache, selected, page_table, kv_lens, cu_q,
                                    scale, k_scale, v_scale, out)
    if done is not NotImplemented:
        return _done(done, "selected_attention")
    tokens, heads, dim, q_stride, dev = _rows(q, "q")
    cache, kv_heads, cd = _cache(k_cache, v_cache, k_scale, v_scale, dev)
    if cd != dim or not kv_heads or heads % kv_heads:
        raise ValueError(f"q is {list(q.shape)} for a cache of {kv_heads} kv heads of {cd}")
    if not isinstance(selected, torch.Tensor) or selected.get_device() != dev or \
            selected.dtype is not torch.int32 or selected.dim() != 3 or \
            selected.shape[:2] != (tokens, kv_heads) or not selected.is_contiguous() or \
            not 0 < selected.shape[2] <= 1024:
        raise ValueError(f"selected must be a contiguous int32 [{tokens}, {kv_heads}, 1 to 1024] on "
                         f"GPU {dev}")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    if out is None:
        out = _empty(q)
    elif not isinstance(out, torch.Tensor) or out.get_device() != dev or \
            out.dtype is not torch.float32 or out.shape != q.shape or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous float32 {list(q.shape)} on GPU {dev}")
    _call(load().hypno_hip_selected_attention_dev, "selected_attention", dev, out.data_ptr(),
          q.data_ptr(), q_stride, heads, cache, _batch(page_table, kv_lens, cu_q, tokens, dev),
          scale, selected.data_ptr(), selected.shape[2])
    return out
