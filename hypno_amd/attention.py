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
(-1 for a freed one, say) is not written, and what reads it is NaN.

The caches are [pages, kv_heads, page_size, head_dim], float16, or int8 with
float32 k_scale and v_scale [pages, kv_heads, page_size]: one scale a token and kv
head.  Pages may be strided (a pool of [pages, layers, ...]); the rest is contiguous.

Arguments that cannot be right raise ValueError; a library failure raises
HypnoHipError.
"""
from __future__ import annotations

import ctypes
import math

from ._lib import KvBatch, KvCache, check, load

__all__ = ["append_kv", "paged_attention"]

_STYLES = {"halves": 0, "pairs": 1}  # HYPNO_HIP_ROPE_*


def _torch():
    import torch
    return torch


def _rows(t, what: str, heads=None, head_dim=None):
    """A [tokens, heads, head_dim] float32 tensor whose heads are contiguous: its
    floats from one token to the next."""
    torch = _torch()
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise ValueError(f"{what} must be a GPU tensor")
    if t.dtype != torch.float32 or t.dim() != 3:
        raise ValueError(f"{what} must be float32 [tokens, heads, head_dim], got {t.dtype} "
                         f"{list(t.shape)}")
    n, h, d = t.shape
    if (heads is not None and h != heads) or (head_dim is not None and d != head_dim):
        raise ValueError(f"{what} is {list(t.shape)}, expected [tokens, {heads}, {head_dim}]")
    if t.numel() and ((d > 1 and t.stride(2) != 1) or (h > 1 and t.stride(1) != d)):
        raise ValueError(f"{what}: the heads of a token must be contiguous")
    if n <= 1 or not t.numel():
        return h * d
    if t.stride(0) < h * d:
        raise ValueError(f"{what}: tokens overlap")
    return t.stride(0)


def _page_stride(t, what: str) -> int:
    """Elements from one page to the next, 0 if there is one page or none."""
    inner = 1
    for i in range(t.dim() - 1, 0, -1):
        if t.shape[i] > 1 and t.stride(i) != inner:
            raise ValueError(f"{what}: the elements of a page must be contiguous")
        inner *= t.shape[i]
    if t.shape[0] <= 1 or t.stride(0) == inner:
        return 0
    if t.stride(0) < inner:
        raise ValueError(f"{what}: pages overlap")
    return t.stride(0)


def _cache(k_cache, v_cache, k_scale, v_scale, device):
    torch = _torch()
    for t, what in ((k_cache, "k_cache"), (v_cache, "v_cache")):
        if not isinstance(t, torch.Tensor) or t.device != device:
            raise ValueError(f"{what} must be a tensor on {device}")
    dtype, shape = k_cache.dtype, k_cache.shape
    if dtype not in (torch.float16, torch.int8):
        raise ValueError(f"k_cache must be float16 or int8, got {dtype}")
    if len(shape) != 4 or v_cache.shape != shape or v_cache.dtype != dtype:
        raise ValueError("k_cache and v_cache must be [pages, kv_heads, page_size, head_dim] of "
                         "one type")
    strides = [_page_stride(k_cache, "k_cache"), _page_stride(v_cache, "v_cache"), 0, 0]
    ks = vs = None
    if dtype == torch.int8:
        for i, (t, what) in enumerate(((k_scale, "k_scale"), (v_scale, "v_scale"))):
            if not isinstance(t, torch.Tensor) or t.device != device or \
                    t.dtype != torch.float32 or t.shape != shape[:3]:
                raise ValueError(f"{what} must be float32 [pages, kv_heads, page_size] on "
                                 f"{device} beside an int8 cache")
            strides[2 + i] = _page_stride(t, what)
        ks, vs = k_scale.data_ptr(), v_scale.data_ptr()
    elif k_scale is not None or v_scale is not None:
        raise ValueError("a float16 cache has no scales")
    return KvCache(int(dtype == torch.int8), k_cache.data_ptr(), v_cache.data_ptr(), ks, vs,
                   *shape, *strides)


def _batch(page_table, kv_lens, cu_q, tokens: int, device):
    torch = _torch()
    for t, what, dim in ((page_table, "page_table", 2), (kv_lens, "kv_lens", 1),
                         (cu_q, "cu_q", 1)):
        if not isinstance(t, torch.Tensor) or t.device != device or t.dtype != torch.int32 or \
                t.dim() != dim or not t.is_contiguous():
            raise ValueError(f"{what} must be a contiguous int32 tensor of {dim} dimension(s) on "
                             f"{device}")
    n = kv_lens.shape[0]
    if page_table.shape[0] != n or cu_q.shape[0] != n + 1:
        raise ValueError(f"page_table {list(page_table.shape)}, kv_lens [{n}] and cu_q "
                         f"[{cu_q.shape[0]}] are not of one batch")
    return KvBatch(cu_q.data_ptr(), kv_lens.data_ptr(), page_table.data_ptr(), n,
                   page_table.shape[1], tokens)


def _call(fn, where: str, device, *args) -> None:
    torch = _torch()
    stream = torch.cuda.current_stream(device).cuda_stream
    if torch.cuda.current_device() == device.index:
        check(fn(*args, stream), where)
    else:
        with torch.cuda.device(device):
            check(fn(*args, stream), where)


def append_kv(q, k, v, k_cache, v_cache, page_table, kv_lens, cu_q, inv_freq=None,
              style: str = "halves", k_scale=None, v_scale=None, out=None):
    """Rotates the new tokens' q and k to their positions, writes k and v to their
    places in the cache, and returns the rotated q (a new tensor, or `out`, which may
    be q).  inv_freq: float32 [rot_dim / 2], pair j turns by position * inv_freq[j];
    None: no rotation.  style "halves": pair j is elements j and j + rot_dim / 2;
    "pairs": 2j and 2j + 1.  q may be None (k and v only).  int8 caches: see
    include/hypno_hip.h for the codes."""
    torch = _torch()
    if style not in _STYLES:
        raise ValueError(f"style must be 'halves' or 'pairs', got {style!r}")
    k_stride = _rows(k, "k")
    tokens, kv_heads, dim = k.shape
    device = k.device
    v_stride = _rows(v, "v", kv_heads, dim)
    heads = q_stride = o_stride = 0
    qp = op = fp = None
    rot = 0
    if q is not None:
        q_stride = _rows(q, "q", None, dim)
        heads = q.shape[1]
        if out is None:
            out = torch.empty((tokens, heads, dim), dtype=torch.float32, device=device)
        o_stride = _rows(out, "out", heads, dim)
        if q.shape[0] != tokens or out.shape[0] != tokens or q.device != device or \
                out.device != device:
            raise ValueError("q, k and out differ in tokens or device")
        qp, op = q.data_ptr(), out.data_ptr()
    elif out is not None:
        raise ValueError("out without q")
    if v.shape[0] != tokens or v.device != device:
        raise ValueError("k and v differ in tokens or device")
    if inv_freq is not None:
        if not isinstance(inv_freq, torch.Tensor) or inv_freq.device != device or \
                inv_freq.dtype != torch.float32 or inv_freq.dim() != 1 or \
                not inv_freq.is_contiguous():
            raise ValueError(f"inv_freq must be a contiguous float32 [rot_dim / 2] on {device}")
        rot, fp = 2 * inv_freq.shape[0], inv_freq.data_ptr()
        if rot > dim:
            raise ValueError(f"inv_freq has {rot // 2} values for a head_dim of {dim}")
    cache = _cache(k_cache, v_cache, k_scale, v_scale, device)
    if cache.kv_heads != kv_heads or cache.head_dim != dim:
        raise ValueError(f"k is {list(k.shape)} for a cache of {cache.kv_heads} kv heads of "
                         f"{cache.head_dim}")
    batch = _batch(page_table, kv_lens, cu_q, tokens, device)
    _call(load().hypno_hip_append_kv_dev, "append_kv", device, ctypes.byref(cache),
          ctypes.byref(batch), op, o_stride, qp, q_stride, heads, k.data_ptr(), k_stride,
          v.data_ptr(), v_stride, fp, rot, _STYLES[style])
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
    torch = _torch()
    q_stride = _rows(q, "q")
    tokens, heads, dim = q.shape
    device = q.device
    cache = _cache(k_cache, v_cache, k_scale, v_scale, device)
    if cache.head_dim != dim or not cache.kv_heads or heads % cache.kv_heads:
        raise ValueError(f"q is {list(q.shape)} for a cache of {cache.kv_heads} kv heads of "
                         f"{cache.head_dim}")
    if window < 0:
        raise ValueError("window must not be negative")
    if max_kv_len is not None and max_kv_len < 0:
        raise ValueError("max_kv_len must not be negative")
    if scale is None:
        scale = 1.0 / math.sqrt(dim)
    if out is None:
        out = torch.empty((tokens, heads, dim), dtype=torch.float32, device=device)
    elif not isinstance(out, torch.Tensor) or out.device != device or \
            out.dtype != torch.float32 or out.shape != q.shape or not out.is_contiguous():
        raise ValueError(f"out must be a contiguous float32 {list(q.shape)} on {device}")
    batch = _batch(page_table, kv_lens, cu_q, tokens, device)
    _call(load().hypno_hip_paged_attention_dev, "paged_attention", device, out.data_ptr(),
          q.data_ptr(), q_stride, heads, ctypes.byref(cache), ctypes.byref(batch), float(scale),
          int(window), int(max_kv_len or 0))
    return out
