"""Many sequences over one paged INT8 KV cache (no counterpart in the
reference, which serves one request at a time over contiguous caches).

A cache is the tuple (k_codes, k_scales, v_codes, v_scales) of symmetric int8
codes [pages,Hkv,page_size,D] and fp16 scales [pages,Hkv,page_size], the "s8"
format of kv_append and int8_quantized_sdpa in pages; a pool of several layers
has a leading layer axis. A batch is described by three int32 tensors on the
device that no call reads back:

  page_table [B,M]  the pages of each sequence; an entry outside the pool is
                    no page
  lengths    [B]    tokens of each sequence, the new ones included: at most
                    M * page_size (and taken as that where they are more)
  starts     [B+1]  the packed rows of each sequence's new tokens are
                    starts[b] .. starts[b+1] - 1, its last token the last one

Like every sparkq operator these enqueue on the current stream of the tensors'
device and return without synchronising. Each call's scratch comes from torch's
allocator, so threads on one stream and captured graphs share none.
"""

from __future__ import annotations

import math
import struct

import torch

from . import _lib
from .ext import _HALF, _out_buffer, _ptr

__all__ = ["PagedKVCache", "kv_pages_compact", "kv_pages_evict", "kv_pages_fork",
           "paged_key_bounds", "paged_kv_append", "paged_kv_mass", "paged_page_scores",
           "paged_quantized_sdpa", "paged_sparse_sdpa", "select_top"]


_T = torch.Tensor
_CONTIGUOUS = torch.contiguous_format
# int64 arrays for a call (bytes: a fifth of a ctypes array's time)
_I64x2, _I64x3, _I64x4, _I64x6, _I64x8, _I64x12 = (struct.Struct(f"{n}q").pack
                                                   for n in (2, 3, 4, 6, 8, 12))
_CODE = {torch.float32: _lib.F32, torch.float16: _lib.F16, torch.bfloat16: _lib.BF16}


def _check_cache(op, cache, ndim):
    """((k_codes, k_scales, v_codes, v_scales), their GPU, codes' shape) of a
    cache with `ndim` axes in its codes."""
    kc, ks, vc, vs = cache if len(cache) == 4 else (None,) * 4
    if not (isinstance(kc, _T) and isinstance(ks, _T) and isinstance(vc, _T) and isinstance(vs, _T)):
        raise ValueError(f"{op}: the cache is (k_codes, k_scales, v_codes, v_scales)")
    shape, scales = kc.shape, ks.shape
    if (len(shape) != ndim or vc.shape != shape or scales != shape[:-1] or vs.shape != scales
            or kc.dtype is not torch.int8 or vc.dtype is not torch.int8
            or ks.dtype is not torch.float16 or vs.dtype is not torch.float16):
        raise ValueError(f"{op}: the cache holds int8 codes [pages,Hkv,page_size,D] and fp16 "
                         "scales [pages,Hkv,page_size] of keys and of values")
    index = kc.get_device()
    if ks.get_device() != index or vc.get_device() != index or vs.get_device() != index:
        raise ValueError(f"{op}: the cache's tensors must live on one device")
    return kc, ks, vc, vs, index, shape


def _need_gpu(op, index):
    if index < 0:
        raise ValueError(f"{op} requires GPU execution")


def _check_ints(op, index, name, t, shape):
    if t.dtype is not torch.int32 or t.shape != shape:
        raise ValueError(f"{op}: {name} must be an int32 tensor of shape {list(shape)}")
    if t.get_device() != index:
        raise ValueError(f"{op}: {name} must live on the cache's device")
    if shape[-1] > 1 and t.stride(-1) != 1:
        raise ValueError(f"{op}: the last axis of {name} must be contiguous")


def _check_rows(op, index, page_table, lengths):
    """(sequences, pages per row) of a batch's table and lengths."""
    shape = page_table.shape
    if len(shape) != 2 or shape[1] < 1:
        raise ValueError(f"{op}: expected page_table [B,M] and lengths [B]")
    b, width = shape
    if not (page_table.dtype is torch.int32 and page_table.is_contiguous()
            and page_table.get_device() == index and lengths.dtype is torch.int32
            and lengths.shape == (b,) and lengths.is_contiguous()
            and lengths.get_device() == index):  # (one test of what is nearly always so)
        _check_ints(op, index, "page_table", page_table, shape)
        _check_ints(op, index, "lengths", lengths, (b,))
    return b, width


def _check_batch(op, index, page_table, starts, lengths):
    """(sequences, pages per row) of a batch."""
    b, width = _check_rows(op, index, page_table, lengths)
    if not (starts.dtype is torch.int32 and starts.shape == (b + 1,) and starts.is_contiguous()
            and starts.get_device() == index):
        _check_ints(op, index, "starts", starts, (b + 1,))
    return b, width


def _strides(op, kc, ks, vc, vs):
    a0, a1, a2, a3 = kc.stride()
    b0, b1, b2, b3 = vc.stride()
    if a3 != 1 or b3 != 1:
        raise ValueError(f"{op}: the codes' innermost axes must be contiguous")
    return _I64x12(a0, a1, a2, *ks.stride(), b0, b1, b2, *vs.stride())


def _rows16(t):
    """(t, its strides) with rows that 16-byte loads can read: itself, or a copy."""
    n = 16 // t.element_size()
    st = t.stride()
    if st[2] == 1 and st[0] % n == 0 and st[1] % n == 0 and t.data_ptr() % 16 == 0:
        return t, st
    t = t.clone(memory_format=torch.contiguous_format)
    return t, t.stride()


def _check_attention(op, queries, hkv, d, index, mask, scale, max_new):
    if queries.ndim != 3 or queries.shape[2] != d or not queries.shape[1] \
            or queries.shape[1] % hkv:
        raise ValueError(f"{op}: queries must be [T,Hq,{d}] with Hq divisible by {hkv}")
    if queries.dtype not in _HALF:
        raise ValueError(f"{op} requires float16 or bfloat16 queries")
    if queries.get_device() != index:
        raise ValueError(f"{op}: queries must live on the cache's device")
    if mask is not None and mask != "causal":
        raise ValueError(f"{op} takes mask=None or mask='causal'")
    if not isinstance(scale, (float, int)) or not math.isfinite(scale):
        raise ValueError("scale must be a finite Python number")
    _check_max_new(op, max_new)


def _check_max_new(op, max_new):
    if type(max_new) is not int or max_new < 1:
        raise ValueError(f"{op}: max_new must be a positive Python int")


def _out_dtype(queries, out_dtype):
    out_dtype = queries.dtype if out_dtype is None else out_dtype
    if out_dtype is not queries.dtype and out_dtype is not torch.float32:
        raise ValueError("out_dtype must be the query dtype or torch.float32")
    return out_dtype


def paged_kv_append(keys, values, cache, page_table, starts, lengths):
    """Quantize a batch's new tokens into their pages, in place: keys and
    values [T,Hkv,D] (float16, bfloat16 or float32; views of a packed
    projection are read in place), one layer's cache. The formula is
    kv_quantize_s8's. Rows that fall to no sequence, tokens before position 0
    and tokens without a page are skipped. Sequences that append must not share
    the page they append to: kv_pages_fork gives each its own. Calls that write
    one cache are ordered by their stream."""
    op = "paged_kv_append"
    kc, ks, vc, vs, index, (pages, hkv, page, d) = _check_cache(op, cache, 4)
    if keys.ndim != 3 or keys.shape[1:] != (hkv, d) or values.shape != keys.shape:
        raise ValueError(f"{op}: keys and values must be [T,{hkv},{d}] like the cache")
    dtype = keys.dtype
    if dtype not in _CODE or values.dtype is not dtype:
        raise ValueError(f"{op}: keys and values must be float16, bfloat16 or float32, both alike")
    if keys.get_device() != index or values.get_device() != index:
        raise ValueError(f"{op}: keys and values must live on the cache's device")
    b, width = _check_batch(op, index, page_table, starts, lengths)
    strides = _strides(op, kc, ks, vc, vs)
    _need_gpu(op, index)
    (keys, kst), (values, vst) = _rows16(keys), _rows16(values)
    _lib.launch("sparkq_paged_kv_append", index, keys.data_ptr(), values.data_ptr(), kc.data_ptr(),
                ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), page_table.data_ptr(),
                starts.data_ptr(), lengths.data_ptr(), keys.shape[0], b, hkv, d, pages, width,
                page_table.stride(0), page, _CODE[dtype], _I64x4(kst[0], kst[1], vst[0], vst[1]),
                strides)


def paged_quantized_sdpa(queries, cache, page_table, starts, lengths, *, scale, max_new: int,
                         mask="causal", out_dtype=None, out=None, return_lse: bool = False):
    """Attention of a batch's new tokens over their pages: queries [T,Hq,D]
    (float16 or bfloat16) -> [T,Hq,D]. With mask="causal" row i of a
    sequence's n new tokens sees its tokens 0 .. length - n + i, with None all
    of them; tokens without a page are hidden, a row that sees nothing is zero,
    and one that sees a value scale that is not finite has no finite values.
    max_new is the most new tokens that a sequence has (1: a decode step). Rows
    that fall to no sequence, or to more than max_new of one, are left as they
    are in `out`, and hold anything in a new tensor. Codes and scales of keys lie
    as those of values do (the same strides), a page's scales of a head together.
    A weight times its value's scale is held in 22 bits in calls of up to 16 rows
    a sequence and KV head (max_new * Hq / Hkv: decode steps, a few drafted
    tokens) and wherever out_dtype is float32; in others, with 16-bit outputs, in
    float16's 11, which their own rounding is near (float32 outputs cost up to a
    quarter more time there). Scores, normalizer and sums are fp32.

    With return_lse the result is (out, lse [T,Hq] float32): the natural logarithm of
    the sum of each row's exponentiated scores, -inf where it sees nothing. Values and
    their scales have no part in it, finite or not."""
    op = "paged_quantized_sdpa"
    kc, ks, vc, vs, index, (pages, hkv, page, d) = _check_cache(op, cache, 4)
    _check_attention(op, queries, hkv, d, index, mask, scale, max_new)
    t, heads, _ = shape = queries.shape
    dtype, out_dtype = queries.dtype, _out_dtype(queries, out_dtype)
    b, width = _check_batch(op, index, page_table, starts, lengths)
    strides = _strides(op, kc, ks, vc, vs)
    _need_gpu(op, index)
    queries, qst = _rows16(queries)
    out = torch.empty_like(queries, dtype=out_dtype, memory_format=_CONTIGUOUS) if out is None \
        else _out_buffer(out, shape, out_dtype, kc.device)
    need = _lib.lib().sparkq_paged_sdpa_workspace_bytes(t, b, heads, hkv, d, max_new, width * page)
    ws = kc.new_empty(need) if need else None  # (int8: bytes)
    head = (queries.data_ptr(), kc.data_ptr(), ks.data_ptr(), vc.data_ptr(), vs.data_ptr(),
            page_table.data_ptr(), starts.data_ptr(), lengths.data_ptr(), out.data_ptr())
    tail = (t, b, heads, hkv, d, pages, width, page_table.stride(0), page, max_new,
            1 if mask is not None else 0, _CODE[dtype], _CODE[out_dtype], scale,
            _I64x2(qst[0], qst[1]), strides, _ptr(ws), need)
    if not return_lse:
        _lib.launch("sparkq_paged_sdpa", index, *head, *tail)
        return out
    lse = kc.new_empty((t, heads), dtype=torch.float32)
    _lib.launch("sparkq_paged_sdpa_lse", index, *head, lse.data_ptr(), *tail)
    return out, lse


# --- long contexts: which pages a query attends, which tokens a cache keeps -------

def _key_strides(op, kc, ks):
    a0, a1, a2, a3 = kc.stride()
    if a3 != 1:
        raise ValueError(f"{op}: the codes' innermost axes must be contiguous")
    return _I64x6(a0, a1, a2, *ks.stride())


def _check_bounds(op, bounds, index, shape):
    """Strides of bounds [pages,Hkv,2,D]."""
    if not isinstance(bounds, _T) or bounds.dtype is not torch.bfloat16 or bounds.shape != shape:
        raise ValueError(f"{op}: bounds must be a bfloat16 tensor of shape {list(shape)}")
    if bounds.get_device() != index:
        raise ValueError(f"{op}: bounds must live on the cache's device")
    st = bounds.stride()
    if st[3] != 1 or st[2] != shape[3]:
        raise ValueError(f"{op}: the last two axes of bounds must be contiguous")
    return _I64x2(st[0], st[1])


def paged_key_bounds(cache, bounds, page_table, starts, lengths, *, max_new: int):
    """Bounds of the keys of the pages that a batch's new tokens lie in, in place:
    bounds [pages,Hkv,2,D] bfloat16, in each channel the least key of the page's
    tokens rounded down, and the largest rounded up. Called after paged_kv_append
    with its batch, it keeps the bounds of one layer's cache; each page is read as a
    whole, so copies of pages (kv_pages_fork) need no bounds of their own before.
    max_new is the most new tokens that a sequence has. A page with a key scale that
    is not finite is bounded by bfloat16's largest numbers. Sequences with new tokens
    must not share the pages that these lie in."""
    op = "paged_key_bounds"
    kc, ks, _, _, index, (pages, hkv, page, d) = _check_cache(op, cache, 4)
    bst = _check_bounds(op, bounds, index, (pages, hkv, 2, d))
    _check_max_new(op, max_new)
    b, width = _check_batch(op, index, page_table, starts, lengths)
    strides = _key_strides(op, kc, ks)
    _need_gpu(op, index)
    _lib.launch("sparkq_paged_key_bounds", index, kc.data_ptr(), ks.data_ptr(), bounds.data_ptr(),
                page_table.data_ptr(), starts.data_ptr(), lengths.data_ptr(), b, hkv, d, pages,
                width, page_table.stride(0), page, max_new, strides, bst)


def paged_page_scores(queries, bounds, page_table, starts, lengths, *, page_size: int, scale,
                      max_new: int, mask="causal"):
    """Scores of the pages that a batch's new tokens see, (scores [T,Hkv,M] float32,
    seen [T] int32): for row t, KV head h and entry j of its sequence's table row

        max over the head's query heads g of  scale * sum_d max(q[t,g,d] lo, q[t,g,d] hi)

    with the bounds of that page [pages,Hkv,2,D]: no logit of the row with a key of
    the page is larger, but for the rounding of an fp32 sum ((2 D + 2) 2^-24 of its
    terms' sizes; with float16 queries also 2^-39 of the page's largest bound times
    scale * sum |q|). (scale < 0: with min for max.) -inf where the row sees nothing of
    the page, or there is none; a head whose sum is NaN does not count.
    seen counts the pages that each row sees, for select_top:

        scores, seen = paged_page_scores(...)
        pages = select_top(scores, count, lengths=seen, first=1, last=2)
        out = paged_sparse_sdpa(queries, cache, pages, ...)

    Rows that fall to no sequence, or to more than max_new of one, hold anything."""
    op = "paged_page_scores"
    if not isinstance(bounds, _T) or bounds.ndim != 4 or bounds.shape[2] != 2:
        raise ValueError(f"{op}: bounds must be a bfloat16 tensor of shape [pages,Hkv,2,D]")
    (pages, hkv, _, d), index = bounds.shape, bounds.get_device()
    bst = _check_bounds(op, bounds, index, bounds.shape)
    _check_attention(op, queries, hkv, d, index, mask, scale, max_new)
    if type(page_size) is not int or page_size < 16 or page_size > 1024 or page_size & (page_size - 1):
        raise ValueError(f"{op}: page_size must be a power of two from 16 to 1024")
    b, width = _check_batch(op, index, page_table, starts, lengths)
    _need_gpu(op, index)
    queries, qst = _rows16(queries)
    t, heads, _ = queries.shape
    scores = bounds.new_empty((t, hkv, width), dtype=torch.float32)
    seen = bounds.new_empty(t, dtype=torch.int32)
    _lib.launch("sparkq_paged_page_scores", index, queries.data_ptr(), bounds.data_ptr(),
                page_table.data_ptr(), starts.data_ptr(), lengths.data_ptr(), scores.data_ptr(),
                seen.data_ptr(), t, b, heads, hkv, d, pages, width, page_table.stride(0), page_size,
                max_new, 1 if mask is not None else 0, _CODE[queries.dtype], scale,
                _I64x2(qst[0], qst[1]), bst)
    return scores, seen


def select_top(x, count: int, *, lengths=None, first: int = 0, last: int = 0):
    """Places of the `count` largest values of each row of x [...,R,H,N] (float32, 3
    or 4 axes): [...,R,H,count] int32 in ascending order, -1 behind them where a row
    has fewer values. Of row r only the first lengths[r] values count (int32 [R], the
    same for all layers; N without). The first `first` and the last `last` of these
    are taken whatever they are, and among equal values those at the lowest places;
    NaN counts as -inf. first + last is at most count."""
    op = "select_top"
    if not isinstance(x, _T) or x.dtype is not torch.float32 or x.ndim not in (3, 4):
        raise ValueError(f"{op} takes a float32 tensor [R,H,N] or [layers,R,H,N]")
    for name, v, least in (("count", count, 1), ("first", first, 0), ("last", last, 0)):
        if type(v) is not int or v < least:
            raise ValueError(f"{op}: {name} must be a Python int of at least {least}")
    if first + last > count:
        raise ValueError(f"{op}: first and last together must be no more than count")
    (rows, heads, n), index = x.shape[-3:], x.get_device()
    if not n or not heads:
        raise ValueError(f"{op}: rows must not be empty")
    if n > 1 and x.stride(-1) != 1:
        raise ValueError(f"{op}: the last axis of x must be contiguous")
    if lengths is not None:
        _check_ints(op, index, "lengths", lengths, (rows,))
    _need_gpu(op, index)
    layers, st = (x.shape[0], x.stride()) if x.ndim == 4 else (1, (0, *x.stride()))
    out = x.new_empty((*x.shape[:-1], count), dtype=torch.int32)
    _lib.launch("sparkq_select_top", index, x.data_ptr(), _ptr(lengths), out.data_ptr(), layers,
                rows, heads, n, count, first, last, _I64x3(*st[:3]))
    return out


def paged_sparse_sdpa(queries, cache, selected, page_table, starts, lengths, *, scale,
                      max_new: int, mask="causal", out_dtype=None, out=None):
    """paged_quantized_sdpa over selected pages: row t sees, of the tokens that it
    sees there, those of the pages selected[t,h] for KV head h: selected [T,Hkv,count]
    int32, places in its sequence's row of page_table, as select_top returns them.
    Places outside the row (-1), and pages that are absent or that t does not see,
    count for nothing, and a page that is named twice counts twice. Weights times
    value scales are held in 22 bits; scores, normalizer and sums are fp32."""
    op = "paged_sparse_sdpa"
    kc, ks, vc, vs, index, (pages, hkv, page, d) = _check_cache(op, cache, 4)
    _check_attention(op, queries, hkv, d, index, mask, scale, max_new)
    t, heads, _ = shape = queries.shape
    out_dtype = _out_dtype(queries, out_dtype)
    if not isinstance(selected, _T) or selected.ndim != 3 or not selected.shape[2]:
        raise ValueError(f"{op}: selected must be an int32 tensor [T,Hkv,count]")
    count = selected.shape[2]
    _check_ints(op, index, "selected", selected, (t, hkv, count))
    b, width = _check_batch(op, index, page_table, starts, lengths)
    strides = _strides(op, kc, ks, vc, vs)
    _need_gpu(op, index)
    queries, qst = _rows16(queries)
    out = torch.empty_like(queries, dtype=out_dtype, memory_format=_CONTIGUOUS) if out is None \
        else _out_buffer(out, shape, out_dtype, kc.device)
    need = _lib.lib().sparkq_paged_sparse_workspace_bytes(t, heads, hkv, d, count, page)
    ws = kc.new_empty(need) if need else None  # (int8: bytes)
    _lib.launch("sparkq_paged_sparse_sdpa", index, queries.data_ptr(), kc.data_ptr(),
                ks.data_ptr(), vc.data_ptr(), vs.data_ptr(), selected.data_ptr(),
                page_table.data_ptr(), starts.data_ptr(), lengths.data_ptr(), out.data_ptr(), t, b,
                heads, hkv, d, count, pages, width, page_table.stride(0), page, max_new,
                1 if mask is not None else 0, _CODE[queries.dtype], _CODE[out_dtype], scale,
                _I64x2(qst[0], qst[1]), _I64x2(selected.stride(0), selected.stride(1)), strides,
                _ptr(ws), need)
    return out


def _check_mass(op, mass, index, shape):
    if not isinstance(mass, _T) or mass.dtype is not torch.float32 or mass.shape != shape:
        raise ValueError(f"{op}: mass must be a float32 tensor of shape {list(shape)}")
    if mass.get_device() != index:
        raise ValueError(f"{op}: mass must live on the cache's device")
    if mass.stride(-1) != 1:
        raise ValueError(f"{op}: the last axis of mass must be contiguous")


def paged_kv_mass(queries, lse, cache, mass, page_table, starts, lengths, *, scale, max_new: int,
                  mask="causal"):
    """The attention weight that each cached token gathers, in place: mass
    [B,Hkv,M*page_size] float32 grows by the sum of

        exp(scale * q[t,g] . k - lse[t,g])

    over a sequence's new tokens t that see the token and the query heads g of the KV
    head, with queries, cache, scale and mask of the attention and the lse [T,Hq]
    that paged_quantized_sdpa(return_lse=True) returned for them. A batch's new tokens
    start from 0, whatever mass holds there, so a step's tokens are weighed once. Sums
    are fp32, in one order. max_new is the most new tokens that a sequence has; those of
    one past it add nothing. What is seen by a row whose lse is NaN, or has a key
    scale that is not finite, has no finite sum. At most 128 query heads to a KV head."""
    op = "paged_kv_mass"
    kc, ks, _, _, index, (pages, hkv, page, d) = _check_cache(op, cache, 4)
    _check_attention(op, queries, hkv, d, index, mask, scale, max_new)
    t, heads, _ = queries.shape
    if not isinstance(lse, _T) or lse.dtype is not torch.float32 or lse.shape != (t, heads):
        raise ValueError(f"{op}: lse must be a float32 tensor of shape {[t, heads]}")
    if lse.get_device() != index:
        raise ValueError(f"{op}: lse must live on the cache's device")
    b, width = _check_batch(op, index, page_table, starts, lengths)
    _check_mass(op, mass, index, (b, hkv, width * page))
    strides = _key_strides(op, kc, ks)
    _need_gpu(op, index)
    queries, qst = _rows16(queries)
    lse = lse.contiguous()
    _lib.launch("sparkq_paged_kv_mass", index, queries.data_ptr(), lse.data_ptr(), kc.data_ptr(),
                ks.data_ptr(), mass.data_ptr(), page_table.data_ptr(), starts.data_ptr(),
                lengths.data_ptr(), t, b, heads, hkv, d, pages, width, page_table.stride(0), page,
                max_new, 1 if mask is not None else 0, _CODE[queries.dtype], scale,
                _I64x2(qst[0], qst[1]), _I64x2(mass.stride(0), mass.stride(1)), strides)


def _pool(op, cache):
    """(tensors in the C order, their GPU, layers, pages, page_size, bytes of a
    page's codes and scales, strides) of a pool [layers,pages,...] or of one
    layer [pages,...]."""
    layered = len(cache) == 4 and getattr(cache[0], "ndim", 0) == 5
    kc, ks, vc, vs, index, shape = _check_cache(op, cache, 5 if layered else 4)
    pages, hkv, page, d = shape[-4:]
    layers = shape[0] if layered else 1
    cb, sb = hkv * page * d, hkv * page * 2
    bufs = kc.data_ptr(), vc.data_ptr(), ks.data_ptr(), vs.data_ptr()
    if kc.is_contiguous() and vc.is_contiguous() and ks.is_contiguous() and vs.is_contiguous():
        return bufs, index, layers, pages, page, cb, sb, \
            _I64x8(pages * cb, cb, pages * cb, cb, pages * sb, sb, pages * sb, sb)
    st = []
    for t, inner, size in ((kc, (page * d, d, 1), 1), (vc, (page * d, d, 1), 1),
                           (ks, (page, 1), 2), (vs, (page, 1), 2)):
        s = t.stride()
        k = len(inner)
        if any(x != y and n > 1 for x, y, n in zip(s[-k:], inner, t.shape[-k:])):
            raise ValueError(f"{op}: a page must be contiguous in every tensor of the cache")
        st += (s[0] * size if layered else 0, s[-k - 1] * size)
    return bufs, index, layers, pages, page, cb, sb, _I64x8(*st)


def kv_pages_fork(cache, page_table, lengths, parents=None, new_tokens=None, *,
                  return_overfull: bool = False):
    """One step of a batch's pages, in every layer of the pool: row i of the
    new batch continues sequence parents[i] (itself without parents; -1 starts
    empty) and gets pages for new_tokens[i] more tokens. Returns (page_table
    [rows,M], lengths [rows] with the new tokens, missing [1]).

    A row has room for M * page_size tokens, and its length stops there: were
    more of them appended, they would land on tokens that are there already, of
    other rows too. So a row must have the room. PagedKVCache sees to that; who
    does not know the lengths on the host asks for `overfull` [1] with
    return_overfull (a fourth result): the number of rows that have not, on the
    device, to be read like `missing` before anything is appended.

    Pages that no new row holds are free: dropping a sequence frees its own,
    and sequences may share all pages of a prefix. Free pages go in ascending
    order to the rows in order. The partly filled last page of a row that gets
    tokens becomes its own: where another row holds it too the row gets a copy
    (the first of its writers keeps it where all its holders are writers).
    `missing` counts the pages that the pool was short of; when it is not 0
    their entries are -1 and nothing was copied, so the old table and lengths
    still stand."""
    op = "kv_pages_fork"
    bufs, index, layers, pages, page, cb, sb, st = _pool(op, cache)
    b, width = _check_rows(op, index, page_table, lengths)
    rows = b
    if parents is not None:
        rows = parents.shape[0] if parents.ndim == 1 else -1
        _check_ints(op, index, "parents", parents, (rows,))
    if new_tokens is not None:
        _check_ints(op, index, "new_tokens", new_tokens, (rows,))
    _need_gpu(op, index)
    if rows == b:
        table = torch.empty_like(page_table, memory_format=_CONTIGUOUS)
        after = torch.empty_like(lengths)
    else:
        table, after = page_table.new_empty((rows, width)), lengths.new_empty(rows)
    missing = lengths.new_empty(1)
    need = _lib.lib().sparkq_kv_pages_workspace_bytes(rows, pages)
    ws = cache[0].new_empty(need)  # (int8: bytes)
    _lib.launch("sparkq_kv_pages_fork", index, *bufs, page_table.data_ptr(), lengths.data_ptr(),
                _ptr(parents), _ptr(new_tokens), page_table.stride(0), table.data_ptr(),
                after.data_ptr(), missing.data_ptr(), st, b, rows, width, pages, layers, page, cb,
                sb, ws.data_ptr(), need)
    if return_overfull:
        return table, after, missing, ws[4:8].view(torch.int32)
    return table, after, missing


def kv_pages_compact(cache, page_table, lengths):
    """Move the pages in use to the front of the pool, in every layer: with U
    of them, those numbered U or higher go, in order, to the free numbers below
    U. Returns (page_table [B,M], used [1] = U)."""
    op = "kv_pages_compact"
    bufs, index, layers, pages, page, cb, sb, st = _pool(op, cache)
    b, width = _check_rows(op, index, page_table, lengths)
    _need_gpu(op, index)
    table = torch.empty_like(page_table, memory_format=_CONTIGUOUS)
    used = lengths.new_empty(1)
    need = _lib.lib().sparkq_kv_pages_workspace_bytes(b, pages)
    ws = cache[0].new_empty(need)  # (int8: bytes)
    _lib.launch("sparkq_kv_pages_compact", index, *bufs, page_table.data_ptr(), lengths.data_ptr(),
                page_table.stride(0), table.data_ptr(), used.data_ptr(), st, b, width, pages,
                layers, page, cb, sb, ws.data_ptr(), need)
    return table, used


def kv_pages_evict(cache, keep, page_table, lengths, *, mass=None):
    """Sequences of more than `count` tokens keep `count` of them: those that keep
    [layers,B,Hkv,count] int32 (of one layer's cache [B,Hkv,count]) lists in ascending
    order for each layer and KV head, as select_top(mass, count, lengths=lengths)
    returns them. They move to the front of the sequence's pages, in their order, and
    their mass ([layers,B,Hkv,M*page_size] float32) with them. Returns (page_table
    [B,M], lengths [B], missing [1]).

    Shorter sequences stay as they are. A page that is written and that another
    sequence holds too is replaced by a free one, in ascending order to the sequences
    in order, as kv_pages_fork deals them; the rest are written in place. `missing`
    counts the pages that the pool was short of; when it is not 0 nothing was moved,
    and table and lengths are the old ones. An entry i of keep that is below i, or not
    below the length, stands for token i. Positions of tokens in a cache are then no
    longer those of the text, which matters to who rotates later tokens (keys are
    rotated before they are appended), and bounds of written pages have to be taken
    again."""
    op = "kv_pages_evict"
    bufs, index, layers, pages, page, cb, _, st = _pool(op, cache)
    hkv, d = cache[0].shape[-3], cache[0].shape[-1]
    b, width = _check_rows(op, index, page_table, lengths)
    lead = (layers,) if cache[0].ndim == 5 else ()
    if not isinstance(keep, _T) or not keep.ndim or not keep.shape[-1]:
        raise ValueError(f"{op}: keep must be an int32 tensor {[*lead, b, hkv]} + [count]")
    count = keep.shape[-1]
    _check_ints(op, index, "keep", keep, (*lead, b, hkv, count))
    mst = None
    if mass is not None:
        _check_mass(op, mass, index, (*lead, b, hkv, width * page))
        mst = _I64x3(*(mass.stride() if lead else (0, *mass.stride()))[:3])
    _need_gpu(op, index)
    keep = keep.contiguous()
    table = torch.empty_like(page_table, memory_format=_CONTIGUOUS)
    after, missing = torch.empty_like(lengths), lengths.new_empty(1)
    need = _lib.lib().sparkq_kv_pages_workspace_bytes(b, pages)
    ws = cache[0].new_empty(need)  # (int8: bytes)
    _lib.launch("sparkq_kv_pages_evict", index, *bufs, keep.data_ptr(), _ptr(mass),
                page_table.data_ptr(), lengths.data_ptr(), page_table.stride(0), table.data_ptr(),
                after.data_ptr(), missing.data_ptr(), st, mst, b, hkv, d, count, width, pages,
                layers, page, ws.data_ptr(), need)
    return table, after, missing


def _compact_bounds(bounds, page_table, lengths, page_size):
    """Moves the bounds [layers,pages,Hkv,2,D] of pages as kv_pages_compact moves these: a
    page's bounds in four pieces, in the place of its codes and scales."""
    layers, pages, hkv, _, d = bounds.shape
    index, (b, width) = bounds.get_device(), page_table.shape
    piece = hkv * d  # bytes: a quarter of a page's
    table, used = torch.empty_like(page_table), lengths.new_empty(1)
    need = _lib.lib().sparkq_kv_pages_workspace_bytes(b, pages)
    ws = bounds.new_empty(need, dtype=torch.int8)
    _lib.launch("sparkq_kv_pages_compact", index, *(bounds.data_ptr() + i * piece for i in range(4)),
                page_table.data_ptr(), lengths.data_ptr(), page_table.stride(0), table.data_ptr(),
                used.data_ptr(), _I64x8(*(4 * piece * pages, 4 * piece) * 4), b, width, pages, layers,
                page_size, piece, piece, ws.data_ptr(), need)


class PagedKVCache:
    """A pool of pages for the layers of a model, and the batch that holds
    them: `pages` pages of `page_size` tokens, at most `max_pages` of them to a
    sequence. A step is

        starts = cache.step(new_tokens, parents)     # pages for the new tokens
        for each layer l:                            # positions: lengths - n .. lengths - 1
            cache.append(l, keys, values)            # packed rows [T,Hkv,D]
            out = cache.attend(l, queries, scale=...)

    and compact() moves the pages in use to the front of the pool.

    No row may hold more than max_pages * page_size tokens. The host counts each
    row's: a step that would exceed it is short of pages like one that the pool
    has none for (`missing`), and until undo() has taken it back the cache refuses
    to append, attend, compact or step. `lengths` may be lowered in place (tokens
    that are taken back) or set, not raised in place.

    With bounds=True append() keeps the bounds of each page's keys, and

        out = cache.attend_pages(l, queries, scale=..., count=32)

    attends the `count` pages of each KV head that score highest instead of all. With
    mass=True attend(), called once for a step and layer, adds up the attention weight
    that each token gathers, and

        cache.evict(count)                           # between steps

    leaves each row the `count` tokens that gathered most. (After it lengths are no
    longer positions: count these apart.) What a token added to the others' weight stays
    there when it is taken back by lowering `lengths`. A step of drafted tokens is
    therefore attended by paged_quantized_sdpa(..., return_lse=True), and paged_kv_mass
    adds the weights of the accepted rows to mass[l] (with starts of their own and the
    lowered lengths) once it is known which these are."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, *,
                 page_size: int = 64, max_pages: int = 128, batch: int = 0, device="cuda",
                 bounds: bool = False, mass: bool = False):
        if min(layers, pages, kv_heads, max_pages) < 1 or batch < 0:
            raise ValueError("layers, pages, kv_heads and max_pages must be positive")
        if head_dim not in (64, 128, 256):
            raise ValueError("head_dim must be 64, 128 or 256")
        if page_size not in (16, 32, 64, 128, 256, 512, 1024):
            raise ValueError("page_size must be a power of two from 16 to 1024")
        shape = (layers, pages, kv_heads, page_size)
        self.cache = tuple(
            torch.zeros((*shape, head_dim), dtype=torch.int8, device=device) if codes else
            torch.zeros(shape, dtype=torch.float16, device=device) for codes in (1, 0, 1, 0))
        self.page_size, self.max_pages = page_size, max_pages
        dev = self.cache[0].device
        self.bounds = torch.zeros((layers, pages, kv_heads, 2, head_dim), dtype=torch.bfloat16,
                                  device=dev) if bounds else None
        self.mass = torch.zeros((layers, batch, kv_heads, max_pages * page_size),
                                device=dev) if mass else None
        self.page_table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros((batch,), dtype=torch.int32, device=dev)
        self.starts = torch.zeros((batch + 1,), dtype=torch.int32, device=dev)
        self.missing = torch.zeros((1,), dtype=torch.int32, device=dev)
        self.max_new = 0
        self._last, self._full, self._counts = None, False, [0] * batch

    @property
    def lengths(self):
        """Tokens of each row, the new ones included (int32, on the device)."""
        return self._lengths

    @lengths.setter
    def lengths(self, value):
        self._lengths, self._counts = value, None  # (counted when a step needs it)

    def _after(self, new_tokens, parents):
        """Tokens of each row after a step. Lengths are read from the device only
        where they are not known, or may have been lowered and that matters."""
        rows, read = self.page_table.shape[0], self._counts is None
        while True:
            counts = self._lengths.tolist() if read else self._counts
            before = counts if parents is None else \
                [counts[p] if 0 <= p < rows else 0 for p in parents]
            after = [n + k for n, k in zip(before, new_tokens)]
            if read or max(after, default=0) <= self.max_pages * self.page_size:
                return after
            read = True

    def _ready(self):
        if self._full:
            raise ValueError("the last step would fill rows past max_pages * page_size tokens: "
                             "take it back with undo()")

    def step(self, new_tokens, parents=None):
        """Start a step: the batch's rows continue `parents` (itself without)
        and get new_tokens[i] tokens each (a list of Python ints). Returns the
        packed rows' starts. Enqueued without waiting for the device, but not in a
        graph's capture: its numbers come from the host. `missing` then counts the
        pages that the pool, or rows of max_pages, were short of (on the device): a
        caller that may run short reads it before the step's first append, and
        takes the step back with undo()."""
        self._ready()
        dev = self.page_table.device
        if dev.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("a step takes its numbers from the host and cannot be captured")
        new_tokens = [int(n) for n in new_tokens]
        if any(n < 0 for n in new_tokens):
            raise ValueError("new_tokens must not be negative")
        rows = self.page_table.shape[0] if parents is None else len(parents)
        if len(new_tokens) != rows:
            raise ValueError(f"new_tokens must have an entry for each of the {rows} rows")
        ends = [0]
        for n in new_tokens:
            ends.append(ends[-1] + n)
        parents = None if parents is None else [int(p) for p in parents]
        after = self._after(new_tokens, parents)
        host = new_tokens + ends + (parents or [])
        if dev.type == "cuda":
            # from pinned memory, which torch keeps until the copy is done: a copy from
            # pageable memory would wait for all that the stream has still to do
            ints = torch.tensor(host, dtype=torch.int32, pin_memory=True).to(dev, non_blocking=True)
        else:
            ints = torch.tensor(host, dtype=torch.int32, device=dev)
        if parents is not None:
            parents = ints[2 * rows + 1:]
        last = (self.page_table, self._lengths, self._counts, self.starts, self.max_new, self.mass)
        short = sum(max(0, -(-n // self.page_size) - self.max_pages) for n in after)
        if short:  # no page is touched: the tokens without a place would fall on others
            room = self.max_pages * self.page_size
            self.page_table = self.page_table.new_full((rows, self.max_pages), -1)
            self._lengths = ints.new_tensor([min(n, room) for n in after])
            self.missing, self._full = self.missing.new_full((1,), short), True
        else:
            # (first what may fail for want of memory: the fork cannot be taken back)
            mass = self.mass if self.mass is None or parents is None else self._mass_of(parents)
            self.page_table, self._lengths, self.missing = kv_pages_fork(
                self.cache, self.page_table, self._lengths, parents, ints[:rows])
            self.mass = mass
        self._last, self._counts = last, after
        self.starts, self.max_new = ints[rows:2 * rows + 1], max(new_tokens, default=0)
        return self.starts

    def _mass_of(self, parents):
        """Mass of rows that continue `parents`; what starts empty has only new tokens, which
        start from 0."""
        layers, rows, *shape = self.mass.shape
        if rows == 0:
            return self.mass.new_zeros((layers, parents.shape[0], *shape))
        return self.mass.index_select(1, parents.clamp(0, rows - 1))

    def undo(self):
        """Take back a step that was short of pages, before anything of it was
        appended: the batch is what it was, and a smaller step can follow. Reads
        `missing`. A step that was not short may have copied pages over those of
        sequences that it dropped, and stands."""
        if self._last is None:
            raise ValueError("there is no step to take back")
        if self.missing.item() == 0:
            raise ValueError("the last step was not short of pages")
        (self.page_table, self._lengths, self._counts, self.starts, self.max_new,
         self.mass) = self._last
        self._last, self._full = None, False

    def layer(self, index: int):
        return tuple(t[index] for t in self.cache)

    def append(self, index: int, keys, values):
        self._ready()
        paged_kv_append(keys, values, self.layer(index), self.page_table, self.starts,
                        self.lengths)
        if self.bounds is not None:
            paged_key_bounds(self.layer(index), self.bounds[index], self.page_table, self.starts,
                             self.lengths, max_new=max(self.max_new, 1))
        self._last = None  # what is appended cannot be taken back

    def attend(self, index: int, queries, *, scale, mask="causal", out_dtype=None, out=None):
        self._ready()
        batch = self.page_table, self.starts, self.lengths
        kw = {"scale": scale, "max_new": max(self.max_new, 1), "mask": mask}
        if self.mass is None:
            return paged_quantized_sdpa(queries, self.layer(index), *batch, out_dtype=out_dtype,
                                        out=out, **kw)
        out, lse = paged_quantized_sdpa(queries, self.layer(index), *batch, out_dtype=out_dtype,
                                        out=out, return_lse=True, **kw)
        paged_kv_mass(queries, lse, self.layer(index), self.mass[index], *batch, **kw)
        return out

    def attend_pages(self, index: int, queries, *, scale, count: int, first: int = 1, last: int = 2,
                     mask="causal", out_dtype=None, out=None):
        """Attention over `count` pages of each KV head for each new token: the first
        `first` and last `last` that it sees, and those whose bounds allow the largest
        logits."""
        self._ready()
        if self.bounds is None:
            raise ValueError("attend_pages needs a cache with bounds=True")
        if self.mass is not None:
            raise ValueError("a cache with mass=True attends all tokens: attention over selected "
                             "pages does not say what the others gather")
        batch = self.page_table, self.starts, self.lengths
        kw = {"scale": scale, "max_new": max(self.max_new, 1), "mask": mask}
        scores, seen = paged_page_scores(queries, self.bounds[index], *batch,
                                         page_size=self.page_size, **kw)
        pages = select_top(scores, count, lengths=seen, first=first, last=last)
        return paged_sparse_sdpa(queries, self.layer(index), pages, *batch, out_dtype=out_dtype,
                                 out=out, **kw)

    def evict(self, count: int, *, first: int = 0, last: int = 0):
        """Rows of more than `count` tokens keep `count` of them, in each layer and KV head
        its own: the first `first`, the last `last`, and those of the rest that gathered
        the most attention weight. To be called between steps, when every layer has appended
        and attended the last one's tokens, which are then old ones: refused before the
        first append of a step with new tokens. Returns `missing` (on the device, like
        step's): pages that the pool was short of, as what is written must not be shared;
        when it is not 0 all is as it was."""
        self._ready()
        if self.mass is None:
            raise ValueError("evict needs a cache with mass=True")
        if self._last is not None and self.max_new:
            raise ValueError("evict comes between steps, and the last one's tokens are not in the "
                             "cache: append and attend them, or take a step that was short of "
                             "pages back with undo()")
        keep = select_top(self.mass, count, lengths=self._lengths, first=first, last=last)
        before = self._lengths
        self.page_table, self._lengths, self.missing = kv_pages_evict(
            self.cache, keep, self.page_table, before, mass=self.mass)
        self._last = None  # (the host's counts stay: they are no less than the tokens)
        self.starts, self.max_new = torch.zeros_like(self.starts), 0
        if self.bounds is not None and self.page_table.shape[0]:
            # all tokens of the rows that changed as new ones
            ends = torch.where(self._lengths < before, self._lengths, 0).cumsum(0, dtype=torch.int32)
            starts = torch.cat([ends.new_zeros(1), ends])
            for index in range(self.cache[0].shape[0]):
                paged_key_bounds(self.layer(index), self.bounds[index], self.page_table, starts,
                                 self._lengths, max_new=count)
        return self.missing

    def compact(self):
        """Returns the number of pages in use (on the device): the pages from
        it on are free."""
        self._ready()
        self._last = None
        before = self.page_table
        self.page_table, used = kv_pages_compact(self.cache, before, self.lengths)
        if self.bounds is not None:
            _compact_bounds(self.bounds, before, self.lengths, self.page_size)
        return used
