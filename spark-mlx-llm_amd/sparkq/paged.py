"""Many sequences over one paged INT8 KV cache (no counterpart in the
reference, which serves one request at a time over contiguous caches).

A cache is the tuple (k_codes, k_scales, v_codes, v_scales) of symmetric int8
codes [pages,Hkv,page_size,D] and fp16 scales [pages,Hkv,page_size], the "s8"
format of kv_append and int8_quantized_sdpa in pages; a pool of several layers
has a leading layer axis. A batch is described by three int32 tensors on the
device that no call reads back:

  page_table [B,M]  the pages of each sequence; an entry outside the pool is
                    no page
  lengths    [B]    tokens of each sequence, the new ones included
  starts     [B+1]  the packed rows of each sequence's new tokens are
                    starts[b] .. starts[b+1] - 1, its last token the last one

Like every sparkq operator these enqueue on the current stream of the tensors'
device and return without synchronising. Each call's scratch comes from torch's
allocator, so threads on one stream and captured graphs share none.
"""

from __future__ import annotations

import ctypes
import math

import torch

from . import _lib
from .ext import _HALF, _REAL, _out_buffer, _ptr, _require_device

__all__ = ["PagedKVCache", "kv_pages_compact", "kv_pages_fork", "paged_kv_append",
           "paged_quantized_sdpa"]


def _check_cache(op, cache, ndim):
    """(pages, Hkv, page_size, D) of a cache with `ndim` axes in its codes."""
    if len(cache) != 4 or any(not isinstance(t, torch.Tensor) for t in cache):
        raise ValueError(f"{op}: the cache is (k_codes, k_scales, v_codes, v_scales)")
    kc, ks, vc, vs = cache
    if (kc.ndim != ndim or kc.dtype != torch.int8 or vc.dtype != torch.int8
            or ks.dtype != torch.float16 or vs.dtype != torch.float16
            or vc.shape != kc.shape or ks.shape != kc.shape[:-1] or vs.shape != ks.shape):
        raise ValueError(f"{op}: the cache holds int8 codes [pages,Hkv,page_size,D] and fp16 "
                         "scales [pages,Hkv,page_size] of keys and of values")
    dev = kc.device
    if ks.device != dev or vc.device != dev or vs.device != dev:
        raise ValueError(f"{op}: the cache's tensors must live on one device")
    return kc.shape[-4:]


def _check_device(op, cache, *tensors):
    """On the GPU, all of them on the cache's."""
    _require_device(op, cache[0], *tensors)
    if any(t.device != cache[0].device for t in tensors):
        raise ValueError(f"{op}: every tensor must live on the cache's device")


def _check_ints(op, device, **tensors):
    for name, (t, shape) in tensors.items():
        if t.dtype != torch.int32 or t.shape != shape or (t.ndim and t.stride(-1) != 1
                                                          and t.shape[-1] > 1):
            raise ValueError(f"{op}: {name} must be an int32 tensor of shape {list(shape)}, its "
                             "last axis contiguous")
        if t.device != device:
            raise ValueError(f"{op}: {name} must live on the cache's device")


def _batch(op, cache, page_table, starts, lengths):
    if page_table.ndim != 2 or lengths.ndim != 1:
        raise ValueError(f"{op}: expected page_table [B,M], lengths [B] and starts [B+1]")
    b, width = page_table.shape
    if width < 1:
        raise ValueError(f"{op}: page_table has no columns")
    _check_ints(op, cache[0].device, page_table=(page_table, (b, width)),
                lengths=(lengths, (b,)), starts=(starts, (b + 1,)))
    return b, width


def _strides(cache):
    kc, ks, vc, vs = cache
    if kc.stride(-1) != 1 or vc.stride(-1) != 1:
        raise ValueError("the cache's innermost axes must be contiguous")
    return (ctypes.c_int64 * 12)(*kc.stride()[:3], *ks.stride(), *vc.stride()[:3], *vs.stride())


def _rows16(t):
    """t with rows that 16-byte loads can read: itself, or a copy."""
    n = 16 // t.element_size()
    st = t.stride()
    if st[2] == 1 and st[0] % n == 0 and st[1] % n == 0 and t.data_ptr() % 16 == 0:
        return t
    return t.contiguous() if not t.is_contiguous() else t.clone()


def paged_kv_append(keys, values, cache, page_table, starts, lengths):
    """Quantize a batch's new tokens into their pages, in place: keys and
    values [T,Hkv,D] (float16, bfloat16 or float32; views of a packed
    projection are read in place), one layer's cache. The formula is
    kv_quantize_s8's. Rows that fall to no sequence, tokens before position 0
    and tokens without a page are skipped. Sequences that append must not share
    the page they append to: kv_pages_fork gives each its own."""
    op = "paged_kv_append"
    pages, hkv, page, d = _check_cache(op, cache, 4)
    if keys.ndim != 3 or keys.shape[1:] != (hkv, d) or values.shape != keys.shape:
        raise ValueError(f"{op}: keys and values must be [T,{hkv},{d}] like the cache")
    if keys.dtype not in _REAL or values.dtype != keys.dtype:
        raise ValueError(f"{op}: keys and values must be float16, bfloat16 or float32, both alike")
    b, width = _batch(op, cache, page_table, starts, lengths)
    _check_device(op, cache, keys, values)
    strides = _strides(cache)
    keys, values = _rows16(keys), _rows16(values)
    xst = (ctypes.c_int64 * 4)(*keys.stride()[:2], *values.stride()[:2])
    kc, ks, vc, vs = cache
    _lib.call("sparkq_paged_kv_append", _ptr(keys), _ptr(values), _ptr(kc), _ptr(ks), _ptr(vc),
              _ptr(vs), _ptr(page_table), _ptr(starts), _ptr(lengths), keys.shape[0], b, hkv, d,
              pages, width, page_table.stride(0), page, _lib.dtype_code(keys.dtype), xst, strides,
              _lib.stream_handle(kc.device), device=kc.device)


def paged_quantized_sdpa(queries, cache, page_table, starts, lengths, *, scale, max_new: int,
                         mask="causal", out_dtype=None, out=None):
    """Attention of a batch's new tokens over their pages: queries [T,Hq,D]
    (float16 or bfloat16) -> [T,Hq,D]. With mask="causal" row i of a
    sequence's n new tokens sees its tokens 0 .. length - n + i, with None all
    of them; tokens without a page are hidden, and a row that sees nothing is
    zero. max_new is the most new tokens that a sequence has (1: a decode
    step). Rows that fall to no sequence, or to more than max_new of one, are
    left as they are in `out`, and hold anything in a new tensor."""
    op = "paged_quantized_sdpa"
    pages, hkv, page, d = _check_cache(op, cache, 4)
    if queries.ndim != 3 or queries.shape[2] != d or queries.shape[1] < 1 \
            or queries.shape[1] % hkv:
        raise ValueError(f"{op}: queries must be [T,Hq,{d}] with Hq divisible by {hkv}")
    if queries.dtype not in _HALF:
        raise ValueError(f"{op} requires float16 or bfloat16 queries")
    if mask not in (None, "causal"):
        raise ValueError(f"{op} takes mask=None or mask='causal'")
    if not isinstance(scale, (float, int)) or not math.isfinite(scale):
        raise ValueError("scale must be a finite Python number")
    if type(max_new) is not int or max_new < 1:
        raise ValueError(f"{op}: max_new must be a positive Python int")
    out_dtype = queries.dtype if out_dtype is None else out_dtype
    if out_dtype not in (queries.dtype, torch.float32):
        raise ValueError("out_dtype must be the query dtype or torch.float32")
    b, width = _batch(op, cache, page_table, starts, lengths)
    _check_device(op, cache, queries)
    strides = _strides(cache)
    t, heads = queries.shape[:2]
    q = _rows16(queries)
    y = _out_buffer(out, (t, heads, d), out_dtype, queries.device)
    lib = _lib.lib()
    need = lib.sparkq_paged_sdpa_workspace_bytes(t, b, heads, hkv, d, max_new, width * page)
    ws = _lib.scratch(q.device, need)
    qst = (ctypes.c_int64 * 2)(*q.stride()[:2])
    kc, ks, vc, vs = cache
    code = _lib.dtype_code
    _lib.call("sparkq_paged_sdpa", _ptr(q), _ptr(kc), _ptr(ks), _ptr(vc), _ptr(vs),
              _ptr(page_table), _ptr(starts), _ptr(lengths), _ptr(y), t, b, heads, hkv, d, pages,
              width, page_table.stride(0), page, max_new, 1 if mask is not None else 0,
              code(q.dtype), code(out_dtype), float(scale), qst, strides, _ptr(ws), need,
              _lib.stream_handle(q.device), device=q.device)
    return y


def _pool(op, cache):
    """(layers, pages, page_size, code and scale bytes of a page, strides) of a
    pool [layers,pages,...] or of one layer [pages,...]."""
    ndim = cache[0].ndim if len(cache) == 4 and isinstance(cache[0], torch.Tensor) else 0
    pages, hkv, page, d = _check_cache(op, cache, 5 if ndim == 5 else 4)
    kc, ks, vc, vs = cache
    st = []
    for t in (kc, vc, ks, vs):
        e, s = t.element_size(), t.stride()
        inner = (page * d, d, 1) if t.dtype == torch.int8 else (page, 1)
        if s[-len(inner):] != inner:
            raise ValueError(f"{op}: a page must be contiguous in every tensor of the cache")
        lead = s[:-len(inner)]
        st += [lead[0] * e if ndim == 5 else 0, lead[-1] * e]
    layers = kc.shape[0] if ndim == 5 else 1
    if layers < 1:
        raise ValueError(f"{op}: the pool has no layers")
    return layers, pages, page, hkv * page * d, hkv * page * 2, (ctypes.c_int64 * 8)(*st)


def kv_pages_fork(cache, page_table, lengths, parents=None, new_tokens=None):
    """One step of a batch's pages, in every layer of the pool: row i of the
    new batch continues sequence parents[i] (itself without parents; -1 starts
    empty) and gets pages for new_tokens[i] more tokens. Returns (page_table
    [rows,M], lengths [rows] with the new tokens, missing [1]).

    Pages that no new row holds are free: dropping a sequence frees its own,
    and sequences may share all pages of a prefix. Free pages go in ascending
    order to the rows in order. The partly filled last page of a row that gets
    tokens becomes its own: where another row holds it too the row gets a copy
    (the first of its writers keeps it where all its holders are writers).
    `missing` counts the pages that the pool was short of; when it is not 0
    their entries are -1 and nothing was copied, so the old table and lengths
    still stand."""
    op = "kv_pages_fork"
    layers, pages, page, cb, sb, st = _pool(op, cache)
    if page_table.ndim != 2 or page_table.shape[1] < 1 or lengths.ndim != 1:
        raise ValueError(f"{op}: expected page_table [B,M] and lengths [B]")
    b, width = page_table.shape
    rows = b if parents is None else parents.shape[0] if parents.ndim == 1 else -1
    checks = {"page_table": (page_table, (b, width)), "lengths": (lengths, (b,))}
    if parents is not None:
        checks["parents"] = (parents, (rows,))
    if new_tokens is not None:
        checks["new_tokens"] = (new_tokens, (rows,))
    kc, ks, vc, vs = cache
    dev = kc.device
    _check_ints(op, dev, **checks)
    _check_device(op, cache)
    table = torch.empty((rows, width), dtype=torch.int32, device=dev)
    after = torch.empty((rows,), dtype=torch.int32, device=dev)
    missing = torch.empty((1,), dtype=torch.int32, device=dev)
    need = _lib.lib().sparkq_kv_pages_workspace_bytes(rows, pages)
    ws = _lib.scratch(dev, need)
    _lib.call("sparkq_kv_pages_fork", _ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs), _ptr(page_table),
              _ptr(lengths), _ptr(parents), _ptr(new_tokens), page_table.stride(0), _ptr(table),
              _ptr(after), _ptr(missing), st, b, rows, width, pages, layers, page, cb, sb,
              _ptr(ws), need, _lib.stream_handle(dev), device=dev)
    return table, after, missing


def kv_pages_compact(cache, page_table, lengths):
    """Move the pages in use to the front of the pool, in every layer: with U
    of them, those numbered U or higher go, in order, to the free numbers below
    U. Returns (page_table [B,M], used [1] = U)."""
    op = "kv_pages_compact"
    layers, pages, page, cb, sb, st = _pool(op, cache)
    if page_table.ndim != 2 or page_table.shape[1] < 1 or lengths.ndim != 1:
        raise ValueError(f"{op}: expected page_table [B,M] and lengths [B]")
    b, width = page_table.shape
    kc, ks, vc, vs = cache
    dev = kc.device
    _check_ints(op, dev, page_table=(page_table, (b, width)), lengths=(lengths, (b,)))
    _check_device(op, cache)
    table = torch.empty((b, width), dtype=torch.int32, device=dev)
    used = torch.empty((1,), dtype=torch.int32, device=dev)
    need = _lib.lib().sparkq_kv_pages_workspace_bytes(b, pages)
    ws = _lib.scratch(dev, need)
    _lib.call("sparkq_kv_pages_compact", _ptr(kc), _ptr(vc), _ptr(ks), _ptr(vs), _ptr(page_table),
              _ptr(lengths), page_table.stride(0), _ptr(table), _ptr(used), st, b, width, pages,
              layers, page, cb, sb, _ptr(ws), need, _lib.stream_handle(dev), device=dev)
    return table, used


class PagedKVCache:
    """A pool of pages for the layers of a model, and the batch that holds
    them: `pages` pages of `page_size` tokens, at most `max_pages` of them to a
    sequence. A step is

        starts = cache.step(new_tokens, parents)     # pages for the new tokens
        for each layer l:
            cache.append(l, keys, values)            # packed rows [T,Hkv,D]
            out = cache.attend(l, queries, scale=...)

    and compact() moves the pages in use to the front of the pool."""

    def __init__(self, layers: int, pages: int, kv_heads: int, head_dim: int, *,
                 page_size: int = 64, max_pages: int = 128, batch: int = 0, device="cuda"):
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
        self.page_table = torch.full((batch, max_pages), -1, dtype=torch.int32, device=dev)
        self.lengths = torch.zeros((batch,), dtype=torch.int32, device=dev)
        self.starts = torch.zeros((batch + 1,), dtype=torch.int32, device=dev)
        self.missing = torch.zeros((1,), dtype=torch.int32, device=dev)
        self.max_new = 0

    def step(self, new_tokens, parents=None):
        """Start a step: the batch's rows continue `parents` (itself without)
        and get new_tokens[i] tokens each (a list of Python ints). Returns the
        packed rows' starts. `missing` then counts the pages that the pool was
        short of (on the device)."""
        new_tokens = [int(n) for n in new_tokens]
        if any(n < 0 for n in new_tokens):
            raise ValueError("new_tokens must not be negative")
        rows = self.page_table.shape[0] if parents is None else len(parents)
        if len(new_tokens) != rows:
            raise ValueError(f"new_tokens must have an entry for each of the {rows} rows")
        ends = [0]
        for n in new_tokens:
            ends.append(ends[-1] + n)
        dev = self.page_table.device
        host = new_tokens + ends + ([] if parents is None else [int(p) for p in parents])
        ints = torch.tensor(host, dtype=torch.int32, device=dev)
        if parents is not None:
            parents = ints[2 * rows + 1:]
        self.page_table, self.lengths, self.missing = kv_pages_fork(
            self.cache, self.page_table, self.lengths, parents, ints[:rows])
        self.starts, self.max_new = ints[rows:2 * rows + 1], max(new_tokens, default=0)
        return self.starts

    def layer(self, index: int):
        return tuple(t[index] for t in self.cache)

    def append(self, index: int, keys, values):
        paged_kv_append(keys, values, self.layer(index), self.page_table, self.starts,
                        self.lengths)

    def attend(self, index: int, queries, *, scale, mask="causal", out_dtype=None, out=None):
        return paged_quantized_sdpa(queries, self.layer(index), self.page_table, self.starts,
                                    self.lengths, scale=scale, max_new=max(self.max_new, 1),
                                    mask=mask, out_dtype=out_dtype, out=out)

    def compact(self):
        """Returns the number of pages in use (on the device): the pages from
        it on are free."""
        self.page_table, used = kv_pages_compact(self.cache, self.page_table, self.lengths)
        return used
