"""Operators of long contexts over a paged INT8 KV cache, as cases that can be
timed: the bounds of each page's keys, the scores of pages for a query, the
selection of the largest scores, the attention over selected pages, the
attention weight that each cached token gathers, and the eviction of tokens.

Where `own` is false run() computes an operator's plain form in elementary
torch operations; where it is true it makes the framework's calls. exact()
restates the operators in float64.

Cache: (k_codes [layers,P,Hkv,page,D] int8, k_scales [layers,P,Hkv,page] fp16,
v_codes, v_scales); one layer of it for all but the eviction. A key is code *
scale, exact in fp32. Bounds [P,Hkv,2,D] bf16: per page and channel the least
key rounded down, and the largest rounded up.
"""

import math
import os
import random
import sys

import numpy as np
import torch

own = False

_DEV = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# query heads, KV heads, head dim
_HEADS = {"32x8x128": (32, 8, 128), "16x4x256": (16, 4, 256), "20x4x128": (20, 4, 128),
          "16x2x64": (16, 2, 64)}
_FIRST, _LAST = 1, 2  # pages that every query attends: the first, and the last two


def _sparkq():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "spark-mlx-llm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import sparkq

    return sparkq


def listed():
    return [
        # one decoded token of each of 16 sequences: the pages that they lie in
        {"name": "bounds_16", "kind": "bounds", "b": 16, "new": 1, "n": 2000, "page": 64,
         "heads": "32x8x128", "mix": 1},
        # three prompt chunks of odd lengths, larger heads, small pages
        {"name": "bounds_3x2000", "kind": "bounds", "b": 3, "new": 2000, "n": 4000, "page": 16,
         "heads": "16x4x256", "mix": 2},
        # the pages of 64 sequences of up to 32768 tokens, for a decode step
        {"name": "scores_64x32768", "kind": "scores", "b": 64, "new": 1, "n": 32768, "page": 64,
         "heads": "32x8x128", "mix": 3, "dtype": "bf16"},
        # for each token of a prompt's chunk
        {"name": "scores_512x16384", "kind": "scores", "b": 1, "new": 512, "n": 16384, "page": 32,
         "heads": "20x4x128", "mix": 0, "dtype": "f16"},
        # 32 pages for each KV head of 16 decoded tokens: latency
        {"name": "select_16x8x512", "kind": "select", "layers": 0, "b": 16, "h": 8, "n": 512,
         "count": 32, "first": 1, "last": 2, "mix": 4},
        # the tokens that 16 sequences keep in 8 layers
        {"name": "select_8x16x8x8192", "kind": "select", "layers": 8, "b": 16, "h": 8, "n": 8192,
         "count": 2048, "first": 4, "last": 256, "mix": 5},
        # one decoded token over 32 pages of a long sequence: latency
        {"name": "sparse_1x32768", "kind": "sparse", "b": 1, "new": 1, "n": 32768, "page": 64,
         "count": 32, "heads": "32x8x128", "mix": 0, "dtype": "bf16"},
        # a serving batch's decode step, odd counts of small pages, larger heads
        {"name": "sparse_64x16384", "kind": "sparse", "b": 64, "new": 1, "n": 16384, "page": 32,
         "count": 77, "heads": "16x4x256", "mix": 6, "dtype": "f16"},
        # the weights of a serving batch's decode step
        {"name": "mass_64x8192", "kind": "mass", "b": 64, "new": 1, "n": 8192, "page": 64,
         "heads": "32x8x128", "mix": 7, "dtype": "bf16"},
        # of a prompt's last chunk
        {"name": "mass_2048x8192", "kind": "mass", "b": 1, "new": 2048, "n": 8192, "page": 64,
         "heads": "32x8x128", "mix": 0, "dtype": "bf16"},
        # a few short sequences, one continued twice, reduced in a small model
        {"name": "evict_4", "kind": "evict", "b": 4, "n": 900, "page": 32, "count": 500,
         "layers": 2, "heads": "20x4x128", "mix": 8},
        # a batch's long sequences in eight layers
        {"name": "evict_24", "kind": "evict", "b": 24, "n": 6000, "page": 64, "count": 1500,
         "layers": 8, "heads": "32x8x128", "mix": 9},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["bounds", "scores", "select", "sparse", "sparse", "mass", "mass", "evict"])
    heads = rng.choice(sorted(_HEADS))
    mix = rng.randint(10, 9999)
    page = rng.choice([16, 32, 64, 128])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    if kind == "select":
        n = _log(rng, 1, 20000)
        count = _log(rng, 1, n)
        first = rng.randint(0, min(4, count))
        rows = max(1, min(128, 4_000_000 // (8 * n)))
        return {"kind": kind, "layers": rng.choice([0, 1, 4]), "b": rng.randint(1, rows) // 4 + 1,
                "h": rng.choice([1, 2, 4, 8]), "n": n, "count": count, "first": first,
                "last": rng.randint(0, count - first), "mix": mix}
    if kind == "evict":
        count = _log(rng, 10, 1500)
        return {"kind": kind, "b": rng.randint(1, 16), "n": count + _log(rng, 1, 4000), "page": page,
                "count": count, "layers": rng.randint(1, 4), "heads": heads, "mix": mix}
    # decode, the verification of a few drafted tokens, or a chunk
    new = rng.choice([1, 1, rng.randint(2, 8), _log(rng, 9, 500)])
    b = _log(rng, 1, 48) if new <= 8 else rng.randint(1, 3)
    n = new + _log(rng, 8, 12000)
    case = {"kind": kind, "b": b, "new": new, "n": n, "page": page, "heads": heads, "mix": mix}
    if kind == "sparse":
        case["new"] = new = min(new, 64)
        case["count"] = min(_log(rng, _FIRST + _LAST, 64), max(_FIRST + _LAST, 2048 // page))
    if kind != "bounds":
        case["dtype"] = dtype
    return case


# ---------------------------------------------------------------------------
# what a case's batch looks like: from the case alone, so that work() knows it
# ---------------------------------------------------------------------------

def _batch(case):
    """(new tokens, lengths with them) of each sequence. A single sequence has
    exactly the case's sizes. In a batch the first is the longest; with chunks
    (new > 8) every second one decodes a single token; one of eight is idle."""
    rng = random.Random(case["mix"])
    b, new, n = case["b"], case["new"], case["n"]
    news, lens = [new], [n]
    while len(lens) < b:
        i = len(lens)
        k = 1 if new > 8 and i % 2 else (new if new <= 8 else rng.randint(max(1, new // 2), new))
        if i % 8 == 7:
            k = 0
        news.append(k)
        lens.append(max(k, _log(rng, max(1, n // 64), n)))
    return news, lens


def _pages_of(n, page):
    return -(-n // page)


def _touched(case):
    """(pages, tokens in them) that hold a sequence's new tokens, in sum."""
    news, lens = _batch(case)
    pages = tokens = 0
    for k, n in zip(news, lens):
        if k:
            first = (n - k) // case["page"]
            pages += _pages_of(n, case["page"]) - first
            tokens += n - first * case["page"]
    return pages, tokens


def _evicted(case):
    """Lengths, and for each row how many leading pages it shares with the row
    before (every fourth row is a second continuation of that one)."""
    rng = random.Random(case["mix"])
    lens = [case["n"]] + [_log(rng, max(1, case["n"] // 8), case["n"]) for _ in range(case["b"] - 1)]
    shared = [0] * case["b"]
    for i in range(1, case["b"], 4):
        shared[i] = min(lens[i], lens[i - 1]) // case["page"]
    return lens, shared


def _gen(seed):
    return torch.Generator(device=_DEV).manual_seed(int(seed))


def _randn(gen, *shape, dtype=torch.float32, std=1.0):
    return torch.randn(shape, generator=gen, device=_DEV).mul_(std).to(dtype)


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=_DEV)


def _pool(gen, layers, pages, hkv, page, d):
    """A cache in use: codes over the whole range, a scale for each row."""
    out = []
    for _ in range(2):
        codes = torch.empty((layers, pages, hkv, page, d), dtype=torch.int8, device=_DEV)
        codes.view(layers, -1).random_(-127, 128, generator=gen)
        scales = torch.rand((layers, pages, hkv, page), generator=gen, device=_DEV)
        out += [codes, (0.01 + 0.02 * scales).half()]
    return tuple(out)


def _table(gen, counts, pages, width):
    """`counts` pages in random order for each sequence, -1 elsewhere."""
    ids = torch.randperm(pages, generator=gen, device=_DEV)[: sum(counts)].to(torch.int32)
    table = torch.full((len(counts), width), -1, dtype=torch.int32, device=_DEV)
    live = torch.arange(width, device=_DEV)[None] < torch.tensor(counts, device=_DEV)[:, None]
    table[live] = ids
    return table


def prepare(case, seed):
    gen = _gen(seed)
    s = {"kind": case["kind"]}
    {"select": _prepare_select, "evict": _prepare_evict}.get(case["kind"], _prepare_batch)(case, gen, s)
    return s


def _prepare_select(case, gen, s):
    rng = random.Random(case["mix"])
    shape = (case["layers"],) * bool(case["layers"]) + (case["b"], case["h"], case["n"])
    # gathered weights: over many orders of magnitude, and nothing for some
    x = _randn(gen, *shape, std=2.0).exp_()
    x[torch.rand(shape, generator=gen, device=_DEV) < 0.1] = 0
    s["x"] = x
    s["lengths"] = _ints([case["n"]] + [_log(rng, max(1, case["n"] // 4), case["n"])
                                        for _ in range(case["b"] - 1)])
    s["count"], s["first"], s["last"] = case["count"], case["first"], case["last"]


def _prepare_evict(case, gen, s):
    _, hkv, d = _HEADS[case["heads"]]
    page, layers, count = case["page"], case["layers"], case["count"]
    lens, shared = _evicted(case)
    width = _pages_of(case["n"], page)
    # room for what a step of every row asks for, and copies of shared pages
    pages = sum(_pages_of(n, page) for n in lens) + case["b"] * (_pages_of(count, page) + 1)
    s["cache"] = _pool(gen, layers, pages, hkv, page, d)
    s["page"] = page
    s["table"] = _table(gen, [_pages_of(n, page) for n in lens], pages, width)
    for i, k in enumerate(shared):
        s["table"][i, :k] = s["table"][i - 1, :k]
    s["lengths"] = _ints(lens)
    s["mass"] = _randn(gen, layers, len(lens), hkv, width * page, std=2.0).exp_()
    # the heaviest tokens, the first four and the last sixteenth, in order
    at = torch.arange(width * page, device=_DEV)
    n = s["lengths"].long()[:, None, None]
    w = s["mass"].masked_fill((at < 4) | (at >= n - count // 16), math.inf)
    w = w.masked_fill(at >= n, -1.0)
    keep = w.topk(min(count, width * page), -1).indices.sort(-1).values
    keep = torch.where(torch.arange(keep.shape[-1], device=_DEV) < n, keep, -1)
    s["keep"] = keep.int()


def _prepare_batch(case, gen, s):
    hq, hkv, d = _HEADS[case["heads"]]
    kind, page = case["kind"], case["page"]
    news, lens = _batch(case)
    width = _pages_of(case["n"], page)
    counts = [_pages_of(v, page) for v in lens]
    pages, t = sum(counts) + 3, sum(news)
    s["page"], s["new"], s["scale"] = page, max(news), d ** -0.5
    s["table"] = _table(gen, counts, pages, width)
    s["lengths"] = _ints(lens)
    s["starts"] = _ints([0] + torch.tensor(news).cumsum(0).tolist())
    if kind != "scores":
        s["cache"] = tuple(x[0] for x in _pool(gen, 1, pages, hkv, page, d))
    if kind in ("bounds", "scores"):
        # the ranges of a page's keys: around a mean of their own
        mid = _randn(gen, pages, hkv, 1, d)
        half = 0.5 + torch.rand((pages, hkv, 1, d), generator=gen, device=_DEV)
        s["bounds"] = torch.cat([mid - half, mid + half], 2).bfloat16()
    if kind == "bounds":
        return
    s["q"] = _randn(gen, t, hq, d, dtype=_TYPES[case["dtype"]])
    if kind == "sparse":
        s["pages"] = _lists(case, gen, t, hkv, news, lens)
    if kind == "mass":
        s["lse"] = _lse(s)
        s["mass"] = torch.rand((len(lens), hkv, width * page), generator=gen, device=_DEV)


def _lists(case, gen, t, hkv, news, lens):
    """Pages of each packed row and KV head, ascending, -1 past a row's own:
    the first, the last two, and others."""
    page = case["page"]
    seen = [_pages_of(n - k + i + 1, page) for n, k in zip(lens, news) for i in range(k)]
    seen = torch.tensor(seen, device=_DEV)[:, None, None]
    at = torch.arange(_pages_of(case["n"], page), device=_DEV)
    x = torch.rand((t, hkv, at.shape[0]), generator=gen, device=_DEV)
    x = x.masked_fill((at < _FIRST) | (at >= seen - _LAST), 2.0).masked_fill(at >= seen, -1.0)
    ids = x.topk(min(case["count"], at.shape[0]), -1).indices.sort(-1).values
    return torch.where(ids < seen, ids, -1).int()


def _lse(s):
    """Logarithm of the sum of each row's exponentiated scores, [T,Hq] fp32."""
    out = torch.empty(s["q"].shape[:2], device=_DEV)
    for b, rows, score in _score_rows(s):
        out[rows] = torch.logsumexp(score, -1).T
    return out


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    kind = s["kind"]
    if kind == "bounds":
        if own:
            _sparkq().paged_key_bounds(s["cache"], s["bounds"], s["table"], s["starts"],
                                       s["lengths"], max_new=s["new"])
        else:
            _bounds(s)
        return s["bounds"]
    if kind == "scores":
        if own:
            return _sparkq().paged_page_scores(s["q"], s["bounds"], s["table"], s["starts"],
                                               s["lengths"], page_size=s["page"],
                                               scale=s["scale"], max_new=s["new"])
        return _scores(s)
    if kind == "select":
        if own:
            return _sparkq().select_top(s["x"], s["count"], lengths=s["lengths"],
                                        first=s["first"], last=s["last"])
        return _select(s)
    if kind == "sparse":
        if own:
            return _sparkq().paged_sparse_sdpa(s["q"], s["cache"], s["pages"], s["table"],
                                               s["starts"], s["lengths"], scale=s["scale"],
                                               max_new=s["new"])
        return _sparse(s)
    if kind == "mass":
        if own:
            _sparkq().paged_kv_mass(s["q"], s["lse"], s["cache"], s["mass"], s["table"],
                                    s["starts"], s["lengths"], scale=s["scale"],
                                    max_new=s["new"])
        else:
            _mass(s)
        return s["mass"]
    if own:
        table, lengths, missing = _sparkq().kv_pages_evict(s["cache"], s["keep"], s["table"],
                                                           s["lengths"], mass=s["mass"])
    else:
        table, lengths, missing = _evict(s)
    return (table, lengths, missing, *s["cache"], s["mass"])


def _rows(s):
    """(sequence, last token that it sees) of each packed row."""
    starts = s["starts"].long()
    t = torch.arange(int(s["q"].shape[0]), device=_DEV)
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    return b, s["lengths"].long()[b] - starts[b + 1] + t


def _bounds(s):
    kc, ks = s["cache"][:2]
    page, table = s["page"], s["table"].long()
    at = torch.arange(table.shape[1], device=_DEV)
    n = s["lengths"].long()[:, None]
    count = (s["starts"][1:] - s["starts"][:-1]).long()[:, None]
    b, j = ((count > 0) & (at >= (n - count) // page) & (at * page < n)).nonzero(as_tuple=True)
    ids = table[b, j]
    x = kc[ids].float() * ks[ids].float()[..., None]
    live = (j[:, None] * page + torch.arange(page, device=_DEV) < n[b])[:, None, :, None]
    lo = x.masked_fill(~live, math.inf).amin(2)
    hi = x.masked_fill(~live, -math.inf).amax(2)
    s["bounds"][ids, :, 0] = -_up(-lo)
    s["bounds"][ids, :, 1] = _up(hi)


def _up(x):
    """fp32 rounded up to bf16."""
    bits = x.contiguous().view(torch.int32)
    cut = bits & -65536
    return torch.where((cut != bits) & (bits >= 0), cut + 65536, cut).view(torch.float32).bfloat16()


def _scores(s):
    q, bounds, table = s["q"].float(), s["bounds"], s["table"]
    b, last = _rows(s)
    hkv = bounds.shape[1]
    out = torch.empty((q.shape[0], hkv, table.shape[1]), device=_DEV)
    at = torch.arange(table.shape[1], device=_DEV)
    for i in range(table.shape[0]):
        rows = (b == i).nonzero()[:, 0]
        if not rows.shape[0]:
            continue
        lo, hi = bounds[table[i].clamp(min=0).long()].float().permute(2, 1, 3, 0)
        x = q[rows].reshape(rows.shape[0], hkv, -1, q.shape[2]).permute(1, 2, 0, 3)
        y = torch.matmul(x.clamp(min=0), hi[:, None].contiguous())
        y += torch.matmul(x.clamp(max=0), lo[:, None].contiguous())
        y = (y * s["scale"]).amax(1).transpose(0, 1)
        hidden = (at * s["page"] > last[rows, None]) | (table[i] < 0)
        out[rows] = y.masked_fill(hidden[:, None], -math.inf)
    return out, (last // s["page"] + 1).int()


def _select(s):
    x, n = s["x"], s["lengths"].long()[:, None, None]
    at = torch.arange(x.shape[-1], device=_DEV)
    rank = ((at < s["first"]) | (at >= n - s["last"])).int().masked_fill(at >= n, -1).expand(x.shape)
    order = x.sort(dim=-1, descending=True, stable=True).indices
    again = rank.gather(-1, order).sort(dim=-1, descending=True, stable=True).indices
    top = order.gather(-1, again)[..., : s["count"]].sort(-1).values
    short = top.new_full((*x.shape[:-1], max(0, s["count"] - x.shape[-1])), x.shape[-1])
    top = torch.cat([top, short], -1)
    # of a row with fewer values than `count` all are taken, and others behind them
    return torch.where(torch.arange(s["count"], device=_DEV) < n, top, -1).int()


def _sparse(s):
    kc, ks, vc, vs = s["cache"]
    q, page = s["q"], s["page"]
    b, last = _rows(s)
    t, hq, d = q.shape
    hkv = kc.shape[1]
    heads = torch.arange(hkv, device=_DEV)[:, None]
    out = []
    for r in range(0, t, 64):
        j = s["pages"][r:r + 64].long()
        ids = s["table"].long()[b[r:r + 64, None, None], j.clamp(min=0)]
        pos = j[..., None] * page + torch.arange(page, device=_DEV)
        see = ((j[..., None] >= 0) & (pos <= last[r:r + 64, None, None, None])).flatten(2)[:, :, None]
        k = (kc[ids, heads].float() * ks[ids, heads].float()[..., None]).flatten(2, 3)
        x = q[r:r + 64].float().reshape(-1, hkv, hq // hkv, d)
        score = torch.matmul(x, k.transpose(2, 3).contiguous()) * s["scale"]
        del k
        score = score.masked_fill(~see, -math.inf)
        p = torch.exp(score - score.amax(-1, keepdim=True))
        p = p / p.sum(-1, keepdim=True)
        v = (vc[ids, heads].float() * vs[ids, heads].float()[..., None]).flatten(2, 3)
        out.append(torch.matmul(p, v).reshape(-1, hq, d))
    return torch.cat(out).to(q.dtype)


def _score_rows(s):
    """(sequence, its packed rows, fp32 scores [Hq,rows,tokens], -inf where
    hidden) of each sequence that has rows."""
    kc, ks = s["cache"][:2]
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    hq, d = s["q"].shape[1:]
    hkv = kc.shape[1]
    for b, n in enumerate(lengths):
        rows = slice(starts[b], starts[b + 1])
        new = rows.stop - rows.start
        if not new:
            continue
        ids = s["table"][b, : _pages_of(n, s["page"])].long()
        k = (kc[ids].float() * ks[ids].float()[..., None]).permute(1, 3, 0, 2).reshape(hkv, d, -1)
        x = s["q"][rows].float().reshape(new, hkv, -1, d).permute(1, 2, 0, 3).reshape(hkv, -1, d)
        score = torch.matmul(x, k[..., :n].contiguous()).reshape(hq, new, n) * s["scale"]
        token = torch.arange(n, device=_DEV)
        last = n - new + torch.arange(new, device=_DEV)[:, None]
        yield b, rows, score.masked_fill_(token > last, -math.inf)


def _mass(s):
    hkv = s["mass"].shape[1]
    for b, rows, score in _score_rows(s):
        n, new = score.shape[2], score.shape[1]
        w = torch.exp(score - s["lse"][rows].T[..., None]).reshape(hkv, -1, n).sum(1)
        s["mass"][b, :, n - new:n] = 0
        s["mass"][b, :, :n] += w


def _evict(s):
    table, page, count = s["table"].long(), s["page"], s["keep"].shape[-1]
    pages, width = s["cache"][0].shape[1], s["table"].shape[1]
    n = s["lengths"].long()
    at = torch.arange(width, device=_DEV)
    held = at < -(-n // page)[:, None]
    holders = torch.bincount(table[held], minlength=pages)
    less = n > count
    written = less[:, None] & (at < _pages_of(count, page))
    fresh = written & (holders[table.clamp(min=0)] > 1)
    free = (holders == 0).nonzero()[:, 0]
    rank = (fresh.reshape(-1).cumsum(0) - 1).reshape(fresh.shape)
    short = (fresh.sum() - free.shape[0]).clamp(min=0)
    after = torch.where(less, n.clamp(max=count), n)
    given = torch.cat([free, free.new_full((fresh.numel(),), -1)])[rank.clamp(min=0)]
    to = torch.where(fresh, given, table)
    to = torch.where(at < -(-after // page)[:, None], to, -1)
    i = torch.arange(count, device=_DEV)
    if short == 0:
        rows = less.nonzero()[:, 0]
        for layer in range(s["cache"][0].shape[0]):
            src = s["keep"][layer, rows].long()  # [rows,Hkv,count]
            heads = torch.arange(src.shape[1], device=_DEV)[:, None]
            ids = table[rows[:, None, None], src // page]
            dst = to[rows][:, None, i // page]
            for buf in s["cache"]:
                buf[layer][dst, heads, i % page] = buf[layer][ids, heads, src % page]
            s["mass"][layer, rows, :, :count] = s["mass"][layer, rows].gather(-1, src)
    return to.int(), after.int(), short.int().reshape(1)


# ---------------------------------------------------------------------------
# the work that no implementation can do without
# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "select":
        rng = random.Random(case["mix"])
        lens = [case["n"]] + [_log(rng, max(1, case["n"] // 4), case["n"])
                              for _ in range(case["b"] - 1)]
        rows = max(1, case["layers"]) * case["h"]
        return {"bytes": 4 * rows * (sum(lens) + case["b"] * case["count"]), "flops": 0}
    hq, hkv, d = _HEADS[case["heads"]]
    page = case["page"]
    if kind == "evict":
        lens, _ = _evicted(case)
        kept = sum(case["count"] for n in lens if n > case["count"])
        one = 2 * (d + 2) + 4  # a token's keys, values and weight, in a layer and head
        return {"bytes": case["layers"] * hkv * kept * (2 * one + 4), "flops": 0}
    news, lens = _batch(case)
    t = sum(news)
    if kind == "bounds":
        pages, tokens = _touched(case)
        return {"bytes": hkv * (tokens * (d + 2) + 4 * d * pages), "flops": 3 * hkv * tokens * d}
    read = [(v, k) for v, k in zip(lens, news) if k]
    table = 4 * sum(_pages_of(v, page) for v, _ in read)
    if kind == "scores":
        pages = sum(_pages_of(v, page) for v, _ in read)
        seen = sum(k * _pages_of(v, page) for v, k in read)
        return {"bytes": 2 * t * hq * d + 4 * pages * hkv * d + table
                + 4 * t * hkv * _pages_of(case["n"], page), "flops": 4 * hq * d * seen}
    if kind == "sparse":
        distinct = pairs = 0.0
        for v, k in read:
            p = _pages_of(v, page)
            c = min(case["count"], p)
            pairs += k * min(c * page, v)
            # (on average, of lists that are chosen apart from one another)
            distinct += min(v, page * (p * (1 - (1 - c / p) ** k) if c < p else p))
        return {"bytes": int(4 * t * hq * d + 2 * distinct * hkv * (d + 2)
                             + 4 * t * hkv * case["count"]), "flops": int(4 * hq * d * pairs)}
    tokens = sum(v for v, _ in read)
    pairs = sum(k * v - k * (k - 1) // 2 for v, k in read)
    return {"bytes": 2 * t * hq * d + 4 * t * hq + tokens * hkv * (d + 2 + 8) + table,
            "flops": 2 * hq * d * pairs}


# ---------------------------------------------------------------------------
# the definitions in float64, one sequence, row or page at a time
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"bounds": _exact_bounds, "scores": _exact_scores, "select": _exact_select,
            "sparse": _exact_sparse, "mass": _exact_mass, "evict": _exact_evict}[case["kind"]](s)


def _exact_bounds(s):
    kc, ks = s["cache"][:2]
    out = s["bounds"].double()
    table, starts, lengths = s["table"].tolist(), s["starts"].tolist(), s["lengths"].tolist()
    page = s["page"]

    def ceil8(x):  # to eight bits, upwards
        m, e = torch.frexp(x)
        return torch.ldexp(torch.ceil(m * 256), e - 8)

    for b, n in enumerate(lengths):
        new = starts[b + 1] - starts[b]
        for j in range((n - new) // page, _pages_of(n, page)) if new else ():
            p, k = table[b][j], min(page, n - j * page)
            x = kc[p, :, :k].double() * ks[p, :, :k].double()[..., None]
            out[p, :, 0] = -ceil8(-x.amin(1))
            out[p, :, 1] = ceil8(x.amax(1))
    return out


def _exact_scores(s):
    q, bounds = s["q"].double(), s["bounds"].double()
    starts, lengths, page = s["starts"].tolist(), s["lengths"].tolist(), s["page"]
    t, hq, _ = q.shape
    hkv = bounds.shape[1]
    out = q.new_full((t, hkv, s["table"].shape[1]), -math.inf)
    seen = torch.zeros(t, dtype=torch.int32, device=_DEV)
    for b, n in enumerate(lengths):
        rows = slice(starts[b], starts[b + 1])
        if rows.start == rows.stop:
            continue
        own_pages = _pages_of(n, page)
        ids = s["table"][b, :own_pages].long()
        for h in range(hkv):
            lo, hi = bounds[ids, h, 0], bounds[ids, h, 1]
            mid, half = (lo + hi) / 2, (hi - lo) / 2
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                x = q[rows, g]
                y = (x @ mid.T + x.abs() @ half.T) * s["scale"]
                out[rows, h, :own_pages] = torch.maximum(out[rows, h, :own_pages], y)
        for i in range(rows.start, rows.stop):
            k = (n - rows.stop + i) // page + 1
            seen[i] = k
            out[i, :, k:] = -math.inf
    return out, seen


def _exact_select(s):
    x, lengths, count = s["x"].cpu().numpy(), s["lengths"].tolist(), s["count"]
    flat = x.reshape(-1, len(lengths), *x.shape[-2:])
    out = np.full((*flat.shape[:-1], count), -1, dtype=np.int32)
    for layer in range(flat.shape[0]):
        for b, n in enumerate(lengths):
            at = np.arange(n)
            forced = (at < s["first"]) | (at >= n - s["last"])
            for h in range(flat.shape[2]):
                row = np.where(forced, np.inf, flat[layer, b, h, :n])
                top = np.sort(np.argsort(-row, kind="stable")[:count])
                out[layer, b, h, : len(top)] = top
    return torch.from_numpy(out.reshape(*x.shape[:-1], count)).to(_DEV)


def _exact_sparse(s):
    kc, ks, vc, vs = s["cache"]
    q, starts, lengths = s["q"].double(), s["starts"].tolist(), s["lengths"].tolist()
    lists, table, page = s["pages"].tolist(), s["table"].tolist(), s["page"]
    hq, d = q.shape[1:]
    hkv = kc.shape[1]
    group = hq // hkv
    out = torch.zeros_like(q)
    for b, n in enumerate(lengths):
        for t in range(starts[b], starts[b + 1]):
            last = n - starts[b + 1] + t
            for h in range(hkv):
                picked = [j for j in lists[t][h] if j >= 0]
                # only the last of them, in order, can be cut by what the row sees
                live = sum(min(page, last + 1 - j * page) for j in picked)
                ids = torch.tensor([table[b][j] for j in picked], device=_DEV)
                k = (kc[ids, h].double() * ks[ids, h, :, None].double()).reshape(-1, d)[:live]
                v = (vc[ids, h].double() * vs[ids, h, :, None].double()).reshape(-1, d)[:live]
                w = torch.softmax((q[t, h * group:(h + 1) * group] @ k.T) * s["scale"], -1)
                out[t, h * group:(h + 1) * group] = w @ v
    return out


def _exact_mass(s):
    kc, ks = s["cache"][:2]
    q, lse = s["q"].double(), s["lse"].double()
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    hq, d = q.shape[1:]
    hkv = kc.shape[1]
    out = s["mass"].double()
    for b, n in enumerate(lengths):
        rows = slice(starts[b], starts[b + 1])
        new = rows.stop - rows.start
        if not new:
            continue
        ids = s["table"][b, : _pages_of(n, s["page"])].long()
        see = torch.ones((new, n), dtype=torch.bool, device=_DEV).tril(n - new)
        out[b, :, n - new:n] = 0
        for h in range(hkv):
            k = (kc[ids, h].double() * ks[ids, h, :, None].double()).reshape(-1, d)[:n]
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                w = torch.exp((q[rows, g] @ k.T) * s["scale"] - lse[rows, g, None])
                out[b, h, :n] += torch.where(see, w, 0.0).sum(0)
    return out


def _exact_evict(s):
    page, pages, width = s["page"], s["cache"][0].shape[1], s["table"].shape[1]
    old, lens, count = s["table"].tolist(), s["lengths"].tolist(), s["keep"].shape[-1]
    rows = [r[: _pages_of(n, page)] for r, n in zip(old, lens)]
    holders = {}
    for r in rows:
        for p in r:
            holders[p] = holders.get(p, 0) + 1
    free = [p for p in range(pages) if p not in holders]
    given, table, after = 0, [], []
    for r, n in zip(rows, lens):
        if n > count:
            new = []
            for p in r[: _pages_of(count, page)]:
                if holders[p] > 1:
                    p = free[given]
                    given += 1
                new.append(p)
            r, n = new, count
        table.append(r + [-1] * (width - len(r)))
        after.append(n)
    before = s["cache"]
    cache, mass = [t.clone() for t in before], s["mass"].clone()
    for b, n in enumerate(lens):
        if n <= count:
            continue
        was, now = _ints(rows[b]).long(), _ints(table[b]).long()
        for layer in range(mass.shape[0]):
            for h in range(mass.shape[2]):
                src = s["keep"][layer, b, h].long()
                i = torch.arange(count, device=_DEV)
                mass[layer, b, h, :count] = s["mass"][layer, b, h, src]
                for x, y in zip(before, cache):
                    y[layer, now[i // page], h, i % page] = x[layer, was[src // page], h, src % page]
    return (_ints(table), _ints(after), _ints([max(0, given - len(free))]), *cache, mass)
