"""Operators of a serving step over one paged INT8 KV cache, as cases that can
be timed: the norm and rotation of queries and keys in front of it, the
quantized append, the attention of new tokens, and the forking and compacting
of its pages.

Where `own` is false run() computes an operator's plain form in elementary
torch operations; where it is true it makes the framework's calls. exact()
restates the operators in float64.

Cache: (k_codes [layers,P,Hkv,page,D] int8, k_scales [layers,P,Hkv,page] fp16,
v_codes, v_scales); one layer of it for the append and the attention. Codes
are compared as the whole numbers that they are: the quotient of a 16-bit
value and an fp16 scale is never nearer to a rounding tie than 2^-19 of itself,
so every correct quantizer gives the same ones.
"""

import math
import os
import random
import sys

import torch

own = False

_DEV = "cuda"
_TYPES = {"bf16": torch.bfloat16, "f16": torch.float16}
# query heads, KV heads, head dim
_HEADS = {"32x8x128": (32, 8, 128), "16x4x256": (16, 4, 256), "20x4x128": (20, 4, 128)}
_EPS = 1e-6
_BASE = 1e6


def _sparkq():
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                        "spark-mlx-llm_amd")
    if path not in sys.path:
        sys.path.insert(0, path)
    import sparkq

    return sparkq


def listed():
    return [
        # queries and keys of one decoded token
        {"name": "norm_rope_1", "kind": "norm_rope", "t": 1, "heads": "32x8x128", "dims": 128,
         "dtype": "bf16"},
        # of a long prompt chunk
        {"name": "norm_rope_4096", "kind": "norm_rope", "t": 4096, "heads": "32x8x128",
         "dims": 128, "dtype": "bf16"},
        # one decoded token of each of 16 sequences into their pages
        {"name": "append_16", "kind": "append", "b": 16, "new": 1, "n": 2000, "page": 64,
         "heads": "32x8x128", "mix": 1, "dtype": "bf16"},
        # three prompt chunks of odd lengths, larger heads, small pages
        {"name": "append_3x2000", "kind": "append", "b": 3, "new": 2000, "n": 4000, "page": 16,
         "heads": "16x4x256", "mix": 2, "dtype": "f16"},
        # one decoded token over a cache of one middling sequence: latency
        {"name": "decode_1x4095", "kind": "sdpa", "b": 1, "new": 1, "n": 4095, "page": 64,
         "heads": "32x8x128", "mix": 0, "dtype": "bf16"},
        # a serving batch's decode step, lengths from short to long
        {"name": "decode_64x8192", "kind": "sdpa", "b": 64, "new": 1, "n": 8192, "page": 64,
         "heads": "32x8x128", "mix": 3, "dtype": "bf16"},
        # one prompt's last chunk over what it has cached before
        {"name": "chunk_2048x8192", "kind": "sdpa", "b": 1, "new": 2048, "n": 8192, "page": 64,
         "heads": "32x8x128", "mix": 0, "dtype": "bf16"},
        # prompt chunks and decoded tokens in one batch, larger heads, odd lengths
        {"name": "mixed_24x1000", "kind": "sdpa", "b": 24, "new": 1000, "n": 4000, "page": 32,
         "heads": "16x4x256", "mix": 4, "dtype": "f16"},
        # a beam search step of 8 beams: reordered, their last pages copied
        {"name": "fork_8", "kind": "fork", "b": 8, "n": 700, "page": 32, "pages": 512,
         "layers": 4, "heads": "32x8x128", "mix": 5},
        # a sampling step of 256 sequences with shared prefixes, some of which end
        {"name": "fork_256", "kind": "fork", "b": 256, "n": 500, "page": 64, "pages": 2048,
         "layers": 8, "heads": "32x8x128", "mix": 6},
        # a few sequences left in a small pool
        {"name": "compact_4", "kind": "compact", "b": 4, "n": 900, "page": 32, "pages": 256,
         "layers": 4, "heads": "32x8x128", "mix": 7},
        # a large pool, under half of it in use
        {"name": "compact_96", "kind": "compact", "b": 96, "n": 900, "page": 64, "pages": 2048,
         "layers": 8, "heads": "32x8x128", "mix": 8},
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["norm_rope", "append", "sdpa", "sdpa", "sdpa", "fork", "compact"])
    dtype = rng.choice(["bf16", "bf16", "f16"])
    heads = rng.choice(sorted(_HEADS))
    mix = rng.randint(10, 9999)
    page = rng.choice([16, 32, 64, 128])
    if kind == "norm_rope":
        d = _HEADS[heads][2]
        return {"kind": kind, "t": _log(rng, 1, 4096), "heads": heads,
                "dims": rng.choice([d, d, d // 2]), "dtype": dtype}
    if kind == "append":
        new = _log(rng, 1, 2000)
        b = rng.randint(1, max(1, min(64, 6000 // new)))
        return {"kind": kind, "b": b, "new": new, "n": new + _log(rng, 1, 2000), "page": page,
                "heads": heads, "mix": mix, "dtype": dtype}
    if kind == "sdpa":
        if rng.random() < 0.5:  # decode, or the verification of a few drafted tokens
            return {"kind": kind, "b": _log(rng, 1, 64), "new": rng.choice([1, 1, 1, 4]),
                    "n": _log(rng, 8, 8192), "page": page, "heads": heads, "mix": mix,
                    "dtype": dtype}
        new = _log(rng, 8, 1000)
        return {"kind": kind, "b": rng.randint(1, 12), "new": new,
                "n": new + _log(rng, 1, 3000), "page": page, "heads": heads, "mix": mix,
                "dtype": dtype}
    b = _log(rng, 2, 200)
    n = _log(rng, 20, 900)
    return {"kind": kind, "b": b, "n": n, "page": page,
            "pages": b * (-(-n // page) + 2) + rng.randint(1, 400),
            "layers": rng.randint(1, 4), "heads": "32x8x128", "mix": mix}


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


def _rows(case):
    """A page case's sequences: lengths before the step, parents, new tokens.
    Every fourth sequence shares its parent with the one before it; one of
    sixteen ends."""
    rng = random.Random(case["mix"])
    b, n = case["b"], case["n"]
    lens = [n] + [_log(rng, max(1, n // 8), n) for _ in range(b - 1)]
    parents = [i - 1 if i % 4 == 1 else (-1 if i % 16 == 15 else i) for i in range(b)]
    return lens, parents, [1] * b


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


def _table(gen, lens, page, pages, width):
    """Pages in random order for sequences of these lengths, -1 elsewhere."""
    counts = [_pages_of(v, page) for v in lens]
    ids = torch.randperm(pages, generator=gen, device=_DEV)[: sum(counts)].to(torch.int32)
    table = torch.full((len(lens), width), -1, dtype=torch.int32, device=_DEV)
    live = torch.arange(width, device=_DEV)[None] < torch.tensor(counts, device=_DEV)[:, None]
    table[live] = ids
    return table


def prepare(case, seed):
    gen = _gen(seed)
    kind = case["kind"]
    s = {"kind": kind}
    if kind == "norm_rope":
        hq, hkv, d = _HEADS[case["heads"]]
        dtype = _TYPES[case["dtype"]]
        # views of the packed projection's rows, as a layer has them
        qkv = _randn(gen, case["t"], hq + 2 * hkv, d, dtype=dtype)
        s["q"], s["k"] = qkv[:, :hq], qkv[:, hq:hq + hkv]
        s["wq"], s["wk"] = ((1 + 0.2 * _randn(gen, d)).to(dtype) for _ in range(2))
        s["pos"] = torch.randint(0, 131072, (case["t"],), generator=gen, device=_DEV,
                                 dtype=torch.int32)
        s["dims"] = case["dims"]
        return s
    hq, hkv, d = _HEADS[case["heads"]]
    page = case["page"]
    s["page"] = page
    if kind in ("append", "sdpa"):
        news, lens = _batch(case)
        dtype = _TYPES[case["dtype"]]
        width = _pages_of(case["n"], page)
        pages = sum(_pages_of(v, page) for v in lens) + 3
        s["cache"] = tuple(t[0] for t in _pool(gen, 1, pages, hkv, page, d))
        s["table"] = _table(gen, lens, page, pages, width)
        s["lengths"] = _ints(lens)
        s["starts"] = _ints([0] + torch.tensor(news).cumsum(0).tolist())
        s["new"] = max(news)
        t = sum(news)
        if kind == "append":
            s["k"], s["v"] = (_randn(gen, t, hkv, d, dtype=dtype) for _ in range(2))
        else:
            s["q"] = _randn(gen, t, hq, d, dtype=dtype)
            s["scale"] = d ** -0.5
        return s
    lens, parents, new = _rows(case)
    s["cache"] = _pool(gen, case["layers"], case["pages"], hkv, page, d)
    s["table"] = _table(gen, lens, page, case["pages"], _pages_of(case["n"], page) + 1)
    s["lengths"], s["parents"], s["new"] = _ints(lens), _ints(parents), _ints(new)
    return s


# ---------------------------------------------------------------------------
# one pass
# ---------------------------------------------------------------------------

def run(s):
    kind = s["kind"]
    if kind == "norm_rope":
        if own:
            return _sparkq().qk_norm_rope(s["q"], s["k"], s["wq"], s["wk"], s["pos"],
                                          dims=s["dims"], eps=_EPS, base=_BASE)
        cos, sin = _angles(s["pos"], s["dims"])
        return (_norm_rope(s["q"], s["wq"], cos, sin, s["dims"]),
                _norm_rope(s["k"], s["wk"], cos, sin, s["dims"]))
    if kind == "append":
        if own:
            _sparkq().paged_kv_append(s["k"], s["v"], s["cache"], s["table"], s["starts"],
                                      s["lengths"])
        else:
            _append(s)
        return s["cache"]
    if kind == "sdpa":
        if own:
            return _sparkq().paged_quantized_sdpa(s["q"], s["cache"], s["table"], s["starts"],
                                                  s["lengths"], scale=s["scale"],
                                                  max_new=s["new"])
        return _attention(s)
    if kind == "fork":
        if own:
            table, lengths, missing = _sparkq().kv_pages_fork(s["cache"], s["table"], s["lengths"],
                                                              s["parents"], s["new"])
        else:
            table, lengths, missing = _fork(s)
        return (table, lengths, missing, *s["cache"])
    if own:
        table, used = _sparkq().kv_pages_compact(s["cache"], s["table"], s["lengths"])
    else:
        table, used = _compact(s)
    return (table, used, *s["cache"])


def _angles(pos, dims):
    i = torch.arange(dims // 2, device=_DEV, dtype=torch.float64)
    theta = pos.double()[:, None] * _BASE ** (-2 * i / dims)
    return theta.cos().float()[:, None], theta.sin().float()[:, None]


def _norm_rope(x, w, cos, sin, dims):
    y = x.float()
    y = y * torch.rsqrt(y.square().mean(-1, keepdim=True) + _EPS) * w.float()
    a, b = y[..., :dims // 2], y[..., dims // 2:dims]
    return torch.cat([a * cos - b * sin, b * cos + a * sin, y[..., dims:]], -1).to(x.dtype)


def _places(s):
    """(page, slot) of each packed new token."""
    starts, page = s["starts"].long(), s["page"]
    t = torch.arange(s["k"].shape[0], device=_DEV)
    b = torch.searchsorted(starts[1:].contiguous(), t, right=True)
    pos = s["lengths"].long()[b] - (starts[b + 1] - starts[b]) + t - starts[b]
    return s["table"].long()[b, pos // page], pos % page


def _append(s):
    ids, slot = _places(s)
    kc, ks, vc, vs = s["cache"]
    for x, codes, scales in ((s["k"], kc, ks), (s["v"], vc, vs)):
        x = x.float()
        sc = (x.abs().amax(-1) / 127).half()
        sc = torch.where(sc == 0, torch.ones_like(sc), sc)
        q = torch.round(x / sc.float()[..., None]).clamp(-127, 127)
        codes[ids, :, slot] = q.to(torch.int8)
        scales[ids, :, slot] = sc


def _values(codes, scales, table):
    """fp32 [B,Hkv,tokens,D] of a batch's pages (page 0 in place of none)."""
    ids = table.clamp(min=0).long()
    x = codes[ids].float() * scales[ids].float()[..., None]
    b, m, h, p, d = x.shape
    return x.transpose(1, 2).reshape(b, h, m * p, d)


def _attention(s):
    kc, ks, vc, vs = s["cache"]
    q, starts, lengths, new = s["q"], s["starts"].long(), s["lengths"].long(), s["new"]
    t, hq, d = q.shape
    b, hkv = lengths.shape[0], kc.shape[1]
    count = starts[1:] - starts[:-1]
    row = torch.arange(new, device=_DEV)
    index = (starts[:-1, None] + row).clamp(max=t - 1)  # [B,new]
    qp = q[index].float().transpose(1, 2).reshape(b, hkv, -1, d)
    k = _values(kc, ks, s["table"]).transpose(2, 3).contiguous()
    score = torch.matmul(qp, k).reshape(b, hq, new, -1) * s["scale"]
    del k
    token = torch.arange(score.shape[-1], device=_DEV)
    last = (lengths - count)[:, None] + row  # [B,new]
    score.masked_fill_((token > last[..., None])[:, None], -math.inf)
    p = torch.exp(score - score.amax(-1, keepdim=True))
    p /= p.sum(-1, keepdim=True)
    out = torch.matmul(p.reshape(b, hkv, -1, p.shape[-1]), _values(vc, vs, s["table"]))
    out = out.reshape(b, hq, new, d).transpose(1, 2)
    return out[row < count[:, None]].to(q.dtype)


def _held(table, lengths, pages, page):
    at = torch.arange(table.shape[1], device=_DEV)
    return (at < -(-lengths // page)[:, None]) & (table >= 0) & (table < pages)


def _fork(s):
    page, pages, width = s["page"], s["cache"][0].shape[1], s["table"].shape[1]
    parents = s["parents"].long()
    n = parents.shape[0]
    order = torch.arange(n, device=_DEV)
    real = (parents >= 0) & (parents < s["table"].shape[0])
    parents = torch.where(real, parents, 0)
    table = s["table"].long()[parents]
    before = torch.where(real, s["lengths"].long()[parents], 0)
    after = (before + s["new"].long()).clamp(max=width * page)
    held = _held(table, before, pages, page)
    table = torch.where(held, table, -1)
    holders = torch.bincount(table[held], minlength=pages + 1)
    # the partly filled last pages that this step's tokens go to
    last = (-(-before // page) - 1).clamp(min=0)
    mine = table.gather(1, last[:, None])[:, 0]
    mine = torch.where((before % page != 0) & (after > before) & (mine >= 0), mine, pages)
    writers = torch.bincount(mine, minlength=pages + 1)
    first = torch.full((pages + 1,), n, device=_DEV).scatter_reduce(0, mine, order, "amin")
    copied = (mine < pages) & ((holders > writers)[mine] | (first[mine] != order))
    at = torch.arange(width, device=_DEV)
    wanted = (at >= -(-before // page)[:, None]) & (at < -(-after // page)[:, None])
    wanted |= copied[:, None] & (at == last[:, None])
    free = (holders[:pages] == 0).nonzero()[:, 0]
    rank = (wanted.reshape(-1).cumsum(0) - 1).reshape(wanted.shape)
    short = (wanted.sum() - free.shape[0]).clamp(min=0)
    given = torch.cat([free, free.new_full((n * width,), -1)])[rank.clamp(min=0)]
    table = torch.where(wanted, given, table)
    to = table.gather(1, last[:, None])[:, 0][copied]
    if short == 0:
        for buf in s["cache"]:
            buf[:, to] = buf[:, mine[copied]]
    return table.int(), after.int(), short.int().reshape(1)


def _compact(s):
    pages, table = s["cache"][0].shape[1], s["table"].long()
    held = _held(table, s["lengths"].long(), pages, s["page"])
    used = torch.bincount(table[held], minlength=pages) > 0
    count = used.sum()
    number = torch.arange(pages, device=_DEV)
    moved = (used & (number >= count)).nonzero()[:, 0]
    to = (~used & (number < count)).nonzero()[:, 0]
    number[moved] = to
    for buf in s["cache"]:
        buf[:, to] = buf[:, moved]
    table = torch.where(held, number[table.clamp(min=0)], -1)
    return table.int(), count.int().reshape(1)


# ---------------------------------------------------------------------------
# the work that no implementation can do without
# ---------------------------------------------------------------------------

def work(case):
    hq, hkv, d = _HEADS[case["heads"]]
    kind = case["kind"]
    if kind == "norm_rope":
        values = case["t"] * (hq + hkv) * d
        return {"bytes": 4 * values + 4 * case["t"] + 4 * d, "flops": 10 * values}
    page = case["page"]
    if kind in ("append", "sdpa"):
        news, lens = _batch(case)
        t = sum(news)
        if kind == "append":
            values = 2 * t * hkv * d
            return {"bytes": 3 * values + 4 * t * hkv, "flops": 4 * values}
        read = [v for v, k in zip(lens, news) if k]
        pairs = sum(k * v - k * (k - 1) // 2 for v, k in zip(lens, news))
        table = 4 * sum(_pages_of(v, page) for v in read)
        return {"bytes": 4 * t * hq * d + 2 * sum(read) * hkv * (d + 2) + table,
                "flops": 4 * hq * d * pairs}
    one = case["layers"] * 2 * hkv * page * (d + 2)  # bytes of a page in every layer
    lens, parents, new = _rows(case)
    width = _pages_of(case["n"], page) + 1
    if kind == "fork":
        # of two children of one parent in the middle of a page one copies it
        moved = sum(1 for i, p in enumerate(parents)
                    if p >= 0 and p == i - 1 and lens[p] % page)
        return {"bytes": 2 * moved * one + 8 * case["b"] * width, "flops": 0}
    used = sum(_pages_of(v, page) for v in lens)
    moved = used * (case["pages"] - used) / case["pages"]  # on average, of random places
    return {"bytes": 2 * moved * one + 8 * case["b"] * width, "flops": 0}


# ---------------------------------------------------------------------------
# the definitions in float64, one sequence or page at a time
# ---------------------------------------------------------------------------

def exact(case, seed):
    s = prepare(case, seed)
    return {"norm_rope": _exact_norm_rope, "append": _exact_append, "sdpa": _exact_sdpa,
            "fork": _exact_fork, "compact": _exact_compact}[case["kind"]](s)


def _exact_norm_rope(s):
    half = s["dims"] // 2
    out = []
    for x, w in ((s["q"], s["wq"]), (s["k"], s["wk"])):
        x = x.double()
        y = x / (x.pow(2).sum(-1, keepdim=True) / x.shape[-1] + _EPS).sqrt() * w.double()
        z = y.clone()
        for i in range(half):
            angle = s["pos"].double() * math.pow(_BASE, -i / half)
            c, n = angle.cos()[:, None], angle.sin()[:, None]
            z[..., i] = y[..., i] * c - y[..., i + half] * n
            z[..., i + half] = y[..., i] * n + y[..., i + half] * c
        out.append(z)
    return tuple(out)


def _exact_append(s):
    kc, ks, vc, vs = (t.clone() for t in s["cache"])
    ks, vs = ks.double(), vs.double()
    table, page = s["table"].tolist(), s["page"]
    starts, lengths = s["starts"].tolist(), s["lengths"].tolist()
    for b, n in enumerate(lengths):
        t, end = starts[b], starts[b + 1]
        while t < end:  # a run of tokens that lie in one page
            pos = n - (end - t)
            at = pos % page
            k = min(end - t, page - at)
            for x, codes, scales in ((s["k"], kc, ks), (s["v"], vc, vs)):
                v = x[t:t + k].double()
                sc = (v.abs().amax(-1) / 127).half().double()
                sc[sc == 0] = 1
                q = (v / sc[..., None]).round().clamp(-127, 127).to(torch.int8)
                codes[table[b][pos // page], :, at:at + k] = q.transpose(0, 1)
                scales[table[b][pos // page], :, at:at + k] = sc.transpose(0, 1)
            t += k
    return kc, ks, vc, vs


def _exact_sdpa(s):
    kc, ks, vc, vs = s["cache"]
    q, starts, lengths = s["q"].double(), s["starts"].tolist(), s["lengths"].tolist()
    hq, d = q.shape[1:]
    hkv = kc.shape[1]
    out = torch.zeros_like(q)
    for b, n in enumerate(lengths):
        rows = slice(starts[b], starts[b + 1])
        new = rows.stop - rows.start
        if not new:
            continue
        ids = s["table"][b, : _pages_of(n, s["page"])].long()
        see = torch.ones((new, n), dtype=torch.bool, device=_DEV).tril(n - new)
        for h in range(hkv):
            k = (kc[ids, h].double() * ks[ids, h, :, None].double()).reshape(-1, d)[:n]
            v = (vc[ids, h].double() * vs[ids, h, :, None].double()).reshape(-1, d)[:n]
            for g in range(h * (hq // hkv), (h + 1) * (hq // hkv)):
                sc = torch.where(see, (q[rows, g] @ k.T) * s["scale"], -math.inf)
                out[rows, g] = torch.softmax(sc, -1) @ v
    return out


def _exact_fork(s):
    page, pages, width = s["page"], s["cache"][0].shape[1], s["table"].shape[1]
    old, lens = s["table"].tolist(), s["lengths"].tolist()
    rows, before, after = [], [], []
    for p, k in zip(s["parents"].tolist(), s["new"].tolist()):
        n = lens[p] if 0 <= p < len(old) else 0
        before.append(n)
        after.append(min(n + k, width * page))
        rows.append(old[p][: _pages_of(n, page)] if n else [])
    holders, writers = {}, {}
    for i, r in enumerate(rows):
        for p in r:
            holders[p] = holders.get(p, 0) + 1
        if before[i] % page and after[i] > before[i]:
            writers.setdefault(r[-1], []).append(i)
    free = [p for p in range(pages) if p not in holders]
    pairs, given = [], 0
    for i, r in enumerate(rows):
        if before[i] % page and after[i] > before[i]:
            w = writers[r[-1]]
            if holders[r[-1]] > len(w) or w[0] != i:
                pairs.append((r[-1], free[given]))
                r = r[:-1] + [free[given]]
                given += 1
        k = _pages_of(after[i], page) - len(r)
        rows[i] = r + free[given:given + k]
        given += k
    table = [r + [-1] * (width - len(r)) for r in rows]
    cache = [t.clone() for t in s["cache"]]
    for a, b in pairs:
        for t in cache:
            t[:, b] = t[:, a]
    return (_ints(table), _ints(after), _ints([max(0, given - len(free))]), *cache)


def _exact_compact(s):
    page = s["page"]
    old, lens = s["table"].tolist(), s["lengths"].tolist()
    rows = [r[: _pages_of(n, page)] for r, n in zip(old, lens)]
    used = sorted({p for r in rows for p in r})
    holes = [p for p in range(len(used)) if p not in set(used)]
    to = dict(zip([p for p in used if p >= len(used)], holes))
    cache = [t.clone() for t in s["cache"]]
    for a, b in to.items():
        for t in cache:
            t[:, b] = t[:, a]
    table = [[to.get(p, p) for p in r] + [-1] * (s["table"].shape[1] - len(r)) for r in rows]
    return (_ints(table), _ints([len(used)]), *cache)
