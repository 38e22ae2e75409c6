"""Plain float64 forms of the paged-cache operators on the CPU, and batches to
run them on. Tables, lengths and starts are Python lists here; every rule of
the operators' documentation is restated one token or one page at a time."""

import math
import random

import torch


def norm_rope(x, w, pos, dims, eps, base, scale=1.0, traditional=False):
    """(result, |parts| that the rotation adds up), float64."""
    x, w = x.double(), w.double()
    y = x / torch.sqrt((x * x).mean(-1, keepdim=True) + eps) * w
    out, parts = y.clone(), y.abs()
    for i in range(dims // 2):
        a, b = (2 * i, 2 * i + 1) if traditional else (i, i + dims // 2)
        t = scale * pos.double() * math.pow(base, -2.0 * i / dims)
        c, s = torch.cos(t)[:, None], torch.sin(t)[:, None]
        out[..., a] = y[..., a] * c - y[..., b] * s
        out[..., b] = y[..., a] * s + y[..., b] * c
        parts[..., a] = parts[..., b] = y[..., a].abs() + y[..., b].abs()
    return out, parts


def quantize(x):
    """(codes, scales) of rows of x, float64: the kv_quantize_s8 formula."""
    x = x.double()
    s = (x.abs().amax(-1) / 127).half()
    s = torch.where(s == 0, torch.ones_like(s), s)
    return torch.clamp(torch.round(x / s.double()[..., None]), -127, 127).to(torch.int8), s


def page_at(table, pages, page, b, pos):
    j = pos // page
    if pos < 0 or j >= len(table[b]) or not 0 <= table[b][j] < pages:
        return None
    return table[b][j]


def rows_of(starts, lengths, t, b, room):
    first = min(max(starts[b], 0), t)
    count = min(max(starts[b + 1], first), t) - first
    return first, count, min(max(lengths[b], 0), room)


def append(keys, values, cache, table, starts, lengths):
    """The cache's tensors (CPU copies) with the new tokens in them."""
    kc, ks, vc, vs = (c.clone() for c in cache)
    pages, _, page, _ = kc.shape
    for b in range(len(lengths)):
        first, count, n = rows_of(starts, lengths, len(keys), b, len(table[b]) * page)
        for i in range(count):
            pos = n - count + i
            p = page_at(table, pages, page, b, pos)
            if p is None:
                continue
            for x, c, s in ((keys, kc, ks), (values, vc, vs)):
                c[p, :, pos % page], s[p, :, pos % page] = quantize(x[first + i])
    return kc, ks, vc, vs


def attention(q, cache, table, starts, lengths, scale, causal=True, max_new=1 << 30):
    """(out, sum p|v| / sum p, largest scale * sum |q||k| of the row, written, the
    largest p / sum p times the largest value scale times sum |code|)."""
    kc, ks, vc, vs = cache
    pages, hkv, page, d = kc.shape
    t, hq, _ = q.shape
    out = torch.zeros((t, hq, d), dtype=torch.float64)
    mass = torch.zeros((t, hq, d), dtype=torch.float64)
    size = torch.zeros((t, hq), dtype=torch.float64)
    done = torch.zeros(t, dtype=torch.bool)
    steps = torch.zeros((t, hq, d), dtype=torch.float64)
    g = hq // hkv
    qd = q.double()
    for b in range(len(lengths)):
        first, count, n = rows_of(starts, lengths, t, b, len(table[b]) * page)
        at = [(page_at(table, pages, page, b, pos), pos) for pos in range(n)]
        at = [(p, pos) for p, pos in at if p is not None]
        ids = torch.tensor([p for p, _ in at], dtype=torch.long)
        pos = torch.tensor([p for _, p in at], dtype=torch.long)
        for i in range(min(count, max_new)):
            done[first + i] = True
            see = pos <= n - count + i if causal else pos < n
            if not bool(see.any()):
                continue
            p, s = ids[see], pos[see] % page
            k = kc[p, :, s].double() * ks[p, :, s].double()[..., None]  # [n, hkv, d]
            v = vc[p, :, s].double() * vs[p, :, s].double()[..., None]
            codes, most = vc[p, :, s].double().abs().sum(0), vs[p, :, s].double().abs().amax(0)
            for h in range(hq):
                sc = (k[:, h // g] @ qd[first + i, h]) * scale
                w = torch.softmax(sc, 0)
                out[first + i, h] = w @ v[:, h // g]
                mass[first + i, h] = w @ v[:, h // g].abs()
                steps[first + i, h] = w.max() * most[h // g] * codes[h // g]
                size[first + i, h] = abs(scale) * (k[:, h // g].abs() @ qd[first + i, h].abs()).max()
    return out, mass, size, done, steps


def held(table, lengths, b, pages, page):
    """Entries of row b's pages, None where one is none."""
    n = min(max(lengths[b], 0), len(table[b]) * page)
    return n, [p if 0 <= p < pages else None for p in table[b][: -(-n // page)]]


def fork(table, lengths, parents, fresh, pages, page):
    """(table, lengths, missing, [(from, to)]) -- the pages copied."""
    width = len(table[0]) if table else 0
    rows, before, after = [], [], []
    for p, k in zip(parents, fresh):
        n, r = held(table, lengths, p, pages, page) if 0 <= p < len(table) else (0, [])
        rows.append(r)
        before.append(n)
        after.append(min(n + max(k, 0), width * page))
    holds = {}
    for r in rows:
        for p in r:
            if p is not None:
                holds[p] = holds.get(p, 0) + 1
    writers = {}
    for i, r in enumerate(rows):
        if before[i] % page and after[i] > before[i] and r[-1] is not None:
            writers.setdefault(r[-1], []).append(i)
    free = [p for p in range(pages) if p not in holds]
    pairs, given = [], 0

    def deal():
        nonlocal given
        given += 1
        return free[given - 1] if given <= len(free) else -1

    for i, r in enumerate(rows):
        w = writers.get(r[-1]) if r else None
        if w and i in w and (holds[r[-1]] > len(w) or w[0] != i):
            old, r[-1] = r[-1], deal()
            pairs.append((old, r[-1]))
        while len(r) < -(-after[i] // page):
            r.append(deal())
    missing = max(0, given - len(free))
    out = [[-1 if p is None else p for p in r] + [-1] * (width - len(r)) for r in rows]
    return out, after, missing, [] if missing else pairs


def compact(table, lengths, pages, page):
    width = len(table[0]) if table else 0
    rows = [held(table, lengths, b, pages, page)[1] for b in range(len(table))]
    used = sorted({p for r in rows for p in r if p is not None})
    holes = [p for p in range(len(used)) if p not in set(used)]
    to = dict(zip([p for p in used if p >= len(used)], holes))
    out = [[-1 if p is None else to.get(p, p) for p in r] + [-1] * (width - len(r)) for r in rows]
    return out, len(used), list(to.items())


def pool(gen, pages, hkv, page, d, layers=None):
    lead = (pages,) if layers is None else (layers, pages)
    out = []
    for _ in range(2):
        out.append(torch.randint(-127, 128, (*lead, hkv, page, d), generator=gen, dtype=torch.int8))
        out.append((0.005 + 0.02 * torch.rand((*lead, hkv, page), generator=gen)).half())
    return tuple(out)


def tables(rng, lengths, page, pages, width):
    """Distinct pages in random order, -1 past a row's own."""
    ids = rng.sample(range(pages), sum(-(-n // page) for n in lengths))
    out = []
    for n in lengths:
        k = -(-n // page)
        out.append([ids.pop() for _ in range(k)] + [-1] * (width - k))
    return out


def batch(seed, lengths, news, hq, hkv, d, page, spare=3, extra_rows=0, width=None):
    """(q, k, v fp32 on the CPU, cache, table, starts) of a batch."""
    rng, gen = random.Random(seed), torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lengths]
    width = width or max(need + [1])
    cache = pool(gen, sum(need) + spare, hkv, page, d)
    table = tables(rng, lengths, page, sum(need) + spare, width)
    starts = [0]
    for n in news:
        starts.append(starts[-1] + n)
    t = starts[-1] + extra_rows
    q, k, v = (torch.randn((t, h, d), generator=gen) for h in (hq, hkv, hkv))
    return q, k, v, cache, table, starts
