"""Plain float64 forms of the long-context operators over a paged cache on the
CPU. Tables, lengths and starts are Python lists; every rule of the operators'
documentation is restated one token, page or row at a time."""

import math

import torch

import paged_reference as ref


def bf16_toward(x, up):
    """float64 to bfloat16, rounded up or down."""
    y = x.bfloat16()
    step = torch.where(y == 0, torch.full_like(x, 2.0 ** -133),
                       2.0 ** (torch.floor(torch.log2(y.double().abs().clamp(min=2.0 ** -126))) - 7))
    wrong = y.double() < x if up else y.double() > x
    # next to a power of two the step below is half as large
    towards_zero = (y.double() > 0) != up
    edge = torch.frexp(y.double().abs()).mantissa == 0.5
    step = torch.where(edge & towards_zero, step / 2, step)
    z = y.double() + (step if up else -step)
    return torch.where(wrong, z, y.double()).bfloat16()


BIG = torch.finfo(torch.bfloat16).max


def bounds(cache, before, table, starts, lengths):
    """The bounds' tensor (a CPU copy) with those of the new tokens' pages in it."""
    kc, ks = cache[:2]
    pages, _, page, _ = kc.shape
    out = before.clone()
    for b in range(len(lengths)):
        _, count, n = ref.rows_of(starts, lengths, 1 << 30, b, len(table[b]) * page)
        for j in sorted({pos // page for pos in range(max(n - count, 0), n)}):
            p = ref.page_at(table, pages, page, b, j * page)
            if p is None:
                continue
            k = min(page, n - j * page)
            x = kc[p, :, :k].double() * ks[p, :, :k].double()[..., None]
            out[p, :, 0] = bf16_toward(x.amin(1), False)
            out[p, :, 1] = bf16_toward(x.amax(1), True)
            odd = ~ks[p, :, :k].isfinite().all(1)
            out[p, odd, 0], out[p, odd, 1] = -BIG, BIG
    return out


def last_seen(n, count, i, causal):
    return min(max(n - count + i, -1), n - 1) if causal else n - 1


def scores(q, bnd, table, starts, lengths, page, scale, causal=True, max_new=1 << 30):
    """(scores, |scale| sum |q||bound| of each, seen, rows that are written)."""
    pages, hkv = bnd.shape[:2]
    t, hq, _ = q.shape
    g = hq // hkv
    width = len(table[0]) if table else 1
    out = torch.full((t, hkv, width), -math.inf, dtype=torch.float64)
    size = torch.zeros((t, hkv, width), dtype=torch.float64)
    seen = torch.zeros(t, dtype=torch.int32)
    done = torch.zeros(t, dtype=torch.bool)
    for b in range(len(lengths)):
        first, count, n = ref.rows_of(starts, lengths, t, b, width * page)
        for i in range(min(count, max_new)):
            r = first + i
            done[r] = True
            seen[r] = last_seen(n, count, i, causal) // page + 1
            for j in range(int(seen[r])):
                p = table[b][j]
                if not 0 <= p < pages:
                    continue
                x = q[r].double().reshape(hkv, g, -1) * scale
                lo, hi = bnd[p, :, 0].double()[:, None], bnd[p, :, 1].double()[:, None]
                out[r, :, j] = torch.maximum(x * lo, x * hi).sum(-1).amax(1)
                size[r, :, j] = (x.abs() * torch.maximum(lo.abs(), hi.abs())).sum(-1).amax(1)
    return out, size, seen, done


def select(x, count, lengths=None, first=0, last=0):
    """x [L,R,H,N] -> [L,R,H,count], one value at a time."""
    layers, rows, heads, n_all = x.shape
    out = torch.full((layers, rows, heads, count), -1, dtype=torch.int32)
    for layer in range(layers):
        for r in range(rows):
            n = n_all if lengths is None else min(max(lengths[r], 0), n_all)
            for h in range(heads):
                v = x[layer, r, h, :n].tolist()
                forced = [i < first or i >= n - last for i in range(n)]
                value = [-math.inf if w != w else w for w in v]
                order = sorted(range(n), key=lambda i: (not forced[i], -value[i], i))
                top = sorted(order[:count])
                out[layer, r, h, : len(top)] = torch.tensor(top, dtype=torch.int32)
    return out


def listed(selected, table, starts, lengths, pages, page, causal=True, max_new=1 << 30):
    """For each KV head: (tables, lengths) of as many sequences as there are packed
    rows, which see what the rows see of their listed pages (ascending lists: the page
    that ends inside is the last). None where no row is written."""
    t, hkv, _ = selected.shape
    out = []
    for h in range(hkv):
        tables, lens = [[] for _ in range(t)], [None] * t
        for b in range(len(lengths)):
            first, count, n = ref.rows_of(starts, lengths, t, b, len(table[b]) * page)
            for i in range(min(count, max_new)):
                lim = last_seen(n, count, i, causal)
                ids, tokens = [], 0
                for j in selected[first + i, h].tolist():
                    if 0 <= j < len(table[b]) and j * page <= lim and 0 <= table[b][j] < pages:
                        ids.append(table[b][j])
                        assert tokens % page == 0, "the page that ends inside is not the last"
                        tokens += min(page, lim + 1 - j * page)
                tables[first + i], lens[first + i] = ids, tokens
        out.append((tables, lens))
    return out


def mass(q, lse, cache, before, table, starts, lengths, scale, causal=True, max_new=1 << 30):
    """(mass, what was added, bound of an fp32 sum's error)."""
    kc, ks = cache[:2]
    pages, hkv, page, d = kc.shape
    t, hq, _ = q.shape
    g = hq // hkv
    out, added, off = before.double().clone(), torch.zeros(before.shape, dtype=torch.float64), \
        torch.zeros(before.shape, dtype=torch.float64)
    for b in range(len(lengths)):
        first, count, n = ref.rows_of(starts, lengths, t, b, len(table[b]) * page)
        if not count:
            continue
        out[b, :, max(n - count, 0):n] = 0
        rows = min(count, max_new)
        for pos in range(n):
            p = ref.page_at(table, pages, page, b, pos)
            if p is None:
                continue
            i0 = next((i for i in range(rows) if last_seen(n, count, i, causal) >= pos), rows)
            if i0 == rows:
                continue
            x = q[first + i0:first + rows].double().reshape(-1, hkv, g, d)
            k = kc[p, :, pos % page].double() * ks[p, :, pos % page].double()[:, None]
            s = (x * k[:, None]).sum(-1) * scale  # [rows,hkv,g]
            size = (x * k[:, None]).abs().sum(-1) * abs(scale)
            z = lse[first + i0:first + rows].double().reshape(-1, hkv, g)
            w = torch.where(z == -math.inf, 0.0, torch.exp(s - z))
            z = torch.where(z == -math.inf, 0.0, z)
            # (d + 8) fp32 steps of the score, three of it and of lse in log2 units, exp2's
            e = (d + 8) * 2.0 ** -24 * size + 2.0 ** -22 * (s.abs() + z.abs()) + 2.0 ** -21
            added[b, :, pos] = w.sum((0, 2))
            off[b, :, pos] = (w * e * 1.01).sum((0, 2)) + w.sum((0, 2)) * (rows * g + 4) * 2.0 ** -24
    return out + added, added, off + 2.0 ** -23 * (out + added).abs() + 2.0 ** -140


def evict(table, lengths, count, pages, page):
    """(table, lengths, missing) after rows of more than `count` keep that many."""
    width = len(table[0]) if table else 0
    rows = [ref.held(table, lengths, b, pages, page) for b in range(len(table))]
    holds = {}
    for _, r in rows:
        for p in r:
            if p is not None:
                holds[p] = holds.get(p, 0) + 1
    free = [p for p in range(pages) if p not in holds]
    out, after, given = [], [], 0
    for n, r in rows:
        if n > count:
            r, n = list(r[: -(-count // page)]), count
            for j, p in enumerate(r):
                if p is not None and holds[p] > 1:
                    r[j] = free[given] if given < len(free) else None
                    given += 1
        out.append([-1 if p is None else p for p in r] + [-1] * (width - len(r)))
        after.append(n)
    missing = max(0, given - len(free))
    if missing:
        out = [[-1 if p is None else p for p in r] + [-1] * (width - len(r)) for _, r in rows]
        after = [n for n, _ in rows]
    return out, after, missing


def moved(cache, mass, keep, table, lengths, new_table, new_lengths):
    """(cache, mass) after it, CPU copies: a pool [layers,...] of them."""
    pages, _, page, _ = cache[0].shape[1:]
    out, m = [c.clone() for c in cache], None if mass is None else mass.clone()
    layers, _, hkv, count = keep.shape
    for b in range(len(lengths)):
        n = min(max(lengths[b], 0), len(table[b]) * page)
        if new_lengths[b] == n:
            continue
        for layer in range(layers):
            for h in range(hkv):
                for i in range(count):
                    k = int(keep[layer, b, h, i])
                    k = i if k < i or k >= n else k
                    p, to = table[b][k // page], new_table[b][i // page]
                    if mass is not None:
                        m[layer, b, h, i] = mass[layer, b, h, k]
                    if not 0 <= to < pages or (p == to and k == i):
                        continue
                    for c, (x, y) in enumerate(zip(cache, out)):
                        y[layer, to, h, i % page] = x[layer, p, h, k % page] if 0 <= p < pages \
                            else c % 2  # codes 0, scales 1
    return out, m
