"""The paged cache's append, forking and compacting against the plain forms
(equal, every byte of the pool included), and all of its operators together."""

import random

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


def _ints(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _same(cache, want):
    for name, a, b in zip(("k codes", "k scales", "v codes", "v scales"), cache, want):
        assert torch.equal(a.cpu(), b), name


# --- append ------------------------------------------------------------------

@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lengths,news,hkv,d,page", [
    ([1], [1], 1, 64, 16),
    ([200, 17, 64, 65, 5], [1, 1, 1, 1, 0], 8, 128, 64),
    ([100, 3, 40], [33, 3, 40], 4, 256, 16),
    ([70] * 40, [2] * 40, 2, 64, 32),
    ([900], [900], 3, 128, 1024),
])
def test_append(gpu, lengths, news, hkv, d, page, dtype):
    import sparkq

    _, k, v, cache, table, starts = ref.batch(1, lengths, news, hkv, hkv, d, page, extra_rows=2)
    k, v = k.to(dtype), v.to(dtype)
    k[0, 0] = 0  # a zero row has scale 1
    dev = tuple(t.to(gpu) for t in cache)
    sparkq.paged_kv_append(k.to(gpu), v.to(gpu), dev, _ints(table, gpu), _ints(starts, gpu),
                           _ints(lengths, gpu))
    _same(dev, ref.append(k, v, cache, table, starts, lengths))


def test_append_skips_what_has_no_place(gpu):
    """Absent and out-of-range pages, more rows than tokens, rows behind the
    last sequence, starts out of range, and a length past the table's row."""
    import sparkq

    lengths, news = [40, 20, 3, 64], [10, 5, 3, 6]
    _, k, v, cache, table, starts = ref.batch(2, lengths, news, 2, 2, 64, 16, extra_rows=4)
    table[0][2] = -1
    table[1][1] = 10 ** 9
    lengths[2] = 1        # 3 rows, one token
    lengths[3] = 1000     # its row of pages holds 64
    dev = tuple(t.to(gpu) for t in cache)
    sparkq.paged_kv_append(k.to(gpu), v.to(gpu), dev, _ints(table, gpu), _ints(starts, gpu),
                           _ints(lengths, gpu))
    _same(dev, ref.append(k, v, cache, table, starts, lengths))
    assert any(not torch.equal(a.cpu(), b) for a, b in zip(dev, cache))
    bad = [-5, 10, 12, 12, 10 ** 6]
    dev = tuple(t.to(gpu) for t in cache)
    sparkq.paged_kv_append(k.to(gpu), v.to(gpu), dev, _ints(table, gpu), _ints(bad, gpu),
                           _ints(lengths, gpu))
    _same(dev, ref.append(k, v, cache, table, bad, lengths))


def test_append_reads_views_and_writes_strided_pools(gpu):
    """Keys and values as views of a packed projection, a table with a wider
    row stride, and a pool whose layers lie between its pages."""
    import sparkq

    lengths, news = [50, 9], [20, 9]
    _, k, v, cache, table, starts = ref.batch(3, lengths, news, 4, 4, 128, 32)
    t = k.shape[0]
    qkv = torch.randn((t, 16, 128)).to(torch.bfloat16)
    qkv[:, 8:12], qkv[:, 12:] = k.to(torch.bfloat16), v.to(torch.bfloat16)
    wide = torch.full((2, 9), 77, dtype=torch.int32)
    wide[:, :2] = torch.tensor(table)
    pages = cache[0].shape[0]
    dev = []
    for c in cache:  # [pages, 3 layers, ...]: the middle one is the cache
        buf = torch.zeros((pages, 3, *c.shape[1:]), dtype=c.dtype, device=gpu)
        buf[:, 1] = c.to(gpu)
        dev.append(buf)
    g = qkv.to(gpu)
    sparkq.paged_kv_append(g[:, 8:12], g[:, 12:], tuple(b[:, 1] for b in dev), wide.to(gpu)[:, :2],
                           _ints(starts, gpu), _ints(lengths, gpu))
    want = ref.append(qkv[:, 8:12], qkv[:, 12:], cache, table, starts, lengths)
    _same([b[:, 1] for b in dev], want)
    assert all(not b[:, 0].any() and not b[:, 2].any() for b in dev)


# --- fork and compact --------------------------------------------------------

def _case(seed, b, page, width, pages, most, sharing):
    """A batch whose rows share prefixes: row i may start with pages of an
    earlier row, in the middle of a page or not."""
    rng = random.Random(seed)
    table, lengths, free = [], [], list(range(pages))
    rng.shuffle(free)
    for i in range(b):
        n = rng.randint(0, most)
        row = []
        if table and rng.random() < sharing:
            j = rng.randrange(len(table))
            n = rng.choice([lengths[j], min(n, lengths[j])])
            row = table[j][: -(-n // page)]
        while len(row) < -(-n // page) and free:
            row.append(free.pop())
        n = min(n, len(row) * page)
        table.append(row + [-1] * (width - len(row)))
        lengths.append(n)
    return rng, table, lengths


def _pool_on(gpu, seed, layers, pages, hkv, page, d):
    gen = torch.Generator().manual_seed(seed)
    cpu = ref.pool(gen, pages, hkv, page, d, layers)
    return cpu, tuple(t.to(gpu) for t in cpu)


def _moved(cpu, pairs):
    """The pool with the pages copied, all sources read first."""
    out = [t.clone() for t in cpu]
    for a, b in pairs:
        for new, old in zip(out, cpu):
            new[:, b] = old[:, a]
    return out


@pytest.mark.parametrize("seed,b,page,width,pages,most", [
    (0, 1, 16, 1, 2, 16), (1, 8, 32, 6, 60, 100), (2, 50, 16, 12, 300, 150),
    (3, 7, 64, 3, 20, 192), (4, 300, 16, 4, 700, 60), (5, 1300, 16, 2, 1500, 30),
    (6, 20, 128, 4, 2500, 500),
    (7, 40, 16, 3, 16384, 40), (8, 40, 16, 90, 17000, 1400)])
@pytest.mark.parametrize("reorder", [False, True])
def test_fork(gpu, seed, b, page, width, pages, most, reorder):
    import sparkq

    rng, table, lengths = _case(seed, b, page, width, pages, most, 0.5)
    rows = b + 3 if reorder else b
    parents = [rng.choice([-1, b, *range(b)]) for _ in range(rows)] if reorder else None
    fresh = [rng.choice([0, 1, 1, rng.randint(0, 2 * page), -2]) for _ in range(rows)]
    if b > 3:
        table[2][0] = rng.choice([-1, pages, 10 ** 9])
    want_t, want_n, missing, pairs = ref.fork(
        table, lengths, parents if reorder else range(b), fresh, pages, page)
    cpu, dev = _pool_on(gpu, seed, 2, pages, 1, page, 64)
    got = sparkq.kv_pages_fork(dev, _ints(table, gpu), _ints(lengths, gpu),
                               _ints(parents, gpu) if reorder else None, _ints(fresh, gpu))
    print(f"[fork] rows={rows} copies={len(pairs)} missing={missing}", flush=True)
    assert got[2].tolist() == [missing]
    assert got[1].tolist() == want_n
    assert got[0].tolist() == want_t
    _same(dev, _moved(cpu, pairs))


def test_fork_short_of_pages_changes_nothing(gpu):
    import sparkq

    table, lengths = [[0, 1, -1], [0, 2, -1]], [24, 24]
    cpu, dev = _pool_on(gpu, 9, 1, 4, 1, 16, 64)
    for parents, fresh, missing in ([0, 0, 1], [1, 1, 1], 0), ([0, 0, 1], [9, 9, 9], 3):
        want = ref.fork(table, lengths, parents, fresh, 4, 16)
        got = sparkq.kv_pages_fork(dev, _ints(table, gpu), _ints(lengths, gpu),
                                   _ints(parents, gpu), _ints(fresh, gpu))
        assert want[2] == missing and got[2].item() == missing
        assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
        _same(dev, _moved(cpu, want[3]))
        assert bool(want[3]) == (missing == 0)
        cpu = tuple(t.cpu() for t in dev)


@pytest.mark.parametrize("seed,b,page,width,pages,most", [
    (0, 1, 16, 1, 2, 16), (1, 8, 32, 6, 60, 100), (2, 50, 16, 12, 500, 150),
    (3, 0, 16, 2, 5, 0), (4, 300, 16, 4, 3000, 60), (5, 5, 1024, 2, 30, 2000),
    (6, 1100, 16, 3, 16384, 40), (7, 40, 16, 90, 17000, 1400)])
def test_compact(gpu, seed, b, page, width, pages, most):
    import sparkq

    rng, table, lengths = _case(seed, b, page, width, pages, most, 0.3)
    if b > 3:
        table[1][0] = rng.choice([-1, pages, 10 ** 9])
    want, used, pairs = ref.compact(table, lengths, pages, page)
    cpu, dev = _pool_on(gpu, seed, 3, pages, 1, page, 64)
    at = _ints(table, gpu) if b else torch.zeros((0, width), dtype=torch.int32, device=gpu)
    got, count = sparkq.kv_pages_compact(dev, at, _ints(lengths, gpu))
    print(f"[compact] used={used} moved={len(pairs)}", flush=True)
    assert count.tolist() == [used] and got.tolist() == want
    _same(dev, _moved(cpu, pairs))


def test_one_layer_and_pages_between_other_data(gpu):
    """A cache of one layer without the layer axis, and a pool whose pages
    hold the layers: [pages, layers, ...] seen as [layers, pages, ...]."""
    import sparkq

    table, lengths = [[5, 7], [5, -1]], [40, 20]
    want, used, pairs = ref.compact(table, lengths, 9, 32)
    gen = torch.Generator().manual_seed(1)
    one = ref.pool(gen, 9, 2, 32, 128)
    dev = tuple(t.to(gpu) for t in one)
    got, _ = sparkq.kv_pages_compact(dev, _ints(table, gpu), _ints(lengths, gpu))
    assert got.tolist() == want and len(pairs) == 2
    for a, c in zip(dev, one):
        w = c.clone()
        for x, y in pairs:
            w[y] = c[x]
        assert torch.equal(a.cpu(), w)
    cpu = ref.pool(gen, 9, 2, 32, 128, layers=4)
    store = [t.transpose(0, 1).contiguous().to(gpu) for t in cpu]
    got, _ = sparkq.kv_pages_compact(tuple(t.transpose(0, 1) for t in store), _ints(table, gpu),
                                     _ints(lengths, gpu))
    assert got.tolist() == want
    _same([t.transpose(0, 1) for t in store], _moved(cpu, pairs))


# --- a run of them together --------------------------------------------------

def test_a_serving_run(gpu):
    """Prompts of different lengths, a fork, decode steps, a dropped sequence
    and a compaction, in two layers. Each attention is held to the float64 form
    over the cache that the device holds, and the pool's codes of each
    sequence to its own tokens quantized."""
    import sparkq

    from test_gpu_paged_sdpa import check

    hq, hkv, d, page = 8, 2, 128, 16
    cache = sparkq.PagedKVCache(2, 40, hkv, d, page_size=page, max_pages=8, batch=3, device=gpu)
    gen = torch.Generator().manual_seed(5)
    told = [[[] for _ in range(3)] for _ in range(2)]  # per layer and row: rotated (k, v) rows
    wq, wk = (torch.ones(d, dtype=torch.bfloat16, device=gpu) for _ in range(2))

    def step(news, parents=None):
        nonlocal told
        starts = cache.step(news, parents)
        assert cache.missing.item() == 0
        if parents is not None:
            told = [[list(rows[p]) if p >= 0 else [] for p in parents] for rows in told]
        t, at = sum(news), starts.tolist()
        lengths = cache.lengths.tolist()
        pos = torch.cat([torch.arange(n - k, n, dtype=torch.int32)
                         for n, k in zip(lengths, news)]).to(gpu)
        for layer in range(2):
            qkv = torch.randn((t, hq + 2 * hkv, d), generator=gen).to(torch.bfloat16).to(gpu)
            q, k = sparkq.qk_norm_rope(qkv[:, :hq], qkv[:, hq:hq + hkv], wq, wk, pos, dims=d,
                                       eps=1e-6)
            v = qkv[:, hq + hkv:]
            cache.append(layer, k, v)
            out = cache.attend(layer, q, scale=d ** -0.5)
            mine = tuple(c.cpu() for c in cache.layer(layer))
            table = cache.page_table.tolist()
            check(out, q.cpu(), mine, table, at, lengths, d ** -0.5)
            for i, n in enumerate(lengths):
                rows = told[layer][i]
                rows += [(k[j].cpu(), v[j].cpu()) for j in range(at[i], at[i + 1])]
                assert len(rows) == n
                for j, (kr, vr) in enumerate(rows):
                    for x, c, s in ((kr, mine[0], mine[1]), (vr, mine[2], mine[3])):
                        codes, sc = ref.quantize(x)
                        p = table[i][j // page]
                        assert torch.equal(c[p, :, j % page], codes)
                        assert torch.equal(s[p, :, j % page], sc)

    step([37, 5, 16])
    step([1, 1, 1])
    step([1, 1, 1, 2], [0, 0, 2, 1])   # two go on from row 0, in the middle of a page
    step([1, 0, 1, 1])
    step([1, 20, 1], [3, 1, -1])       # two end, one starts
    used = cache.compact().item()
    pages = [p for r, n in zip(cache.page_table.tolist(), cache.lengths.tolist())
             for p in r[: -(-n // page)]]
    assert sorted(set(pages)) == list(range(used))
    step([1, 1, 30])
