"""Bounds and scores of pages, selection, attention over selected pages, gathered
weights and eviction against their float64 forms, one operator at a time.

Tolerances. Bounds, places and moved tokens are exact. A score is an fp32 sum of 2 D
exact products (4 D of fp16 queries, which go in as two parts), times the scale:
(4 D + 2) 2^-24 of |scale| sum |q||bound|. Attention over selected pages: what
test_gpu_paged_sdpa says of few rows. The logarithm of a row's sum: the scores'
(D + 8) 2^-24 of `size`, exp2's and log2's 2^-20, n 2^-24 of an fp32 sum of n, and
its own three roundings. Gathered weights: beside their form."""

import math
import random

import pytest
import torch

import paged_long_reference as long
import paged_reference as ref
from test_gpu_paged_sdpa import HEADS, check

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16
BATCHES = [([1], [1], 16), ([33, 70], [33, 0], 16), ([130, 5, 64, 300], [130, 1, 0, 17], 64),
           ([257], [100], 32), ([90, 90, 200], [4, 3, 1], 128), ([1500, 20], [1, 1], 1024),
           ([700, 64, 65, 1, 63], [1, 1, 1, 1, 1], 64)]


def _ints(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _gpu(gpu, table, starts, lengths):
    return _ints(table, gpu), _ints(starts, gpu), _ints(lengths, gpu)


# --- bounds ----------------------------------------------------------------------

@pytest.mark.parametrize("hkv,d", [(8, 128), (4, 256), (1, 64), (5, 64)])
@pytest.mark.parametrize("lengths,news,page", BATCHES)
def test_bounds(gpu, hkv, d, lengths, news, page):
    import sparkq

    _, _, _, cache, table, starts = ref.batch(d, lengths, news, hkv, hkv, d, page)
    cache[1][0, 0, 0] = -0.01  # (not what a quantizer makes)
    before = torch.randn((cache[0].shape[0], hkv, 2, d)).bfloat16()
    got = before.to(gpu)
    sparkq.paged_key_bounds(tuple(t.to(gpu) for t in cache), got, *_gpu(gpu, table, starts, lengths),
                            max_new=max(news))
    assert torch.equal(got.cpu(), long.bounds(cache, before, table, starts, lengths))


@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_bounds_of_keys_that_are_not_finite(gpu, bad):
    """And none from the slots behind a sequence's end, or from absent pages."""
    import sparkq

    lengths, news = [70, 40], [70, 40]
    _, _, _, cache, table, starts = ref.batch(3, lengths, news, 2, 2, 64, 32)
    cache[1][table[0][1], 0, 5] = bad
    cache[1][table[0][2], :, 7:] = bad  # behind the end
    table[1][0] = 10 ** 9
    before = torch.zeros((cache[0].shape[0], 2, 2, 64)).bfloat16()
    got = before.to(gpu)
    sparkq.paged_key_bounds(tuple(t.to(gpu) for t in cache), got, *_gpu(gpu, table, starts, lengths),
                            max_new=100)
    want = long.bounds(cache, before, table, starts, lengths)
    assert want.isfinite().all() and torch.equal(got.cpu(), want)
    assert (want[table[0][1], 0, 1] == long.BIG).all()


def test_bounds_in_strided_tensors_and_of_odd_batches(gpu):
    """Starts that descend, lengths below and past what there is, layers of a pool,
    bounds as a view: the same pages, and nothing else is written."""
    import sparkq

    pool = ref.pool(torch.Generator().manual_seed(4), 9, 3, 16, 64, layers=2)
    table = [[0, 1, 2], [3, -1, 4], [5, 6, 7], [8, 8, 8]]
    starts, lengths = [0, 7, 3, 40, 41], [30, 48, 1000, -5]
    wide = torch.full((9, 2, 3, 2, 64), 7.0, dtype=BF, device=gpu)
    sparkq.paged_key_bounds(tuple(t[1].to(gpu) for t in pool), wide[:, 1],
                            *_gpu(gpu, table, starts, lengths), max_new=48)
    cache = tuple(t[1] for t in pool)
    want = long.bounds(cache, torch.full((9, 3, 2, 64), 7.0, dtype=BF), table, starts, lengths)
    assert torch.equal(wide[:, 1].cpu(), want) and (wide[:, 0] == 7.0).all()


# --- scores ----------------------------------------------------------------------

def check_scores(got, seen, q, bnd, table, starts, lengths, page, scale, causal=True, max_new=1 << 30):
    want, size, n, done = long.scores(q, bnd, table, starts, lengths, page, scale, causal, max_new)
    got, seen = got.cpu().double(), seen.cpu()
    assert torch.equal(seen[done], n[done])
    hidden = want == -math.inf
    assert (got[done][hidden[done]] == -math.inf).all()
    tol = (4 * q.shape[-1] + 2) * 2.0 ** -24 * size + 2.0 ** -140
    off = ((got - want).abs() / tol)[done][~hidden[done]]
    worst = off.max().item() if off.numel() else 0.0
    print(f"[scores] {tuple(got.shape)} largest error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0
    return done


def _bounds(gen, pages, hkv, d):
    mid, half = torch.randn((pages, hkv, 1, d), generator=gen), torch.rand((pages, hkv, 1, d), generator=gen)
    return torch.cat([mid - half, mid + half], 2).bfloat16()


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lengths,news,page", BATCHES)
@pytest.mark.parametrize("dtype", [BF, F16])
def test_scores(gpu, hq, hkv, d, lengths, news, page, dtype):
    import sparkq

    q, _, _, cache, table, starts = ref.batch(d + 2, lengths, news, hq, hkv, d, page)
    q = q.to(dtype)
    bnd = _bounds(torch.Generator().manual_seed(d), cache[0].shape[0], hkv, d)
    got, seen = sparkq.paged_page_scores(q.to(gpu), bnd.to(gpu), *_gpu(gpu, table, starts, lengths),
                                         page_size=page, scale=d ** -0.5, max_new=max(news))
    assert got.shape == (q.shape[0], hkv, len(table[0])) and seen.dtype == torch.int32
    assert check_scores(got, seen, q, bnd, table, starts, lengths, page, d ** -0.5).all()


@pytest.mark.parametrize("new", [1, 5])
@pytest.mark.parametrize("scale", [0.0, -0.3, 2])
@pytest.mark.parametrize("causal", [True, False])
def test_scores_scales_masks_and_absent_pages(gpu, new, scale, causal):
    """Queries as a view of a packed projection, zeros among them, sequences with more
    new tokens than max_new, rows of none."""
    import sparkq

    lengths, news, page = [300, 0, 40, 2000], [new, 0, new + 3, new], 16
    q, _, _, cache, table, starts = ref.batch(5, lengths, news, 12, 2, 128, page, extra_rows=3, width=131)
    table[0][2], table[3][100] = -1, 10 ** 9
    packed = torch.zeros((q.shape[0], 20, 128), dtype=F16)
    packed[:, 4:16] = q.to(F16)
    packed[0, 4:10] = 0
    packed[:, 5, ::3] = -0.0
    bnd = _bounds(torch.Generator().manual_seed(6), cache[0].shape[0], 2, 128)
    kw = {"page_size": page, "scale": scale, "max_new": new, "mask": "causal" if causal else None}
    at = _gpu(gpu, table, starts, lengths)
    got, seen = sparkq.paged_page_scores(packed.to(gpu)[:, 4:16], bnd.to(gpu), *at, **kw)
    done = check_scores(got, seen, packed[:, 4:16], bnd, table, starts, lengths, page, scale, causal, new)
    assert done.sum() == 3 * new


def test_scores_bound_every_logit(gpu):
    """Bounds from the operator: no logit of a row is above its page's score."""
    import sparkq

    lengths, news, page = [400, 77], [9, 1], 32
    q, _, _, cache, table, starts = ref.batch(9, lengths, news, 8, 2, 64, page)
    q = q.to(BF)
    dev = tuple(t.to(gpu) for t in cache)
    bnd = torch.zeros((cache[0].shape[0], 2, 2, 64), dtype=BF, device=gpu)
    whole = _gpu(gpu, table, [0, 400, 477], lengths)  # all tokens as new ones
    sparkq.paged_key_bounds(dev, bnd, *whole, max_new=400)
    got, _ = sparkq.paged_page_scores(q.to(gpu), bnd, *_gpu(gpu, table, starts, lengths),
                                      page_size=page, scale=0.125, max_new=9)
    got = got.cpu().double()
    for b, n in enumerate(lengths):
        for r in range(starts[b], starts[b + 1]):
            for pos in range(n - (starts[b + 1] - r) + 1):
                p = table[b][pos // page]
                k = cache[0][p, :, pos % page].double() * cache[1][p, :, pos % page].double()[:, None]
                logit = (q[r].double().reshape(2, 4, 64) * k[:, None]).sum(-1).amax(1) * 0.125
                assert (got[r, :, pos // page] >= logit - 1e-4).all()


@pytest.mark.parametrize("new", [1, 3])
def test_scores_of_values_that_are_not_finite(gpu, new):
    """A head with a NaN does not count, infinite queries and the largest bounds give
    infinite scores."""
    import sparkq

    q, _, _, cache, table, starts = ref.batch(10, [64], [new], 4, 1, 64, 16)
    for dtype in (BF, F16):
        x = q.to(dtype)
        x[0, 1, 5] = math.nan
        bnd = _bounds(torch.Generator().manual_seed(1), cache[0].shape[0], 1, 64)
        bnd[table[0][1], 0, 0], bnd[table[0][1], 0, 1] = -long.BIG, long.BIG
        at = _gpu(gpu, table, starts, [64])
        kw = {"page_size": 16, "scale": 1.0, "max_new": new}
        got, _ = sparkq.paged_page_scores(x.to(gpu), bnd.to(gpu), *at, **kw)
        less, _ = sparkq.paged_page_scores(x[:, [0, 2, 3, 3]].to(gpu), bnd.to(gpu), *at, **kw)
        assert torch.equal(got[0], less[0]) and (got[:, :, 1] == math.inf).all()
        assert not got.isnan().any()
        x[0] = math.nan
        got, _ = sparkq.paged_page_scores(x.to(gpu), bnd.to(gpu), *at, **kw)
        assert (got[0] == -math.inf).all()
        x[0, 2], x[0, 2, 7] = 0, math.inf
        bnd[:, :, 0], bnd[:, :, 1] = -1, 2
        got, _ = sparkq.paged_page_scores(x.to(gpu), bnd.to(gpu), *at, **kw)
        assert (got[0] == math.inf).all()


# --- selection -------------------------------------------------------------------

@pytest.mark.parametrize("n", [1, 2, 63, 64, 65, 256, 257, 512, 700, 1024, 1025, 4096, 4097, 9000,
                               20000])
@pytest.mark.parametrize("kind", ["normal", "ties", "equal", "odd"])
def test_select(gpu, n, kind):
    import sparkq

    rng, gen = random.Random(n), torch.Generator().manual_seed(n)
    layers, rows, heads = 2, 3, 2
    x = torch.randn((layers, rows, heads, n), generator=gen)
    if kind == "ties":
        x = torch.round(2 * x) / 2
    elif kind == "equal":
        x = torch.full_like(x, -0.0)
        x[..., ::2] = 0.0
    elif kind == "odd":
        for v in (math.nan, math.inf, -math.inf, -0.0, 1e-45, -1e-45, 3.4e38):
            x[torch.rand(x.shape, generator=gen) < 0.1] = v
        x[0, 0] = math.nan
    lengths = [n, n // 2, rng.randint(0, n)]
    for count in sorted({1, n // 3 + 1, n, n + 5}):
        first = rng.randint(0, min(2, count))
        last = rng.randint(0, min(9, count - first))
        got = sparkq.select_top(x.to(gpu), count, lengths=_ints(lengths, gpu), first=first, last=last)
        assert got.dtype == torch.int32
        assert torch.equal(got.cpu(), long.select(x, count, lengths, first, last)), (count, first, last)
    got = sparkq.select_top(x[1].to(gpu), min(n, 3))
    assert torch.equal(got.cpu(), long.select(x[1:], min(n, 3))[0])


@pytest.mark.parametrize("n,count", [(40000, 1), (40000, 33333), (131072, 2048)])
def test_select_of_rows_longer_than_registers_hold(gpu, n, count):
    import sparkq

    x = torch.randn((1, 2, 1, n), generator=torch.Generator().manual_seed(n))
    x[:, 1] = torch.round(x[:, 1] * 8)
    got = sparkq.select_top(x.to(gpu), count, lengths=_ints([n, n - 77], gpu), first=1, last=0)
    assert torch.equal(got.cpu(), long.select(x, count, [n, n - 77], 1, 0))


def test_select_in_views_and_of_lengths_out_of_range(gpu):
    import sparkq

    x = torch.randn((4, 3, 2, 500), generator=torch.Generator().manual_seed(2))
    big = x.to(gpu)
    lengths = [-3, 10 ** 9, 7]
    view = big.transpose(0, 1)[..., 100:400]  # [3 layers, 4 rows, ...]
    got = sparkq.select_top(view, 9, lengths=_ints([*lengths, 300], gpu), first=2, last=3)
    want = long.select(x.transpose(0, 1)[..., 100:400], 9, [*lengths, 300], 2, 3)
    assert torch.equal(got.cpu(), want) and (want[:, 0] == -1).all()
    assert sparkq.select_top(big[:0], 5).shape == (0, 3, 2, 5)
    assert sparkq.select_top(big[:, :0], 5, lengths=_ints([], gpu)).shape == (4, 0, 2, 5)


# --- attention over selected pages -------------------------------------------------

def _lists(rng, table, starts, lengths, page, hkv, count, t):
    """Ascending lists of distinct pages that a row may or may not see."""
    out = torch.full((t, hkv, count), -1, dtype=torch.int32)
    for b, n in enumerate(lengths):
        own = -(-n // page)
        for r in range(starts[b], starts[b + 1]):
            for h in range(hkv):
                k = rng.randint(0, min(count, own))
                pick = sorted(rng.sample(range(own), k))
                out[r, h, :k] = torch.tensor(pick, dtype=torch.int32)
    return out


def check_sparse(got, q, cache, selected, table, starts, lengths, scale, causal=True, max_new=1 << 30):
    pages, hkv, page, _ = cache[0].shape
    g = q.shape[1] // hkv
    done = None
    for h, (tables, lens) in enumerate(long.listed(selected, table, starts, lengths, pages, page,
                                                   causal, max_new)):
        done = [r for r, n in enumerate(lens) if n is not None]
        width = max([1] + [len(tables[r]) for r in done])
        rows = [tables[r] + [-1] * (width - len(tables[r])) for r in done]
        part = slice(h * g, (h + 1) * g)
        check(got[done][:, part], q[done][:, part], tuple(c[:, h:h + 1] for c in cache), rows,
              list(range(len(done) + 1)), [lens[r] for r in done], scale)
    return done


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lengths,news,page", [*BATCHES, ([3000], [2], 16)])
@pytest.mark.parametrize("dtype", [BF, F16])
def test_sparse(gpu, hq, hkv, d, lengths, news, page, dtype):
    import sparkq

    q, _, _, cache, table, starts = ref.batch(d + 5, lengths, news, hq, hkv, d, page)
    q = q.to(dtype)
    sel = _lists(random.Random(d), table, starts, lengths, page, hkv, min(len(table[0]), 41), q.shape[0])
    out = sparkq.paged_sparse_sdpa(q.to(gpu), tuple(t.to(gpu) for t in cache), sel.to(gpu),
                                   *_gpu(gpu, table, starts, lengths), scale=d ** -0.5,
                                   max_new=max(news))
    assert out.dtype == dtype
    assert len(check_sparse(out, q, cache, sel, table, starts, lengths, d ** -0.5)) == q.shape[0]


@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("new", [1, 6])
def test_sparse_lists_of_all_kinds(gpu, causal, new):
    """Pages past what a row sees, outside its table, absent, named twice; lists that
    name nothing; rows past max_new and of no sequence keep what out holds; queries
    and lists as views."""
    import sparkq

    lengths, news, page = [200, 50, 0, 90], [new, new + 2, 0, new], 32
    q, _, _, cache, table, starts = ref.batch(12, lengths, news, 6, 2, 128, page, extra_rows=2, width=9)
    q = q.to(BF)
    table[0][3] = -1
    t = q.shape[0]
    sel = _lists(random.Random(3), table, starts, lengths, page, 2, 7, t)
    sel[0, 0] = torch.tensor([-7, 0, 0, 1, 3, 10 ** 9, 6])  # (page 6 ends inside)
    sel[0, 1] = -1
    wide = torch.zeros((t, 3, 11), dtype=torch.int32)
    wide[:, 1:, 2:9] = sel
    packed = torch.zeros((t, 9, 128), dtype=BF)
    packed[:, 2:8] = q
    out = torch.full((t, 6, 128), 7.0, dtype=torch.float32, device=gpu)
    kw = {"scale": 0.1, "max_new": new, "mask": "causal" if causal else None}
    got = sparkq.paged_sparse_sdpa(packed.to(gpu)[:, 2:8], tuple(x.to(gpu) for x in cache),
                                   wide.to(gpu)[:, 1:, 2:9], *_gpu(gpu, table, starts, lengths), out=out,
                                   out_dtype=torch.float32, **kw)
    assert got.data_ptr() == out.data_ptr()
    done = check_sparse(out, q, cache, sel, table, starts, lengths, 0.1, causal, new)
    rest = [r for r in range(t) if r not in done]
    assert len(rest) == 4 and (out[rest] == 7.0).all()
    assert (out[0, 3:] == 0).all()


def test_sparse_over_all_pages_is_the_attention(gpu):
    """Long lists (more than are looked up at a time), split over the chip."""
    import sparkq

    lengths, news, page = [16 * 1300 - 5, 100], [1, 1], 16
    q, _, _, cache, table, starts = ref.batch(13, lengths, news, 8, 2, 64, page)
    q = q.to(F16)
    sel = torch.arange(1300, dtype=torch.int32).expand(2, 2, -1).contiguous()
    dev, at = tuple(t.to(gpu) for t in cache), _gpu(gpu, table, starts, lengths)
    for rows in (1, 300):  # few rows split a list, many take it in pieces
        x = q.repeat_interleave(rows, 0)
        s = sel.repeat_interleave(rows, 0)
        tab = at[0].repeat_interleave(rows, 0)
        n = at[2].repeat_interleave(rows, 0)
        st = torch.arange(2 * rows + 1, dtype=torch.int32, device=gpu)
        got = sparkq.paged_sparse_sdpa(x.to(gpu), dev, s.to(gpu), tab, st, n, scale=0.125, max_new=1,
                                       out_dtype=torch.float32)
        check(got[[0, rows]], q, cache, table, starts, lengths, 0.125)
        assert torch.equal(got[:rows], got[:1].expand(rows, -1, -1))


@pytest.mark.parametrize("d", [64, 256])
def test_sparse_values_in_any_order_and_hidden_ones(gpu, d):
    """Value scales over fp16's range, of 1 with nothing but zeros, and not finite where
    no row looks."""
    import sparkq

    lengths, news, page = [300, 280], [1, 1], 32
    q, _, _, cache, table, starts = ref.batch(21, lengths, news, 8, 2, d, page)
    for b, n in enumerate(lengths):
        for pos in range(n):
            cache[3][table[b][pos // page], :, pos % page] = 2.0 ** (-24 + (pos if b else n - 1 - pos) * 39 / n)
    cache[2][table[0][2], :, 3] = 0
    cache[3][table[0][2], :, 3] = 1.0
    cache[3][table[1][4]] = math.nan
    cache[1][table[1][4]] = math.inf
    cache[3][table[0][300 // page], :, 300 % page:] = math.inf
    q = q.to(BF)
    sel = torch.tensor([[0, 2, 5, 9], [0, 1, 7, 8]], dtype=torch.int32)[:, None].expand(2, 2, 4).contiguous()
    out = sparkq.paged_sparse_sdpa(q.to(gpu), tuple(t.to(gpu) for t in cache), sel.to(gpu),
                                   *_gpu(gpu, table, starts, lengths), scale=d ** -0.5, max_new=1,
                                   out_dtype=torch.float32)
    check_sparse(out, q, cache, sel, table, starts, lengths, d ** -0.5)


# --- the logarithm of a row's sum, and gathered weights -----------------------------

def _lse(q, cache, table, starts, lengths, scale, causal=True):
    """[T,Hq] float64 and the bound of its error."""
    kc, ks = cache[:2]
    pages, hkv, page, d = kc.shape
    t, hq, _ = q.shape
    out = torch.full((t, hq), -math.inf, dtype=torch.float64)
    tol = torch.zeros((t, hq), dtype=torch.float64)
    for b in range(len(lengths)):
        first, count, n = ref.rows_of(starts, lengths, t, b, len(table[b]) * page)
        at = [(ref.page_at(table, pages, page, b, p), p) for p in range(n)]
        at = [x for x in at if x[0] is not None]
        ids = torch.tensor([x[0] for x in at], dtype=torch.long)
        pos = torch.tensor([x[1] for x in at], dtype=torch.long)
        k = kc[ids, :, pos % page].double() * ks[ids, :, pos % page].double()[..., None]
        for i in range(count):
            see = pos <= long.last_seen(n, count, i, causal)
            if not bool(see.any()):
                continue
            x = q[first + i].double().reshape(hkv, -1, d)
            s = torch.einsum("hgd,nhd->hgn", x, k[see]).reshape(hq, -1) * scale
            size = (torch.einsum("hgd,nhd->hgn", x.abs(), k[see].abs()).reshape(hq, -1) * abs(scale)).amax(-1)
            out[first + i] = torch.logsumexp(s, -1)
            tol[first + i] = (d + 8) * 2.0 ** -24 * size + 2.0 ** -20 + int(see.sum()) * 2.0 ** -24 \
                + 3 * 2.0 ** -24 * (out[first + i].abs() + size)
    return out, tol


@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 128), (16, 4, 256), (8, 8, 64), (5, 5, 256), (32, 1, 64)])
@pytest.mark.parametrize("lengths,news,page", [*BATCHES, ([3000], [1], 64), ([2100], [40], 32)])
@pytest.mark.parametrize("causal", [True, False])
def test_lse(gpu, hq, hkv, d, lengths, news, page, causal):
    """Of every kernel, split contexts among them, with the outputs as without."""
    import sparkq

    q, _, _, cache, table, starts = ref.batch(d + 7, lengths, news, hq, hkv, d, page)
    q = q.to(BF)
    if len(table[0]) > 2:
        table[0][0] = -1
    dev, at = tuple(t.to(gpu) for t in cache), _gpu(gpu, table, starts, lengths)
    for out_dtype in (BF, torch.float32):
        kw = {"scale": d ** -0.5, "max_new": max(news), "mask": "causal" if causal else None,
              "out_dtype": out_dtype}
        out, lse = sparkq.paged_quantized_sdpa(q.to(gpu), dev, *at, return_lse=True, **kw)
        assert torch.equal(out, sparkq.paged_quantized_sdpa(q.to(gpu), dev, *at, **kw))
        want, tol = _lse(q, cache, table, starts, lengths, d ** -0.5, causal)
        lse = lse.cpu().double()
        none = want == -math.inf
        assert (lse[none] == -math.inf).all()
        worst = ((lse - want).abs() / tol)[~none].max().item() if (~none).any() else 0.0
        print(f"[lse] {tuple(lse.shape)} largest error {worst:.3f} of its bound", flush=True)
        assert worst <= 1.0


def check_mass(got, q, lse, cache, before, table, starts, lengths, scale, causal=True, max_new=1 << 30):
    want, added, tol = long.mass(q, lse, cache, before, table, starts, lengths, scale, causal, max_new)
    off = (got.cpu().double() - want).abs() / tol
    print(f"[mass] {tuple(got.shape)} largest error {off.max().item():.3f} of its bound", flush=True)
    assert off.max().item() <= 1.0  # (a NaN fails too)
    return added


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lengths,news,page", BATCHES)
@pytest.mark.parametrize("dtype", [BF, F16])
def test_mass(gpu, hq, hkv, d, lengths, news, page, dtype):
    import sparkq

    q, _, _, cache, table, starts = ref.batch(d + 9, lengths, news, hq, hkv, d, page)
    q = q.to(dtype)
    lse = _lse(q, cache, table, starts, lengths, d ** -0.5)[0].float()
    before = torch.rand((len(lengths), hkv, len(table[0]) * page))
    got = before.to(gpu)
    sparkq.paged_kv_mass(q.to(gpu), lse.to(gpu), tuple(t.to(gpu) for t in cache), got,
                         *_gpu(gpu, table, starts, lengths), scale=d ** -0.5, max_new=max(news))
    added = check_mass(got, q, lse, cache, before, table, starts, lengths, d ** -0.5)
    # every row weighs 1 in all
    rows = torch.tensor([float(n) for n in news], dtype=torch.float64) * (hq // hkv)
    assert torch.allclose(added.sum(-1), rows[:, None].expand(-1, hkv), rtol=1e-5)


@pytest.mark.parametrize("new", [1, 3, 20])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [128, 256])
def test_mass_of_all_kinds_of_batches(gpu, new, causal, d):
    """Absent pages, sequences without new tokens and with more than max_new, rows of no
    sequence, infinite and NaN scales where no row looks, a negative scale, mass in a
    view with an odd page count."""
    import sparkq

    lengths, news, page = [300, 70, 200, 40], [new, 0, new + 5, new], 16
    q, _, _, cache, table, starts = ref.batch(14, lengths, news, 6, 2, d, page, extra_rows=3, width=21)
    q = q.to(F16)
    table[0][3], table[2][11] = -1, 10 ** 9
    cache[1][table[3][2], :, 8:] = math.inf
    cache[1][table[1][0]] = math.nan
    named = {p for r in table for p in r}
    for p in range(cache[0].shape[0]):
        if p not in named:
            cache[1][p] = math.inf
    lse = _lse(q, cache, table, starts, lengths, -0.07, causal)[0].float()
    before = torch.rand((4, 2, 21 * page))
    wide = torch.full((4, 3, 21 * page), 7.0, device=gpu)
    wide[:, 1:] = before.to(gpu)
    sparkq.paged_kv_mass(q.to(gpu), lse.to(gpu), tuple(t.to(gpu) for t in cache), wide[:, 1:],
                         *_gpu(gpu, table, starts, lengths), scale=-0.07, max_new=new,
                         mask="causal" if causal else None)
    check_mass(wide[:, 1:], q, lse, cache, before, table, starts, lengths, -0.07, causal, new)
    assert (wide[:, 0] == 7.0).all()


@pytest.mark.parametrize("new", [1, 30])
def test_mass_of_rows_that_see_nothing(gpu, new):
    """A row whose logarithm is -inf adds nothing (its pages came after it)."""
    import sparkq

    lengths, news = [60], [new]
    q, _, _, cache, table, starts = ref.batch(15, lengths, news, 4, 1, 128, 16)
    q = q.to(BF)
    lse = _lse(q, cache, table, starts, lengths, 0.1)[0].float()
    lse[0, 1:3] = -math.inf
    before = torch.rand((1, 1, 64))
    got = before.to(gpu)
    sparkq.paged_kv_mass(q.to(gpu), lse.to(gpu), tuple(t.to(gpu) for t in cache), got,
                         *_gpu(gpu, table, starts, lengths), scale=0.1, max_new=new)
    check_mass(got, q, lse, cache, before, table, starts, lengths, 0.1)


@pytest.mark.parametrize("lengths,news,page", [([5000, 3, 900], [1, 1, 1], 64),
                                               ([2500, 40], [150, 40], 32)])
def test_mass_of_long_contexts_from_the_attention(gpu, lengths, news, page):
    """With the logarithms that the attention returns, twice over: the second call's new
    tokens start again, the others go on."""
    import sparkq

    q, _, _, cache, table, starts = ref.batch(16, lengths, news, 8, 2, 128, page)
    q = q.to(BF)
    dev, at = tuple(t.to(gpu) for t in cache), _gpu(gpu, table, starts, lengths)
    kw = {"scale": 128 ** -0.5, "max_new": max(news)}
    _, lse = sparkq.paged_quantized_sdpa(q.to(gpu), dev, *at, return_lse=True, **kw)
    got = torch.zeros((len(lengths), 2, len(table[0]) * page), device=gpu)
    for _ in range(2):
        before = got.cpu().clone()
        sparkq.paged_kv_mass(q.to(gpu), lse, dev, got, *at, **kw)
        check_mass(got, q, lse.cpu(), cache, before, table, starts, lengths, 128 ** -0.5)


# --- eviction ----------------------------------------------------------------------

def _keeps(rng, lengths, layers, hkv, count):
    out = torch.full((layers, len(lengths), hkv, count), -1, dtype=torch.int32)
    for layer in range(layers):
        for b, n in enumerate(lengths):
            for h in range(hkv):
                k = min(count, n)
                out[layer, b, h, :k] = torch.tensor(sorted(rng.sample(range(n), k)), dtype=torch.int32)
    return out


def run_evict(gpu, pool, keep, table, lengths, mass):
    import sparkq

    dev = [t.to(gpu) for t in pool]
    m = None if mass is None else mass.to(gpu)
    got = sparkq.kv_pages_evict(dev, keep.to(gpu), _ints(table, gpu), _ints(lengths, gpu), mass=m)
    pages, page = pool[0].shape[1], pool[0].shape[3]
    want = long.evict(table, lengths, keep.shape[-1], pages, page)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1] and got[2].tolist() == [want[2]]
    cache, after = long.moved(pool, mass, keep, table, lengths, want[0], want[1])
    for a, b in zip(dev, cache):
        assert torch.equal(a.cpu(), b)
    if mass is not None:
        assert torch.equal(m.cpu(), after)
    return want


@pytest.mark.parametrize("hkv,d", [(2, 64), (1, 128), (2, 256)])
@pytest.mark.parametrize("lengths,page,count", [
    ([1], 16, 1), ([40, 17, 3], 16, 17), ([40, 17, 3], 16, 16), ([700, 130, 600], 32, 500),
    ([300, 299], 128, 1), ([50], 1024, 49), ([900], 16, 640), ([70, 0, 64], 64, 200)])
def test_evict(gpu, hkv, d, lengths, page, count):
    rng, gen = random.Random(count), torch.Generator().manual_seed(d)
    width = max(-(-n // page) for n in lengths) + 1
    pages = sum(-(-n // page) for n in lengths) + 2
    pool = ref.pool(gen, pages, hkv, page, d, layers=2)
    table = ref.tables(rng, lengths, page, pages, width)
    mass = torch.rand((2, len(lengths), hkv, width * page), generator=gen)
    run_evict(gpu, pool, _keeps(rng, lengths, 2, hkv, count), table, lengths, mass)
    run_evict(gpu, pool, _keeps(rng, lengths, 2, hkv, count), table, lengths, None)


def test_evict_of_shared_pages(gpu):
    """Rows that share a prefix get pages of their own for what is written, and the
    ones that stay keep theirs; short of pages nothing moves."""
    rng, gen = random.Random(1), torch.Generator().manual_seed(1)
    page, lengths = 16, [100, 90, 30, 112, 64]
    table = [[0, 1, 2, 3, 4, 5, 6], [0, 1, 2, 3, 7, 8, -1], [0, 1, -1, -1, -1, -1, -1],
             [9, 10, 11, 12, 13, 14, 15], [9, 10, 11, 12, -1, -1, -1]]
    keep = _keeps(rng, lengths, 1, 2, 40)
    for pages in (30, 28, 27, 17):  # twelve replacements, sixteen pages in use
        pool = ref.pool(gen, pages, 2, page, 64, layers=1)
        mass = torch.rand((1, 5, 2, 7 * page), generator=gen)
        want = run_evict(gpu, pool, keep, table, lengths, mass)
        assert want[2] == max(0, 28 - pages)
        if want[2]:
            assert want[1] == lengths
        else:
            assert want[1] == [40, 40, 30, 40, 40] and want[0][2][:2] == [0, 1]


def test_evict_with_odd_lists_and_absent_pages(gpu):
    """Entries below their place or past the length stand for the place itself, the same
    token may come twice, tokens without a page come as zeros, and a pool of more
    pages than counters fit is planned in the workspace."""
    gen = torch.Generator().manual_seed(2)
    page, lengths = 16, [90, 1000, -4]
    table = [[3, -1, 5, 0, 1, 2], [6, 7, 8, 9, 10, 11], [12] * 6]
    keep = torch.randint(-3, 120, (1, 3, 2, 37), generator=gen, dtype=torch.int32)
    keep[0, 0, 0] = torch.tensor([0, 5, 5, 20, 21, 89, *range(40, 71)])
    mass = torch.rand((1, 3, 2, 96), generator=gen)
    for pages in (14, 20000):
        pool = ref.pool(gen, pages, 2, page, 64, layers=1)
        run_evict(gpu, pool, keep, table, lengths, mass)


def test_evict_of_one_layer(gpu):
    import sparkq

    rng, gen = random.Random(3), torch.Generator().manual_seed(3)
    pool = ref.pool(gen, 12, 2, 32, 128)
    table = ref.tables(rng, [200], 32, 12, 8)
    keep = _keeps(rng, [200], 1, 2, 70)
    dev = [t.to(gpu) for t in pool]
    mass = torch.rand((1, 2, 256), generator=gen)
    m = mass.to(gpu)
    got = sparkq.kv_pages_evict(dev, keep[0].to(gpu), _ints(table, gpu), _ints([200], gpu), mass=m)
    want = long.evict(table, [200], 70, 12, 32)
    assert got[0].tolist() == want[0] and got[1].tolist() == [70]
    cache, after = long.moved([t[None] for t in pool], mass[None], keep, table, [200], *want[:2])
    for a, b in zip(dev, cache):
        assert torch.equal(a.cpu(), b[0])
    assert torch.equal(m.cpu(), after[0])


@pytest.mark.parametrize("hkv,d", [(2, 64), (1, 128), (1, 256)])
def test_evict_in_chunks(gpu, hkv, d):
    """More tokens than a workgroup takes at a time, from all over the row."""
    rng, gen = random.Random(d), torch.Generator().manual_seed(d)
    page, lengths, count = 64, [5000, 2500, 2301, 900], 2300
    width = 80
    pages = sum(-(-n // page) for n in lengths) + 1
    pool = ref.pool(gen, pages, hkv, page, d, layers=2)
    table = ref.tables(rng, lengths, page, pages, width)
    mass = torch.rand((2, len(lengths), hkv, width * page), generator=gen)
    run_evict(gpu, pool, _keeps(rng, lengths, 2, hkv, count), table, lengths, mass)


def test_evict_in_a_strided_pool(gpu):
    """Every second page of a larger pool with the layers inside, mass of a wider tensor:
    what lies between stays as it was."""
    import sparkq

    rng, gen = random.Random(5), torch.Generator().manual_seed(5)
    page, lengths, count = 16, [300, 90, 200], 77
    pool = ref.pool(gen, 40, 2, page, 128, layers=3)
    table = ref.tables(rng, lengths, page, 40, 20)
    mass, keep = torch.rand((3, 3, 2, 20 * page), generator=gen), _keeps(rng, lengths, 3, 2, count)
    wide = [torch.full((40, 2, 3, *t.shape[2:]), 5, dtype=t.dtype, device=gpu) for t in pool]
    dev = [t[:, 1].transpose(0, 1) for t in wide]
    for a, b in zip(dev, pool):
        a.copy_(b)
    m = torch.full((3, 3, 3, 20 * page + 1), 7.0, device=gpu)
    m[:, :, 1:, 1:] = mass.to(gpu)
    got = sparkq.kv_pages_evict(dev, keep.to(gpu), _ints(table, gpu), _ints(lengths, gpu),
                                mass=m[:, :, 1:, 1:])
    want = long.evict(table, lengths, count, 40, page)
    assert got[0].tolist() == want[0] and got[1].tolist() == want[1]
    cache, after = long.moved(pool, mass, keep, table, lengths, want[0], want[1])
    for a, b, t in zip(dev, cache, wide):
        assert torch.equal(a.cpu(), b) and (t[:, 0] == 5).all()
    assert torch.equal(m[:, :, 1:, 1:].cpu(), after)
    assert (m[:, :, 0] == 7.0).all() and (m[..., 0] == 7.0).all()


# --- gathered weight at every count of rows ----------------------------------------

@pytest.mark.parametrize("new", [5, 10, 40])
@pytest.mark.parametrize("causal", [True, False])
@pytest.mark.parametrize("d", [128, 256])
def test_mass_of_all_kinds_of_batches_by_rows(gpu, new, causal, d):
    """15, 30 and 120 rows a KV head, where the ones above have 3, 9 and 60."""
    test_mass_of_all_kinds_of_batches(gpu, new, causal, d)


@pytest.mark.parametrize("new", [1, 4, 8, 16, 17])
@pytest.mark.parametrize("hq,hkv,d", [(8, 2, 64), (8, 2, 128), (4, 1, 256)])
def test_mass_of_many_sequences(gpu, new, hq, hkv, d):
    """More sequences than a wave has lanes, among them long ones that are split and idle
    ones: 4 to 68 rows a KV head."""
    import sparkq

    rng = random.Random(new)
    lengths = [rng.choice([new, new + 1, 40, 333]) for _ in range(70)]
    lengths[3], lengths[66] = 4100, 1999
    lengths = [max(n, new) for n in lengths]
    news = [0 if i % 9 == 7 else new - (i % 2) * (new > 1) for i in range(70)]
    q, _, _, cache, table, starts = ref.batch(new, lengths, news, hq, hkv, d, 32)
    q = q.to(BF)
    dev, at = tuple(t.to(gpu) for t in cache), _gpu(gpu, table, starts, lengths)
    kw = {"scale": d ** -0.5, "max_new": new}
    _, lse = sparkq.paged_quantized_sdpa(q.to(gpu), dev, *at, return_lse=True, **kw)
    before = torch.rand((70, hkv, len(table[0]) * 32))
    got = before.to(gpu)
    sparkq.paged_kv_mass(q.to(gpu), lse, dev, got, *at, **kw)
    check_mass(got, q, lse.cpu(), cache, before, table, starts, lengths, d ** -0.5)


# --- a pool whose offsets need more than 32 bits -----------------------------------

def test_a_pool_past_4_gib(gpu):
    """The same sequences in a small pool and behind 4 GiB of a large one: every result is
    the same, bit for bit."""
    import sparkq

    hkv, d, page, lengths, news = 2, 256, 64, [700, 64, 333], [20, 0, 1]
    q, _, _, cache, table, starts = ref.batch(21, lengths, news, 8, hkv, d, page, spare=4)
    n = cache[0].shape[0]
    small = [t.to(gpu) for t in cache]
    base = 2 ** 32 // (hkv * page * d) + 3
    large = [torch.zeros((base + n, *t.shape[1:]), dtype=t.dtype, device=gpu) for t in cache]
    for a, b in zip(large, small):
        a[base:] = b
    assert large[0].numel() > 2 ** 32
    tables = [table, [[base + p if p >= 0 else p for p in row] for row in table]]
    mass = torch.rand((1, 3, hkv, len(table[0]) * page)).to(gpu)
    q, keep = q.to(F16).to(gpu), _keeps(random.Random(21), lengths, 1, hkv, 250)[0].to(gpu)
    results = []
    for c, tab in zip((small, large), tables):
        at, m = _gpu(gpu, tab, starts, lengths), mass[0].clone()
        bnd = torch.zeros((c[0].shape[0], hkv, 2, d), dtype=BF, device=gpu)
        sparkq.paged_key_bounds(c, bnd, at[0], _ints([0, 700, 764, 1097], gpu), at[2], max_new=700)
        scores, seen = sparkq.paged_page_scores(q, bnd, *at, page_size=page, scale=0.1, max_new=20)
        pages = sparkq.select_top(scores, 3, lengths=seen, first=1, last=1)
        out = sparkq.paged_sparse_sdpa(q, c, pages, *at, scale=0.1, max_new=20)
        full, lse = sparkq.paged_quantized_sdpa(q, c, *at, scale=0.1, max_new=20, return_lse=True)
        for new in (20, 1):  # (of a sequence's first row alone, then)
            sparkq.paged_kv_mass(q, lse, c, m, *at, scale=0.1, max_new=new)
        evicted = sparkq.kv_pages_evict(c, keep, at[0], at[2], mass=m)
        shift = c[0].shape[0] - n
        new_table = torch.where(evicted[0] >= 0, evicted[0] - shift, evicted[0])
        results.append([bnd[shift:], scores, seen, pages, out, full, lse, m, new_table, *evicted[1:],
                        *(t[shift:] for t in c)])
    for a, b in zip(*results):
        assert torch.equal(a, b)


# --- selection at the borders of its kernels ----------------------------------------

@pytest.mark.parametrize("n", [1023, 4095, 8192, 8193, 16384, 16385, 32768, 32769])
@pytest.mark.parametrize("kind", ["normal", "ties"])
def test_select_at_borders(gpu, n, kind):
    test_select(gpu, n, kind)


def test_select_of_many_long_rows(gpu):
    import sparkq

    n = 17001
    x = torch.randn((1, 65, 16, n), generator=torch.Generator().manual_seed(n))
    x[:, ::2] = torch.round(x[:, ::2] * 8)
    lengths = [n - 13 * (i % 5) for i in range(65)]
    got = sparkq.select_top(x.to(gpu), 700, lengths=_ints(lengths, gpu), first=3, last=40)
    assert torch.equal(got.cpu(), long.select(x, 700, lengths, 3, 40))
