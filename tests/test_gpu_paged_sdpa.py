"""paged_quantized_sdpa against the float64 form.

Tolerance of an output o = sum p v / sum p, with mass = sum p|v| / sum p:
 - its rounding: eps/2 of the value that is rounded (the errors below included),
   none in fp32;
 - the weights' one rounding to fp16, in the numerator alone: fp16 has 11 bits,
   so half a step of a weight is at most 2^-11 of it (1 + 2^-11 lies halfway
   between 1 and the next fp16, 1 + 2^-10), in all 2^-11 mass;
 - weights under fp16's normal range, which are rounded to its step of 2^-24
   instead, by 2^-25 of the unit at most. With s the largest score (log2) and V
   the largest value scale a row has seen, the unit is 2^(m + e - 6) with m <=
   s and 2^e <= V, so under 2^-5 V 2^s, and all these roundings
   together add up to less than 2^-30 V 2^s sum |code| / sum p, sum p in units of
   1: 2^-30 of `steps`. (A sharp softmax needs it: where the code of the one
   token that counts is 0, the rest is all there is of want and mass.)
 - the scores: fp32 products of exact operands, summed D at a time, times three
   factors: (D + 8) 2^-24 of scale * sum|q||k| (`size`), twice (numerator and
   normalizer), and exp2's 2^-22;
 - fp32 sums over n weights: n 2^-24, twice.
"""

import math

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu


def _ints(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def check(got, q, cache, table, starts, lengths, scale, causal=True, max_new=1 << 30):
    want, mass, size, done, steps = ref.attention(q, cache, table, starts, lengths, scale, causal,
                                                  max_new)
    d = q.shape[-1]
    n = max([0, *lengths])
    part = 2.0 ** -11 + 2 * (d + 8) * 2.0 ** -24 * size[..., None] + 2.0 ** -20 + n * 2.0 ** -23
    half = 0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -25 if got.dtype == torch.float16 else 2.0 ** -60
    part = 1.01 * part * mass + 2.0 ** -30 * steps
    tol = (half * (want.abs() + part)).clamp(min=tiny) + part
    off = ((got.cpu().double() - want).abs() / tol)[done]
    worst = off.max().item() if off.numel() else 0.0
    print(f"[paged sdpa] {tuple(got.shape)} n={n} largest error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0  # (a NaN fails too)
    return done


def run(gpu, q, cache, table, starts, lengths, max_new, **kw):
    import sparkq

    return sparkq.paged_quantized_sdpa(
        q.to(gpu), tuple(t.to(gpu) for t in cache), _ints(table, gpu), _ints(starts, gpu),
        _ints(lengths, gpu), scale=q.shape[-1] ** -0.5, max_new=max_new, **kw)


HEADS = [(32, 8, 128), (16, 4, 256), (8, 8, 64), (6, 2, 128), (32, 1, 64), (20, 4, 128), (5, 5, 256)]


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lengths,page", [
    ([1], 16), ([33], 16), ([64, 1, 65, 0, 200], 64), ([1000], 32), ([300, 700, 31, 32, 129], 16),
    ([1500, 20], 1024)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_decode(gpu, hq, hkv, d, lengths, page, dtype):
    news = [min(1, n) for n in lengths]
    q, _, _, cache, table, starts = ref.batch(d, lengths, news, hq, hkv, d, page)
    q = q.to(dtype)
    out = run(gpu, q, cache, table, starts, lengths, 1)
    assert out.dtype == dtype
    assert check(out, q, cache, table, starts, lengths, d ** -0.5).all()


@pytest.mark.parametrize("hq,hkv,d", HEADS)
@pytest.mark.parametrize("lengths,news,page", [
    ([7], [7], 16), ([40, 9], [33, 9], 16), ([130, 5, 64, 300], [130, 1, 0, 17], 64),
    ([257], [100], 32), ([90, 90, 90], [4, 3, 1], 128)])
@pytest.mark.parametrize("causal", [True, False])
def test_chunks(gpu, hq, hkv, d, lengths, news, page, causal):
    q, _, _, cache, table, starts = ref.batch(d + 1, lengths, news, hq, hkv, d, page)
    q = q.to(torch.bfloat16)
    out = run(gpu, q, cache, table, starts, lengths, max(news), mask="causal" if causal else None,
              out_dtype=torch.float32)
    assert check(out, q, cache, table, starts, lengths, d ** -0.5, causal).all()


@pytest.mark.parametrize("news", [[1, 1, 1, 1], [20, 1, 5, 40]])
def test_a_long_context_beside_short_ones(gpu, news):
    lengths = [6000, 3, 40, 500]
    lengths = [max(a, b) for a, b in zip(lengths, news)]
    q, _, _, cache, table, starts = ref.batch(7, lengths, news, 8, 2, 128, 64)
    q = q.to(torch.float16)
    out = run(gpu, q, cache, table, starts, lengths, max(news))
    check(out, q, cache, table, starts, lengths, 128 ** -0.5)


@pytest.mark.parametrize("new", [1, 30])
def test_many_sequences(gpu, new):
    lengths = [new + (37 * i) % 90 for i in range(300)]
    news = [(new, 0, 1)[i % 3] for i in range(300)]
    q, _, _, cache, table, starts = ref.batch(8, lengths, news, 4, 2, 64, 16)
    q = q.to(torch.bfloat16)
    out = run(gpu, q, cache, table, starts, lengths, new)
    check(out, q, cache, table, starts, lengths, 64 ** -0.5)


@pytest.mark.parametrize("new,max_new", [(1, 1), (12, 12), (40, 25), (3, 1)])
def test_rows_that_see_nothing_and_rows_left_alone(gpu, new, max_new):
    """More rows than tokens (the first see nothing), absent pages, rows past
    max_new, rows behind the last sequence and a length past the row of pages."""
    lengths, news = [50, 1, 90, 0, 200], [new] * 5
    q, _, _, cache, table, starts = ref.batch(9, lengths, news, 8, 2, 128, 16, extra_rows=3, width=13)
    table[0][1] = -1
    table[2][:6] = [-1, 10 ** 9, -7, -1, -1, -1]  # nothing of it is there
    lengths[4] = 10 ** 6
    q = q.to(torch.bfloat16)
    out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=gpu)
    got = run(gpu, q, cache, table, starts, lengths, max_new, out=out)
    assert got.data_ptr() == out.data_ptr()
    lengths[4] = 13 * 16
    done = check(out, q, cache, table, starts, lengths, 128 ** -0.5, max_new=max_new)
    assert (out.cpu()[~done] == 7.0).all() and not done.all()
    first = starts[2]
    assert (out[first:first + min(new, max_new)] == 0).all()


def test_starts_out_of_range(gpu):
    lengths, news = [30, 30, 30], [5, 5, 5]
    q, _, _, cache, table, _ = ref.batch(10, lengths, news, 4, 2, 64, 16)
    q = q.to(torch.bfloat16)
    for starts in ([-9, 4, 4, 10 ** 9], [3, 9, 12, 15], [0, 0, 0, 0]):
        out = torch.full(q.shape, 7.0, dtype=torch.bfloat16, device=gpu)
        run(gpu, q, cache, table, starts, lengths, 30, out=out)
        done = check(out, q, cache, table, starts, lengths, 64 ** -0.5)
        assert (out.cpu()[~done] == 7.0).all()


@pytest.mark.parametrize("new", [1, 24])
def test_values_that_no_row_may_see(gpu, new):
    """Scales of NaN and infinity behind each sequence's end (its last page's
    tail, pages that no table names) and, under the causal mask, in the last new
    token, which only the last row sees."""
    lengths, news = [70, 33], [new, new]
    q, _, _, cache, table, starts = ref.batch(11, lengths, news, 8, 2, 128, 32)
    kc, ks, vc, vs = cache
    named = {p for r, n in zip(table, lengths) for p in r[: -(-n // 32)]}
    for p in range(kc.shape[0]):
        if p not in named:
            ks[p], vs[p] = math.nan, math.inf
    for r, n in zip(table, lengths):
        ks[r[n // 32], :, n % 32:] = math.inf
        vs[r[n // 32], :, n % 32:] = math.nan
    q = q.to(torch.bfloat16)
    check(run(gpu, q, cache, table, starts, lengths, new), q, cache, table, starts, lengths, 128 ** -0.5)
    if new > 1:
        last = lengths[0] - 1
        ks[table[0][last // 32], :, last % 32] = math.inf
        vs[table[0][last // 32], :, last % 32] = math.nan
        out = run(gpu, q, cache, table, starts, lengths, new).cpu()
        assert out[starts[1] - 1].isnan().all()
        keep = [i for i in range(starts[2]) if i != starts[1] - 1]
        want, mass, *_ = ref.attention(q, cache, table, starts, lengths, 128 ** -0.5)
        assert ((out[keep].double() - want[keep]).abs() <= 2.0 ** -7 * mass[keep] + 1e-9).all()


def test_scales_far_apart(gpu):
    """Values whose scales span fp16's range: the largest decide a row, but a
    row that sees only small ones has their precision."""
    lengths, news = [64], [64]
    q, _, _, cache, table, starts = ref.batch(12, lengths, news, 4, 2, 64, 16)
    kc, ks, vc, vs = cache
    for pos in range(64):
        vs[table[0][pos // 16], :, pos % 16] = 2.0 ** (-24 + pos * 39 / 63)
    q = q.to(torch.bfloat16)
    check(run(gpu, q, cache, table, starts, lengths, 64, out_dtype=torch.float32), q, cache, table,
          starts, lengths, 64 ** -0.5)
    for p in range(vs.shape[0]):
        vs[p] = 6e-8
    check(run(gpu, q, cache, table, starts, lengths, 64, out_dtype=torch.float32), q, cache, table,
          starts, lengths, 64 ** -0.5)


def test_queries_of_any_size(gpu):
    """Rows of very large, very small, zero and infinite queries."""
    lengths, news = [80], [8]
    q, _, _, cache, table, starts = ref.batch(13, lengths, news, 4, 2, 128, 16)
    q[0] *= 1e4
    q[1] *= 1e-6
    q[2] = 0
    q[3] *= 300
    q = q.to(torch.bfloat16)
    check(run(gpu, q, cache, table, starts, lengths, 8), q, cache, table, starts, lengths, 128 ** -0.5)
    q[4, 0, 3] = math.inf
    q[5, 1, 0] = math.nan
    out = run(gpu, q, cache, table, starts, lengths, 8).cpu()
    assert out[4, 0].isnan().all() and out[5, 1].isnan().all()
    assert out[4, 1:].isfinite().all() and out[6:].isfinite().all()


def test_views_and_strided_pools(gpu):
    import sparkq

    lengths, news, hq, hkv, d = [90, 40], [20, 40], 8, 2, 128
    q, _, _, cache, table, starts = ref.batch(14, lengths, news, hq, hkv, d, 32)
    q = q.to(torch.bfloat16)
    t = q.shape[0]
    packed = torch.randn((t, hq + 4, d), device=gpu).to(torch.bfloat16)
    packed[:, :hq] = q.to(gpu)
    dev = [torch.zeros((c.shape[0], 3, *c.shape[1:]), dtype=c.dtype, device=gpu) for c in cache]
    for b, c in zip(dev, cache):
        b[:, 1] = c.to(gpu)
    odd = torch.empty(q.numel() + 1, dtype=q.dtype, device=gpu)[1:].view(q.shape).copy_(q.to(gpu))
    major = q.to(gpu).transpose(0, 1).contiguous().transpose(0, 1)
    for queries in (packed[:, :hq], odd, major):
        out = sparkq.paged_quantized_sdpa(queries, tuple(b[:, 1] for b in dev), _ints(table, gpu),
                                          _ints(starts, gpu), _ints(lengths, gpu),
                                          scale=d ** -0.5, max_new=40)
        check(out, q, cache, table, starts, lengths, d ** -0.5)


def test_pages_past_32_bits(gpu):
    """A pool of over 4 GiB whose last pages are the ones in use."""
    import sparkq

    pages, hkv, page, d = 1100, 8, 2048 // 2, 256  # 2 MiB of codes a page and side
    lengths, news = [2000, 1024], [30, 1]
    q, k, v, small, _, starts = ref.batch(15, lengths, news, 16, hkv, d, page)
    q = q.to(torch.bfloat16)
    cache = (torch.zeros((pages, hkv, page, d), dtype=torch.int8, device=gpu),
             torch.zeros((pages, hkv, page), dtype=torch.float16, device=gpu))
    cache = cache + tuple(torch.zeros_like(t) for t in cache)
    assert cache[0].numel() * 2 > 2 ** 32
    table = [[pages - 1, pages - 3], [pages - 2, -1]]
    for b, s in zip(cache, small):
        b[pages - 3:] = s[:3].to(gpu)
    at = _ints(table, gpu), _ints(starts, gpu), _ints(lengths, gpu)
    near = [[2, 0], [1, -1]]
    sparkq.paged_kv_append(k.half().to(gpu), v.half().to(gpu), cache, *at)
    want = ref.append(k.half(), v.half(), tuple(s[:3] for s in small), near, starts, lengths)
    for a, b in zip(cache, want):
        assert torch.equal(a[pages - 3:].cpu(), b)
        assert not a[: pages - 3].any()
    out = sparkq.paged_quantized_sdpa(q.to(gpu), cache, *at, scale=d ** -0.5, max_new=30)
    check(out, q, want, near, starts, lengths, d ** -0.5)
    moved, used = sparkq.kv_pages_compact(cache, at[0], at[2])
    assert used.item() == 3 and moved.tolist() == [[2, 0], [1, -1]]
    for a, b in zip(cache, want):
        assert torch.equal(a[:3].cpu(), b)
