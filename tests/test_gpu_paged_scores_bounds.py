"""How far page scores are from their formula, and how far a logit can be above its
page's score.

A score is an fp32 sum of 2 D products of 16-bit values, exact each, times the scale: at
most 2 D - 1 additions off by 2^-24 of `size` = |scale| sum |q||bound|, one rounding of
the product and one of the scale (given as a double): (2 D + 2) 2^-24 of `size` with what
a second order adds. fp16 queries take the page's bounds in fp16, shifted so that the
largest, B, comes to 2^14 or more: below 2^-14 fp16's step is 2^-24, so a bound is off by
2^-25 at most, 2^-39 of B, and the score by |scale| sum |q| 2^-39 B."""

import pytest
import torch

import paged_long_reference as long
import paged_reference as ref
from test_gpu_paged_long import _bounds, _gpu

pytestmark = pytest.mark.gpu

BF, F16 = torch.bfloat16, torch.float16


def _slack(q, size, bnd, table, starts, scale, hkv):
    """[T,Hkv,M] what a score may be off by."""
    d = q.shape[-1]
    tol = (2 * d + 2) * 2.0 ** -24 * size + 2.0 ** -140
    if q.dtype == F16:
        total = q.double().abs().sum(-1).reshape(q.shape[0], hkv, -1).amax(-1) * abs(scale)
        for b, row in enumerate(table):
            for j, p in enumerate(row):
                if p >= 0:
                    most = bnd[p].double().abs().amax((1, 2))
                    part = slice(starts[b], starts[b + 1])
                    tol[part, :, j] += total[part] * most * 2.0 ** -39
    return tol


@pytest.mark.parametrize("hq,hkv,d", [(32, 8, 128), (16, 4, 256), (8, 8, 64), (20, 4, 128), (34, 1, 64)])
@pytest.mark.parametrize("lengths,news", [([700, 64, 1], [1, 1, 1]), ([700, 90, 3], [33, 1, 3])])
@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("spread", [0, 12])
def test_scores_have_the_error_of_one_sum(gpu, hq, hkv, d, lengths, news, dtype, spread):
    """With queries and bounds of ordinary sizes, and ones that lie far apart."""
    import sparkq

    page, scale = 32, d ** -0.5
    q, _, _, cache, table, starts = ref.batch(d, lengths, news, hq, hkv, d, page)
    gen = torch.Generator().manual_seed(d + spread)
    bnd = _bounds(gen, cache[0].shape[0], hkv, d)
    sizes = lambda *shape: 2.0 ** (spread * (2 * torch.rand(shape, generator=gen) - 1))  # noqa: E731
    bnd = (bnd.double() * sizes(*bnd.shape[:2], 1, d)).bfloat16()
    q = (q * sizes(*q.shape)).to(dtype)
    at = _gpu(gpu, table, starts, lengths)
    got, _ = sparkq.paged_page_scores(q.to(gpu), bnd.to(gpu), *at, page_size=page, scale=scale,
                                      max_new=max(news))
    want, size, _, _ = long.scores(q, bnd, table, starts, lengths, page, scale)
    tol = _slack(q, size, bnd, table, starts, scale, hkv)
    seen = want > -torch.inf
    worst = ((got.cpu().double() - want).abs() / tol)[seen].max().item()
    print(f"[scores] {tuple(got.shape)} largest error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0 and (got.cpu()[~seen] == -torch.inf).all()


@pytest.mark.parametrize("dtype", [BF, F16])
@pytest.mark.parametrize("new", [1, 9])
@pytest.mark.parametrize("scale", [0.125, -0.3])
def test_no_logit_is_above_its_pages_score(gpu, dtype, new, scale):
    """Key scales over fp16's range, the largest of tokens that half of the channels do
    not hold, and queries whose channels are as far apart."""
    import sparkq

    lengths, news, page, hkv, d = [400, 77], [new, 1], 32, 2, 64
    q, _, _, cache, table, starts = ref.batch(9, lengths, news, 8, hkv, d, page)
    gen = torch.Generator().manual_seed(new)
    kc, ks = cache[:2]
    ks.copy_(2.0 ** (torch.rand(ks.shape, generator=gen) * 34 - 20))
    kc[..., ::2] = torch.where((ks > 2.0 ** -16)[..., None], 0, kc[..., ::2])
    q = q * 2.0 ** (16 * torch.rand(q.shape, generator=gen) - 12)
    q[..., 1::2] *= (torch.rand((*q.shape[:2], 1), generator=gen) < 0.5)  # some look at the small ones alone
    q = q.to(dtype)
    dev = tuple(t.to(gpu) for t in cache)
    bnd = torch.zeros((cache[0].shape[0], hkv, 2, d), dtype=BF, device=gpu)
    sparkq.paged_key_bounds(dev, bnd, *_gpu(gpu, table, [0, 400, 477], lengths), max_new=400)
    got, _ = sparkq.paged_page_scores(q.to(gpu), bnd, *_gpu(gpu, table, starts, lengths), page_size=page,
                                      scale=scale, max_new=new)
    got, bnd = got.cpu().double(), bnd.cpu()
    _, size, _, _ = long.scores(q, bnd, table, starts, lengths, page, scale)
    tol = _slack(q, size, bnd, table, starts, scale, hkv)
    for b, n in enumerate(lengths):
        for r in range(starts[b], starts[b + 1]):
            for pos in range(n - (starts[b + 1] - r) + 1):
                p, j = table[b][pos // page], pos // page
                k = kc[p, :, pos % page].double() * ks[p, :, pos % page].double()[:, None]
                logit = (q[r].double().reshape(hkv, -1, d) * k[:, None]).sum(-1) * scale
                assert (logit.amax(1) <= got[r, :, j] + tol[r, :, j]).all(), (r, pos)
