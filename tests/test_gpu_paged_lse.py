"""The logarithm of a row's sum is that of its scores alone, whatever the values' scales:
spread over fp16's range, zero, or not finite, where the outputs are not finite either
(whatever weight the token has) but the logarithms and the gathered weights are. The
bounds of the errors are those of test_gpu_paged_long."""

import math

import pytest
import torch

import paged_reference as ref
from test_gpu_paged_long import _gpu, _lse, check_mass

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
# (contexts of more than 128 tokens are split here) few rows, tiles of 128 rows, pairs of waves
SHAPES = [(128, 1, 4, 2, 128, 64), (400, 1, 4, 2, 64, 32), (700, 2, 8, 2, 256, 64),
          (128, 40, 4, 1, 64, 16), (400, 40, 8, 2, 128, 64),
          (128, 40, 4, 1, 256, 32), (500, 40, 4, 1, 256, 64)]


def _case(n, new, hq, hkv, d, page, low=()):
    """A batch of one sequence. Every query's first dim is 8, and the tokens `low` have
    scores of about -300 (2^-433 of the others' weight: nothing in fp32)."""
    q, _, _, cache, table, starts = ref.batch(n + new, [n], [new], hq, hkv, d, page)
    q[..., 0] = 8
    kc, ks = cache[:2]
    kc[..., 0] = 0
    for pos in low:
        p, s = table[0][pos // page], pos % page
        kc[p, :, s] = 0
        kc[p, :, s, 0] = -127
        ks[p, :, s] = 300 / (8 * 127 * d ** -0.5)
    return q.to(BF), cache, table, starts


def _run(gpu, q, cache, table, starts, n, new, out_dtype):
    """(out, lse on the CPU), with what lse and the weights have to be checked."""
    import sparkq

    scale = q.shape[-1] ** -0.5
    dev, at = tuple(t.to(gpu) for t in cache), _gpu(gpu, table, starts, [n])
    kw = {"scale": scale, "max_new": new}
    out, lse = sparkq.paged_quantized_sdpa(q.to(gpu), dev, *at, return_lse=True, out_dtype=out_dtype, **kw)
    want, tol = _lse(q, cache, table, starts, [n], scale)
    worst = ((lse.cpu().double() - want).abs() / tol).max().item()
    print(f"[lse] {tuple(lse.shape)} largest error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0  # (a NaN fails too)
    hkv, room = cache[0].shape[1], len(table[0]) * cache[0].shape[2]
    before = torch.rand((1, hkv, room), generator=torch.Generator().manual_seed(n))
    got = before.to(gpu)
    sparkq.paged_kv_mass(q.to(gpu), lse, dev, got, *at, **kw)
    check_mass(got, q, lse.cpu(), cache, before, table, starts, [n], scale)
    return out.cpu()


@pytest.mark.parametrize("n,new,hq,hkv,d,page", SHAPES)
@pytest.mark.parametrize("size", [math.inf, -math.inf, math.nan])
@pytest.mark.parametrize("at", [[5], range(40, 88)])
@pytest.mark.parametrize("out_dtype", [BF, torch.float32])
def test_scales_of_values_that_are_not_finite(gpu, n, new, hq, hkv, d, page, size, at, out_dtype):
    q, cache, table, starts = _case(n, new, hq, hkv, d, page)
    for pos in at:
        cache[3][table[0][pos // page], :, pos % page] = size
    cache[2][table[0][0], :, 5] = 0  # (values of 0 too)
    assert not _run(gpu, q, cache, table, starts, n, new, out_dtype).isfinite().any()


@pytest.mark.parametrize("n,new,hq,hkv,d,page", SHAPES)
@pytest.mark.parametrize("low,at", [(range(32), 5), (range(32, 64), 40), (range(64), 60), ([70], 70)])
@pytest.mark.parametrize("out_dtype", [BF, torch.float32])
def test_scales_that_are_not_finite_of_tokens_without_weight(gpu, n, new, hq, hkv, d, page, low, at, out_dtype):
    """Alone in the half of a block, a block or a part of the context, whose sums count
    for nothing beside the others'."""
    q, cache, table, starts = _case(n, new, hq, hkv, d, page, low)
    cache[3][table[0][at // page], :, at % page] = math.inf
    assert not _run(gpu, q, cache, table, starts, n, new, out_dtype).isfinite().any()


@pytest.mark.parametrize("n,new,hq,hkv,d,page", SHAPES)
@pytest.mark.parametrize("down", [True, False])
@pytest.mark.parametrize("low", [(), range(32)])
def test_scales_of_values_over_the_whole_range(gpu, n, new, hq, hkv, d, page, down, low):
    """From fp16's least to its largest in ascending or descending order, and none."""
    q, cache, table, starts = _case(n, new, hq, hkv, d, page, low)
    for pos in range(n):
        e = -24 + (n - 1 - pos if down else pos) * 39 / n
        cache[3][table[0][pos // page], :, pos % page] = 0.0 if pos % 7 == 3 else 2.0 ** e
    for out_dtype in (BF, torch.float32):
        assert _run(gpu, q, cache, table, starts, n, new, out_dtype).isfinite().all()
    for p in table[0]:
        cache[3][p] = 0.0
    out = _run(gpu, q, cache, table, starts, n, new, BF)
    assert (out == 0).all()
