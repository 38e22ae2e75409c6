"""How many bits the weights of the attention over selected pages keep, 22 whatever the
outputs are, and values that are not finite there: the cases and bounds of
test_gpu_paged_weights, over lists that name every page (whole lists, and ones that are
split over the chip)."""

import pytest
import torch

from test_gpu_paged_weights import KINDS, _case, _check, _ints, _pool

pytestmark = pytest.mark.gpu

# (n, new, hq, hkv, d, page): lists of up to 512 tokens at D <= 128 and 256 at D = 256 stay whole
WHOLE = [(500, 1, 4, 1, 64, 64), (400, 3, 4, 2, 128, 16), (250, 1, 2, 1, 256, 32), (300, 30, 8, 1, 64, 16)]
SPLIT = [(900, 1, 4, 1, 64, 64), (1500, 2, 8, 2, 128, 16), (700, 3, 2, 1, 256, 32), (600, 5, 40, 2, 64, 16)]


def _run(gpu, q, cache, table, n, out_dtype):
    import sparkq

    new, _, d = q.shape
    pages = torch.arange(table.shape[1], dtype=torch.int32, device=gpu)
    lists = pages.expand(new, cache[0].shape[1], -1).contiguous()
    return sparkq.paged_sparse_sdpa(q.to(gpu), cache, lists, table, _ints([0, new], gpu), _ints([n], gpu),
                                    scale=d ** -0.5, max_new=new, out_dtype=out_dtype)


@pytest.mark.parametrize("kind", [*KINDS, "plain"])
@pytest.mark.parametrize("amp", [1.0, 1e-4])
@pytest.mark.parametrize("n,new,hq,hkv,d,page", [*WHOLE, *SPLIT])
def test_no_token_costs_the_others_their_bits(gpu, kind, amp, n, new, hq, hkv, d, page):
    q, kc, ks, vc, vs = _case(kind, amp, n, new, hq, hkv, d, page, seed=n + new)
    q = q.to(torch.bfloat16)
    cache, table = _pool(gpu, kc, ks, vc, vs, page, 1)
    for dtype in (torch.float32, torch.bfloat16):
        _check(_run(gpu, q, cache, table, n, dtype), q, kc, ks, vc, vs, 2.0 ** -22, 2.0 ** -38)


@pytest.mark.parametrize("n,new,hq,hkv,d,page", [*WHOLE, *SPLIT])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_contiguous_caches_bars(gpu, n, new, hq, hkv, d, page, dtype):
    """16-bit outputs within one unit of the rounded float64 ones, float32 ones within 2e-5
    of their norm (11 bits leave 1.5e-4)."""
    import oracle as o
    from helpers import check_rounded16, rel_l2

    q, kc, ks, vc, vs = _case("plain", 1.0, n, new, hq, hkv, d, page, seed=7)
    q = q.to(dtype)
    cache, table = _pool(gpu, kc, ks, vc, vs, page, 2)
    want = torch.zeros((new, hq, d), dtype=torch.float64)
    see = torch.ones((new, n), dtype=torch.bool).tril(n - new)
    for h in range(hq):
        k, v = (c[:, h * hkv // hq].double() * x[:, h * hkv // hq].double()[:, None]
                for c, x in ((kc, ks), (vc, vs)))
        sc = torch.where(see, q[:, h].double() @ k.T * d ** -0.5, -torch.inf)
        want[:, h] = torch.softmax(sc, -1) @ v
    rel = rel_l2(_run(gpu, q, cache, table, n, torch.float32).cpu().numpy(), want.numpy())
    print(f"[weights] relative L2 error {rel:.2e}", flush=True)
    assert rel <= 2e-5
    out = _run(gpu, q, cache, table, n, dtype).cpu()
    check_rounded16(out.view(torch.int16).numpy().view("uint16"), want.numpy(),
                    o.BF16 if dtype == torch.bfloat16 else o.F16)


@pytest.mark.parametrize("n,new,hq,hkv,d,page", [*WHOLE, *SPLIT])
@pytest.mark.parametrize("size", [float("inf"), float("nan")])
@pytest.mark.parametrize("at,low", [([5], ()), (range(64, 192), ()), ([5], range(32)), ([130], range(128, 144))])
def test_visible_scales_that_are_not_finite(gpu, n, new, hq, hkv, d, page, size, at, low):
    """No row that sees one has a finite value, not even where its block, or its part of the
    list (`low`: scores of -300), counts for nothing beside the others."""
    q, kc, ks, vc, vs = _case("plain", 1.0, n, new, hq, hkv, d, page, seed=3)
    vs[list(at)] = size
    vc[list(at)[::2]] = 0
    for pos in low:
        kc[pos], ks[pos] = 0, 300 / (8 * 127 * d ** -0.5)
        kc[pos, :, 0] = -127
    cache, table = _pool(gpu, kc, ks, vc, vs, page, 1)
    for dtype in (torch.float16, torch.float32):
        assert not _run(gpu, q.half(), cache, table, n, dtype).isfinite().any()
