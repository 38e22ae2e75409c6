"""qk_norm_rope against the float64 formula: head dims that every kernel path
takes, partial and interleaved rotations, strided views, far positions.

Tolerance, per element with parts = |ya| + |yb| (the rotation's terms): the
result's rounding, eps/2 of it (2^-25 in fp16's subnormal range), and the fp32
chain: the row's mean of D products (D/64 + 8 roundings of 2^-24), the root, two
products, the cosine and sine of an angle held to 2^-24 turns (8 * 2^-24), two
products and a sum: under 2^-19 of parts for D <= 512."""

import pytest
import torch

from paged_reference import norm_rope

pytestmark = pytest.mark.gpu

EPS, BASE = 1e-6, 1e6


def _check(got, x, w, pos, dims, base=BASE, **kw):
    ref, parts = norm_rope(x.cpu(), w.cpu(), pos.cpu(), dims, EPS, base, **kw)
    got = got.cpu().double()
    tiny = 2.0 ** -25 if x.dtype == torch.float16 else 0.0
    tol = (torch.finfo(x.dtype).eps / 2 * ref.abs()).clamp(min=tiny) * 1.01 + 2.0 ** -19 * parts
    off = ((got - ref).abs() / tol).max().item() if got.numel() else 0.0
    print(f"[norm_rope] {tuple(x.shape)} dims={dims} {kw} largest error {off:.3f} of its bound")
    assert got.shape == ref.shape and off <= 1.0


def _inputs(gpu, t, hq, hkv, d, dtype, seed=0, far=131072):
    gen = torch.Generator().manual_seed(seed)
    qkv = torch.randn((t, hq + 2 * hkv, d), generator=gen).to(dtype).to(gpu)
    w = [(1 + 0.3 * torch.randn(d, generator=gen)).to(dtype).to(gpu) for _ in range(2)]
    pos = torch.randint(0, far, (t,), generator=gen, dtype=torch.int32).to(gpu)
    return qkv[:, :hq], qkv[:, hq:hq + hkv], *w, pos


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("t,hq,hkv,d,dims", [
    (1, 32, 8, 128, 128), (3, 16, 4, 256, 256), (65, 20, 4, 128, 64), (7, 2, 1, 64, 64),
    (1000, 4, 2, 64, 32), (2, 3, 1, 80, 80), (5, 3, 1, 80, 6), (4, 1, 1, 6, 4), (3, 2, 2, 512, 512),
    (2, 1, 1, 100, 50), (9, 2, 1, 96, 48), (3, 2, 1, 128, 8), (33, 1, 1, 256, 200),
    (2, 2, 1, 1000, 1000), (3, 1, 2, 2, 2)])
@pytest.mark.parametrize("traditional", [False, True])
def test_matches_the_formula(gpu, t, hq, hkv, d, dims, traditional, dtype):
    import sparkq

    q, k, wq, wk, pos = _inputs(gpu, t, hq, hkv, d, dtype, seed=d + dims)
    print(f"[case] t={t} heads={hq}/{hkv} d={d} dims={dims} {traditional} {dtype}", flush=True)
    qo, ko = sparkq.qk_norm_rope(q, k, wq, wk, pos, dims=dims, eps=EPS, base=BASE,
                                 traditional=traditional)
    _check(qo, q, wq, pos, dims, traditional=traditional)
    _check(ko, k, wk, pos, dims, traditional=traditional)


def test_positions_of_64_bits_scale_and_base(gpu):
    import sparkq

    q, k, wq, wk, _ = _inputs(gpu, 6, 4, 2, 128, torch.bfloat16)
    # 2^31 is past int32; -3 comes before the first token
    pos = torch.tensor([0, 1, 2 ** 31, 2 ** 31 + 12345, -3, 99999], dtype=torch.int64, device=gpu)
    qo, ko = sparkq.qk_norm_rope(q, k, wq, wk, pos, dims=128, eps=EPS, base=500000.0, scale=0.25)
    # at 2^29 turns a base^(-2i/d) of 53 bits leaves 2^-24 turns: within the bound's angle
    _check(qo, q, wq, pos, 128, base=500000.0, scale=0.25)
    _check(ko, k, wk, pos, 128, base=500000.0, scale=0.25)


def test_layouts_give_the_same_bits(gpu):
    """Packed views, contiguous tensors, rows at odd addresses, a head-major
    layout and a strided last axis: the values are the same, whichever path
    reads them."""
    import sparkq

    q, k, wq, wk, pos = _inputs(gpu, 37, 8, 2, 128, torch.bfloat16, seed=3)
    run = lambda q, k: sparkq.qk_norm_rope(q, k, wq, wk, pos, dims=128, eps=EPS, base=BASE)  # noqa: E731
    want = run(q.contiguous(), k.contiguous())
    odd = [torch.empty(t.numel() + 1, dtype=t.dtype, device=gpu)[1:].view(t.shape).copy_(t)
           for t in (q, k)]
    major = [t.transpose(0, 1).contiguous().transpose(0, 1) for t in (q, k)]
    last = [t.transpose(1, 2).contiguous().transpose(1, 2) for t in (q, k)]
    for name, pair in (("packed", (q, k)), ("odd", odd), ("head major", major), ("last", last)):
        for a, b in zip(run(*pair), want):
            ref = b.float()
            # another path may round the fp32 chain otherwise: a unit of bf16 at most
            assert ((a.float() - ref).abs() <= 2.0 ** -7 * ref.abs() + 1e-6).all(), name
        assert all(x.is_contiguous() for x in run(*pair))


def test_no_rows_and_values_out_of_range(gpu):
    import sparkq

    q, k, wq, wk, pos = _inputs(gpu, 4, 2, 1, 128, torch.bfloat16)
    for t in sparkq.qk_norm_rope(q[:0], k[:0], wq, wk, pos[:0], dims=128, eps=EPS):
        assert t.shape[0] == 0
    q = q.clone()
    q[1, 0, 5] = float("nan")
    q[2, 1] = 0
    qo, ko = sparkq.qk_norm_rope(q, k, wq, wk, pos, dims=128, eps=EPS)
    assert qo[1, 0].isnan().all() and qo[1, 1].isfinite().all()
    assert (qo[2, 1] == 0).all() and ko.isfinite().all()
