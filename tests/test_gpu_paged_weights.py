"""How many bits the paged attention's weights keep, whatever the values of the
other tokens: rows of zeros (which the quantizer stores with scale 1), tokens of
large values and next to no weight, tokens of small values and all the weight.

Tolerance of an output o = sum p v / sum p, v = scale * code, P the largest p *
scale of a token that has a code other than 0:
 - each weight's rounding: `bits` of it. 2^-11, half a step of fp16's 11 bits, in
   tiles with a 16-bit output. Else what fp16 leaves, 2^-11 of the weight at most, is
   a second operand and rounded by 2^-11 in turn: 2^-22;
 - weights under fp16's normal range, rounded to half of 2^-24: with few rows the
   unit puts P at 2^13 or above, so 2^-38 of P each; in tiles at 2^6, less 2^4 by
   which the scales of a block that is taken whole may differ: 2^-27 of P. In all
   that times sum |code|;
 - the scores: fp32 products of exact operands, D of them summed, and three
   factors: each p is off by (D + 8) 2^-24 of its scale * sum |q||k|, in the
   numerator and in the normalizer; exp2 and the rest 2^-20;
 - fp32 sums over n weights: n 2^-24, twice;
 - the output's own rounding, eps / 2 of what is rounded."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def _ints(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _case(kind, amp, n, new, hq, hkv, d, page, seed):
    """(q, k codes, k scales, v codes, v scales) with tokens in order, on the CPU.
    Every query's first dim is 8, which only the special tokens' keys look at."""
    gen = torch.Generator().manual_seed(seed)
    q = torch.randn((new, hq, d), generator=gen)
    q[..., 0] = 8.0
    kc = torch.randint(-127, 128, (n, hkv, d), generator=gen, dtype=torch.int8)
    kc[..., 0] = 0
    ks = (0.005 + 0.02 * torch.rand((n, hkv), generator=gen)).half()
    v = torch.randn((n, hkv, d), generator=gen) * amp
    vs = (v.abs().amax(-1) / 127).half()
    vc = torch.round(v / vs.float()[..., None]).clamp(-127, 127).to(torch.int8)

    def score(at, nats):  # of a token, for every query
        kc[at], ks[at] = 0, abs(nats) / (8 * 127 * d ** -0.5)
        kc[at, :, 0] = 127 if nats > 0 else -127

    first, last = 0, n - new  # the last one that every row sees
    special = {"zero low": [3, last], "zero": [0, n // 2], "zero high": [n // 3],
               "zero block": list(range(64, min(192, last))), "far": [2, last], "sink": [first], "plain": []}[kind]
    for at in special:
        if kind.startswith("zero"):
            vc[at], vs[at] = 0, 1.0
        if kind == "zero low":
            score(at, -40.0)
        elif kind == "zero high":
            score(at, 9.0)
        elif kind == "far":
            score(at, -80.0)
            vs[at] = min(3e7 * amp / 127, 6e4)
        elif kind == "sink":  # nearly all the weight on a value 2^10 times smaller
            score(at, 12.0)
            vs[at] = float(vs[at].max()) / 1024
    return q, kc, ks, vc, vs


def _pool(gpu, kc, ks, vc, vs, page, seed):
    n, hkv, d = kc.shape
    count = -(-n // page)
    ids = torch.randperm(count + 2, generator=torch.Generator().manual_seed(seed))[:count]
    out = []
    for codes, scales in ((kc, ks), (vc, vs)):
        c = torch.randint(-127, 128, (count + 2, hkv, page, d), dtype=torch.int8)
        s = torch.full((count + 2, hkv, page), 0.01, dtype=torch.float16)
        for t in range(n):
            c[ids[t // page], :, t % page] = codes[t]
            s[ids[t // page], :, t % page] = scales[t]
        out += [c.to(gpu), s.to(gpu)]
    return tuple(out), _ints([ids.tolist()], gpu)


def _check(got, q, kc, ks, vc, vs, bits, floor):
    new, hq, d = q.shape
    n, hkv, _ = kc.shape
    g, scale = hq // hkv, d ** -0.5
    half = 0 if got.dtype == torch.float32 else torch.finfo(got.dtype).eps / 2
    worst = 0.0
    got = got.cpu().double()
    for h in range(hq):
        k = kc[:, h // g].double() * ks[:, h // g].double()[:, None]
        c, s = vc[:, h // g].double(), vs[:, h // g].double()
        qh = q[:, h].double()
        see = torch.ones((new, n), dtype=torch.bool).tril(n - new)
        sc = torch.where(see, qh @ k.T * scale, -torch.inf)
        p = torch.softmax(sc, -1)
        size = qh.abs() @ k.abs().T * scale * (d + 8) * 2.0 ** -24
        v = c * s[:, None]
        want, mass = p @ v, p @ v.abs()
        top = (p * s * (c != 0).any(-1)).amax(-1)
        codes = see.double() @ c.abs()
        part = 1.01 * ((bits + 2.0 ** -20 + n * 2.0 ** -23) * mass + floor * top[:, None] * codes
                       + (p * size) @ v.abs() + (p * size).sum(-1, keepdim=True) * mass)
        tol = half * (want.abs() + part) + part + 2.0 ** -126
        off = ((got[:, h] - want).abs() / tol).max().item()
        worst = max(worst, off if off == off else float("inf"))
    print(f"[weights] {tuple(q.shape)} n={n} largest error {worst:.3f} of its bound", flush=True)
    assert worst <= 1.0


KINDS = ["zero low", "zero", "zero high", "zero block", "far", "sink"]


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("amp", [1.0, 1e-3, 1e-4, 2e-5])
@pytest.mark.parametrize("n,new,hq,hkv,d,page", [
    (500, 1, 4, 1, 64, 64), (400, 3, 4, 2, 128, 16), (300, 1, 2, 1, 256, 32),
    (300, 30, 8, 1, 64, 16), (500, 40, 4, 1, 128, 64), (300, 24, 8, 2, 128, 32),
    (400, 50, 4, 1, 256, 64), (300, 40, 4, 1, 256, 16)])
def test_no_token_costs_the_others_their_bits(gpu, kind, amp, n, new, hq, hkv, d, page):
    import sparkq

    q, kc, ks, vc, vs = _case(kind, amp, n, new, hq, hkv, d, page, seed=n + new)
    q = q.to(torch.bfloat16)
    cache, table = _pool(gpu, kc, ks, vc, vs, page, 1)
    few = new * hq // hkv <= 16
    for dtype in (torch.float32, torch.bfloat16):
        out = sparkq.paged_quantized_sdpa(q.to(gpu), cache, table, _ints([0, new], gpu),
                                          _ints([n], gpu), scale=d ** -0.5, max_new=new,
                                          out_dtype=dtype)
        bits = 2.0 ** (-22 if few or dtype == torch.float32 else -11)
        _check(out, q, kc, ks, vc, vs, bits, 2.0 ** (-38 if few else -27))


@pytest.mark.parametrize("n,new,hq,hkv,d,page", [
    (700, 1, 4, 1, 64, 64), (900, 1, 8, 2, 128, 16), (500, 4, 8, 2, 128, 64), (600, 1, 4, 1, 256, 32),
    (900, 40, 8, 2, 128, 64), (300, 100, 4, 1, 64, 16), (400, 50, 4, 1, 256, 32)])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_the_contiguous_caches_bars(gpu, n, new, hq, hkv, d, page, dtype):
    """Weights of 22 bits: with few rows 16-bit outputs are within one unit of the
    rounded float64 ones, where these are not small, and float32 ones have 2e-5 of
    their norm whatever the rows. (A score of D products is off by some sqrt(D)
    2^-24 of its partial sums, independently of the others, as each weight is by
    2^-22, and the output, itself a sum of n terms of either sign, by about as much
    of itself: 16 * 2^-24 * 8 = 8e-6. Weights of 11 bits leave 1.5e-4.)"""
    import sparkq

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
    for out_dtype in (torch.float32, dtype):
        out = sparkq.paged_quantized_sdpa(q.to(gpu), cache, table, _ints([0, new], gpu),
                                          _ints([n], gpu), scale=d ** -0.5, max_new=new,
                                          out_dtype=out_dtype).cpu()
        if out_dtype == torch.float32:
            rel = rel_l2(out.numpy(), want.numpy())
            print(f"[weights] relative L2 error {rel:.2e}", flush=True)
            assert rel <= 2e-5
        elif new * hq // hkv <= 16:
            check_rounded16(out.view(torch.int16).numpy().view("uint16"), want.numpy(),
                            o.BF16 if dtype == torch.bfloat16 else o.F16)


@pytest.mark.parametrize("n,new,hq,hkv,d,page", [
    (400, 1, 4, 2, 128, 64), (400, 40, 4, 1, 64, 16), (400, 40, 8, 2, 128, 64), (400, 40, 4, 1, 256, 32)])
@pytest.mark.parametrize("size", [float("inf"), float("nan")])
@pytest.mark.parametrize("at", [range(64, 192), range(64, 65), range(0, 360)])
def test_visible_scales_that_are_not_finite(gpu, n, new, hq, hkv, d, page, size, at):
    """Whole blocks of them, codes of 0 among them: no row that sees one has a
    finite value."""
    import sparkq

    q, kc, ks, vc, vs = _case("sink", 1.0, n, new, hq, hkv, d, page, seed=3)
    vs[list(at)] = size
    vc[list(at)[::2]] = 0
    cache, table = _pool(gpu, kc, ks, vc, vs, page, 1)
    out = sparkq.paged_quantized_sdpa(q.half().to(gpu), cache, table, _ints([0, new], gpu),
                                      _ints([n], gpu), scale=d ** -0.5, max_new=new)
    assert not out.isfinite().any()
