"""CPU tests of the long-context operators over a paged cache: what they refuse before
any device call (in Python and at the C-ABI), the shapes of their custom ops, what the
cache class does with them, and the plain forms that the GPU tests compare with."""

import math
import random

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import paged_long_reference as long
import paged_reference as ref
import sparkq
from sparkq import paged
from test_paged_host import D, _bad_caches, _change, _refused, cache, i64, ints

BF = torch.bfloat16


# --- refusals in Python ------------------------------------------------------------

def _refuses(call, args, changes):
    for i, value, words in changes:
        with pytest.raises(ValueError, match=words):
            call(*_change(args, i, value))


BATCH = [(ints(3), "page_table"), (ints(3, 0), "page_table"), (ints(3, 2).long(), "int32"),
         (ints(2, 3).t(), "contiguous")]


def test_bounds_refuse():
    args = [cache(), torch.zeros((4, 2, 2, 64), dtype=BF), ints(3, 2), ints(4), ints(3)]
    call = lambda *a: sparkq.paged_key_bounds(*a, max_new=2)  # noqa: E731
    _refuses(call, args, [(0, c, words) for words, c in _bad_caches()])
    _refuses(call, args, [(2, t, words) for t, words in BATCH] + [
        (1, torch.zeros((4, 2, 2, 64)), "bfloat16"), (1, torch.zeros((4, 2, 64), dtype=BF), "shape"),
        (1, torch.zeros((3, 2, 2, 64), dtype=BF), "shape"), (1, None, "bfloat16"),
        (1, torch.zeros((4, 2, 64, 2), dtype=BF).transpose(2, 3), "contiguous"),
        (3, ints(3), "starts"), (4, ints(2), "lengths"), (4, ints(3), "GPU")])
    for bad in (0, True, 1.0, None):
        with pytest.raises(ValueError, match="max_new"):
            sparkq.paged_key_bounds(*args, max_new=bad)


def test_scores_refuse():
    args = [torch.zeros((5, 4, 64), dtype=BF), torch.zeros((4, 2, 2, 64), dtype=BF), ints(3, 2), ints(4),
            ints(3)]
    kw = {"page_size": 16, "scale": 0.1, "max_new": 2}
    call = lambda *a: sparkq.paged_page_scores(*a, **kw)  # noqa: E731
    _refuses(call, args, [(2, t, words) for t, words in BATCH] + [
        (0, torch.zeros((5, 3, 64), dtype=BF), "divisible"), (0, torch.zeros((5, 4, 32), dtype=BF), "queries"),
        (0, torch.zeros((5, 4, 64)), "float16 or bfloat16"), (1, torch.zeros((4, 2, 2, 64)), "bfloat16"),
        (1, torch.zeros((4, 2, 64), dtype=BF), "bounds"), (1, torch.zeros((4, 2, 3, 64), dtype=BF), "bounds"),
        (3, ints(5), "starts"), (4, ints(2), "lengths"), (4, ints(3), "GPU")])
    for change, words in [({"mask": "sliding"}, "mask"), ({"scale": math.nan}, "scale"),
                          ({"max_new": 0}, "max_new"), ({"page_size": 48}, "page_size"),
                          ({"page_size": 8}, "page_size"), ({"page_size": 16.0}, "page_size")]:
        with pytest.raises(ValueError, match=words):
            sparkq.paged_page_scores(*args, **{**kw, **change})


def test_select_refuses():
    x = torch.zeros((3, 2, 9))
    for args, kw, words in [
            ((x.double(), 2), {}, "float32"), ((x[0], 2), {}, "float32"), ((x[None, None], 2), {}, "float32"),
            ((x, 0), {}, "count"), ((x, 2.0), {}, "count"), ((x, True), {}, "count"),
            ((x, 2), {"first": -1}, "first"), ((x, 2), {"last": 1.0}, "last"),
            ((x, 2), {"first": 2, "last": 1}, "together"), ((x[..., :0], 2), {}, "empty"),
            ((x[:, :0], 2), {}, "empty"), ((x.transpose(1, 2), 2), {}, "contiguous"),
            ((x, 2), {"lengths": ints(2)}, "lengths"), ((x, 2), {"lengths": ints(3).long()}, "int32"),
            ((x, 2), {"lengths": ints(3)}, "GPU"), ((x[None], 2), {"lengths": ints(3)}, "GPU")]:
        with pytest.raises(ValueError, match=words):
            sparkq.select_top(*args, **kw)


def test_sparse_attention_refuses():
    args = [torch.zeros((5, 4, 64), dtype=BF), cache(), ints(5, 2, 3), ints(3, 2), ints(4), ints(3)]
    kw = {"scale": 0.1, "max_new": 2}
    call = lambda *a: sparkq.paged_sparse_sdpa(*a, **kw)  # noqa: E731
    _refuses(call, args, [(1, c, words) for words, c in _bad_caches()])
    _refuses(call, args, [(3, t, words) for t, words in BATCH] + [
        (0, torch.zeros((5, 3, 64), dtype=BF), "divisible"), (0, torch.zeros((5, 4, 64)), "float16 or bfloat16"),
        (2, ints(5, 2), "selected"), (2, ints(5, 2, 0), "selected"), (2, None, "selected"),
        (2, ints(4, 2, 3), "selected"), (2, ints(5, 1, 3), "selected"), (2, ints(5, 2, 3).long(), "selected"),
        (2, ints(5, 3, 2).transpose(1, 2), "contiguous"), (5, ints(3), "GPU")])
    for change, words in [({"mask": 1}, "mask"), ({"scale": math.inf}, "scale"), ({"max_new": 0}, "max_new"),
                          ({"out_dtype": torch.float16}, "out_dtype")]:
        with pytest.raises(ValueError, match=words):
            sparkq.paged_sparse_sdpa(*args, **{**kw, **change})


def test_mass_refuses():
    args = [torch.zeros((5, 4, 64), dtype=BF), torch.zeros((5, 4)), cache(), torch.zeros((3, 2, 32)), ints(3, 2),
            ints(4), ints(3)]
    call = lambda *a: sparkq.paged_kv_mass(*a, scale=0.1, max_new=2)  # noqa: E731
    _refuses(call, args, [(2, c, words) for words, c in _bad_caches()])
    _refuses(call, args, [(4, t, words) for t, words in BATCH] + [
        (0, torch.zeros((5, 3, 64), dtype=BF), "divisible"), (1, torch.zeros((5, 2)), "lse"),
        (1, torch.zeros((5, 4), dtype=BF), "lse"), (1, None, "lse"), (3, torch.zeros((3, 2, 31)), "mass"),
        (3, torch.zeros((3, 2, 32), dtype=BF), "mass"), (3, None, "mass"), (3, torch.zeros((2, 2, 32)), "mass"),
        (3, torch.zeros((3, 32, 2)).transpose(1, 2), "contiguous"), (6, ints(3), "GPU")])


def test_eviction_refuses():
    for layers in (None, 3):
        lead = () if layers is None else (layers,)
        args = [cache(layers=layers), ints(*lead, 3, 2, 5), ints(3, 2), ints(3)]
        _refuses(sparkq.kv_pages_evict, args, [(2, t, words) for t, words in BATCH[:3]] + [
            (1, ints(*lead, 3, 2, 0), "keep"), (1, ints(), "keep"), (1, None, "keep"),
            (1, ints(*lead, 2, 2, 5), "keep"), (1, ints(*lead, 3, 1, 5), "keep"),
            (1, ints(*lead, 3, 2, 5).long(), "keep"), (1, ints(9, *lead, 3, 2, 5), "keep"), (3, ints(2), "lengths"),
            (3, ints(3), "GPU")])
        for mass, words in [(torch.zeros((*lead, 3, 2, 31)), "mass"), (torch.zeros((*lead, 3, 2, 32)).half(), "mass"),
                            (torch.zeros((*lead, 3, 32, 2)).transpose(-1, -2), "contiguous"),
                            (torch.zeros((*lead, 3, 2, 32)), "GPU")]:
            with pytest.raises(ValueError, match=words):
                sparkq.kv_pages_evict(*args, mass=mass)
    for words, c in _bad_caches():
        with pytest.raises(ValueError, match=words):
            sparkq.kv_pages_evict(c, ints(3, 2, 5), ints(3, 2), ints(3))


# --- refusals at the C-ABI -----------------------------------------------------------

ST = [2048, 1024, 64, 32, 16, 1]


def test_abi_bounds():
    good = [D, D, D, D, D, D, 3, 2, 64, 4, 2, 2, 16, 2, i64(*ST), i64(256, 128), None]
    _refused("sparkq_paged_key_bounds", good, [
        (0, None, -1, "null"), (2, None, -1, "null"), (3, None, -1, "null"), (14, None, -1, "null"),
        (15, None, -1, "null"), (8, 96, -2, "head dim"), (12, 24, -1, "page_size"), (13, 0, -1, "max_new"),
        (11, 1, -1, "overlap"), (15, i64(256, 64), -1, "overlap"), (15, i64(256, 132), -1, "16-byte"),
        (2, D + 8, -1, "16-byte"), (14, i64(2040, 1024, 64, 32, 16, 1), -1, "16 bytes"),
        (14, i64(2048, 1024, 64, 32, -16, 1), -1, "negative"), (6, -1, -1, "shape")])


def test_abi_scores():
    good = [D, D, D, D, D, D, D, 5, 3, 4, 2, 64, 4, 2, 2, 16, 2, 1, 2, 0.1, i64(256, 64), i64(256, 128), None]
    _refused("sparkq_paged_page_scores", good, [
        (0, None, -1, "null"), (1, None, -1, "null"), (5, None, -1, "null"), (6, None, -1, "null"),
        (9, 3, -1, "divisible"), (11, 80, -2, "head dim"), (15, 24, -1, "page_size"), (16, 0, -1, "max_new"),
        (18, 0, -1, "float16 or bfloat16"), (19, math.inf, -1, "finite"), (20, i64(260, 64), -1, "16-byte"),
        (5, D + 4, -1, "16-byte"), (21, i64(256, 100), -1, "16-byte"), (21, i64(256, 64), -1, "overlap"),
        (7, 2 ** 30, -1, "large"), (14, 1, -1, "overlap")])


def test_abi_select():
    good = [D, D, D, 2, 3, 4, 100, 9, 1, 2, i64(1200, 400, 100), None]
    _refused("sparkq_select_top", good, [
        (0, None, -1, "null"), (2, None, -1, "null"), (10, None, -1, "null"), (6, 0, -1, "shape"),
        (7, 0, -1, "shape"), (5, 0, -1, "shape"), (3, -1, -1, "shape"), (8, -1, -1, "negative"),
        (9, 9, -1, "together"), (8, 10, -1, "together"), (10, i64(-1, 400, 100), -1, "negative"),
        (0, D + 2, -1, "aligned"), (4, 2 ** 22, -1, "large"), (6, 2 ** 31, -1, "large"), (7, 2 ** 30, -1, "large")])


def test_abi_sparse_attention():
    good = [D, D, D, D, D, D, D, D, D, D, 5, 3, 4, 2, 64, 7, 4, 2, 2, 16, 2, 1, 2, 2, 0.1, i64(256, 64),
            i64(14, 7), i64(*ST * 2), D, 1 << 20, None]
    _refused("sparkq_paged_sparse_sdpa", good, [
        (0, None, -1, "null"), (5, None, -1, "null"), (9, None, -1, "null"), (26, None, -1, "null"),
        (12, 3, -1, "divisible"), (14, 80, -2, "head dim"), (15, 0, -1, "count"), (15, 2 ** 28, -1, "count"),
        (20, 0, -1, "max_new"), (22, 0, -1, "float16 or bfloat16"), (23, 1, -1, "out dtype"),
        (26, i64(-1, 7), -1, "negative"), (27, i64(*ST, 2048, 1024, 64, 32, 16, 2), -2, "same strides")])
    from sparkq import _lib

    f = _lib.lib().sparkq_paged_sparse_workspace_bytes
    assert f(0, 32, 8, 128, 32, 64) == f(1, 33, 8, 128, 32, 64) == f(1, 32, 8, 128, 0, 64) == 0
    assert f(1, 32, 8, 128, 2, 64) == 0 and f(4096, 32, 8, 128, 8192, 16) == 0  # whole lists
    assert f(1, 32, 8, 128, 32, 64) == 8 * 16 * 4 * 130 * 4  # parts of 128 tokens, four heads each


def test_abi_mass():
    good = [D, D, D, D, D, D, D, D, 5, 3, 4, 2, 64, 4, 2, 2, 16, 2, 1, 2, 0.1, i64(256, 64), i64(64, 32), i64(*ST),
            None]
    _refused("sparkq_paged_kv_mass", good, [
        (0, None, -1, "null"), (1, None, -1, "null"), (2, None, -1, "null"), (4, None, -1, "null"),
        (22, None, -1, "null"), (23, None, -1, "null"), (10, 3, -1, "divisible"), (16, 24, -1, "page_size"),
        (17, 0, -1, "max_new"), (19, 0, -1, "float16 or bfloat16"), (22, i64(64, 31), -1, "aligned"),
        (22, i64(64, 30), -1, "overlap"), (22, i64(30, 32), -1, "overlap"), (4, D + 8, -1, "16-byte"),
        (21, i64(2 ** 32, 64), -1, "large"), (23, i64(2048, 1024, 64, 32, 16, 2), -2, "contiguous")])


def test_abi_eviction():
    st = i64(8192, 2048, 8192, 2048, 512, 64, 512, 64)
    good = [D, D, D, D, D, D, D, D, 2, D, D, D, st, i64(192, 64, 32), 3, 2, 64, 9, 2, 4, 2, 16, D, 4096, None]
    _refused("sparkq_kv_pages_evict", good, [
        (0, None, -1, "null"), (4, None, -1, "null"), (9, None, -1, "null"), (11, None, -1, "null"),
        (13, None, -1, "null"), (12, None, -1, "strides"), (16, 96, -2, "head dim"), (17, 0, -1, "shape"),
        (15, 0, -1, "shape"), (21, 8, -1, "page_size"), (21, 48, -1, "page_size"), (8, 1, -1, "overlap"),
        (22, None, -4, "workspace"), (23, 8, -4, "workspace"), (13, i64(192, 64, 31), -1, "overlap"),
        (13, i64(192, 31, 32), -1, "overlap"), (12, i64(8192, 2040, 8192, 2048, 512, 64, 512, 64), -1, "apart"),
        (14, 2 ** 30, -1, "large"), (20, 2 ** 20, -1, "large"), (12, i64(0, 2048, 8192, 2048, 512, 64, 512, 64), -1, "layers overlap"),
        (12, i64(8192, 2048, 8192, 2048, 512, 64, 48, 64), -1, "layers overlap")])


# --- custom ops ----------------------------------------------------------------------

def test_fakes_and_a_traced_step():
    m = lambda *shape, dtype=BF: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    c = [m(9, 2, 16, 64, dtype=torch.int8), m(9, 2, 16, dtype=torch.float16)] * 2
    i32 = lambda *shape: m(*shape, dtype=torch.int32)  # noqa: E731

    def step(q, bounds, mass, table, starts, lengths, *c):
        ops, at = torch.ops.sparkq, (table, starts, lengths)
        ops.paged_key_bounds(*c, bounds, *at, 2)
        scores, seen = ops.paged_page_scores(q, bounds, *at, 16, 0.125, 2, True)
        pages = ops.select_top(scores, 3, seen, 1, 1)
        out = ops.paged_sparse_sdpa(q, *c, pages, *at, 0.125, 2, True, torch.float32)
        more, lse = ops.paged_sdpa_lse(q, *c, *at, 0.125, 2, True, None)
        ops.paged_kv_mass(q, lse, *c, mass, *at, 0.125, 2, True)
        keep = ops.select_top(mass, 20, lengths, 0, 4)
        return (scores, seen, pages, out, more, lse, keep, *ops.kv_pages_evict(*c, keep, table, lengths, mass))

    args = (m(5, 4, 64), m(9, 2, 2, 64), m(3, 2, 112, dtype=torch.float32), i32(3, 7), i32(4), i32(3), *c)
    scores, seen, pages, out, more, lse, keep, table, lengths, missing = step(*args)
    assert scores.shape == (5, 2, 7) and scores.dtype == torch.float32 and seen.shape == (5,)
    assert pages.shape == (5, 2, 3) and pages.dtype == keep.dtype == torch.int32 and keep.shape == (3, 2, 20)
    assert out.shape == more.shape == (5, 4, 64) and out.dtype == torch.float32 and more.dtype == BF
    assert lse.shape == (5, 4) and lse.dtype == torch.float32
    assert table.shape == (3, 7) and lengths.shape == (3,) and missing.shape == (1,)
    graph = make_fx(step, tracing_mode="fake")(*args)
    names = {str(n.target) for n in graph.graph.nodes if n.op == "call_function"}
    for name in ("paged_key_bounds", "paged_page_scores", "select_top", "paged_sparse_sdpa", "paged_sdpa_lse",
                 "paged_kv_mass", "kv_pages_evict"):
        assert f"sparkq.{name}.default" in names


# --- the cache class -------------------------------------------------------------------

def test_the_cache_class_refuses():
    make = lambda **kw: sparkq.PagedKVCache(1, 4, 2, 64, page_size=16, max_pages=3, batch=2,  # noqa: E731
                                            device="cpu", **kw)
    q = torch.zeros((0, 4, 64), dtype=BF)
    with pytest.raises(ValueError, match="bounds=True"):
        make().attend_pages(0, q, scale=1.0, count=1)
    with pytest.raises(ValueError, match="mass=True"):
        make(bounds=True, mass=True).attend_pages(0, q, scale=1.0, count=1)
    with pytest.raises(ValueError, match="mass=True"):
        make(bounds=True).evict(5)
    c = make(bounds=True, mass=True)
    assert c.bounds.shape == (1, 4, 2, 2, 64) and c.bounds.dtype == BF
    assert c.mass.shape == (1, 2, 2, 48) and c.mass.dtype == torch.float32
    plain = make()
    assert plain.bounds is None and plain.mass is None


def test_a_full_row_refuses_until_undone_and_mass_follows_parents(monkeypatch):
    def fork(cache, table, lengths, parents=None, new_tokens=None):
        rows = new_tokens.shape[0]
        return (table.new_zeros((rows, table.shape[1])), new_tokens.clone(), table.new_zeros(1))

    monkeypatch.setattr(paged, "kv_pages_fork", fork)
    c = sparkq.PagedKVCache(2, 4, 1, 64, page_size=16, max_pages=2, batch=2, device="cpu", mass=True)
    c.step([4, 9])
    c.mass.copy_(torch.rand(c.mass.shape))
    old = c.mass.clone()
    c.step([1, 1, 1, 2], [1, 0, -1, 7])
    assert torch.equal(c.mass, old[:, [1, 0, 0, 1]])
    c.lengths = torch.tensor([30, 30, 30, 30], dtype=torch.int32)
    kept = c.mass.clone()
    c.step([5, 1, 1, 1])
    assert c.missing.item() == 4 - 3
    for call in (lambda: c.evict(3), lambda: c.attend(0, None, scale=1.0),
                 lambda: c.attend_pages(0, None, scale=1.0, count=1)):
        with pytest.raises(ValueError, match="undo"):
            call()
    c.undo()
    assert torch.equal(c.mass, kept)
    c.step([], [])
    assert c.mass.shape == (2, 0, 1, 32)
    c.step([3], [-1])
    assert c.mass.shape == (2, 1, 1, 32) and not c.mass.any()


# --- the plain forms ---------------------------------------------------------------------

def test_reference_bounds_hold_all_keys_and_are_tight():
    gen = torch.Generator().manual_seed(1)
    x = torch.randn(4000, generator=gen, dtype=torch.float64) * 10.0 ** torch.randint(-9, 9, (4000,), generator=gen)
    x = torch.cat([x, torch.tensor([0.0, 1.0, -1.0, 2.0 ** -24, 255.0, -256.0, 256.5, -255.5])])
    up, down = long.bf16_toward(x, True).double(), long.bf16_toward(x, False).double()
    assert (up >= x).all() and (down <= x).all()
    # each is the nearest such number: the other neighbour of bf16 lies on the wrong side
    for y, other in ((up, -1), (down, 1)):
        z = torch.nextafter(y.bfloat16(), torch.full_like(y, math.inf * other).bfloat16()).double()
        exact = y == x
        assert (exact | ((z < x) if other < 0 else (z > x))).all()
    exact = x.bfloat16().double() == x
    assert torch.equal(up[exact], x[exact]) and torch.equal(down[exact], x[exact])


@pytest.mark.parametrize("seed", range(5))
def test_reference_selection_is_a_stable_sort(seed):
    gen = torch.Generator().manual_seed(seed)
    x = torch.round(3 * torch.randn((2, 3, 2, 40), generator=gen)) / 2
    got = long.select(x, 9)
    want = x.sort(dim=-1, descending=True, stable=True).indices[..., :9].sort(-1).values
    assert torch.equal(got.long(), want)
    forced = long.select(x, 9, [40, 5, 20], 2, 3)
    for r, n in enumerate((40, 5, 20)):
        for row in forced[:, r].reshape(-1, 9).tolist():
            kept = [i for i in row if i >= 0]
            assert len(kept) == min(9, n) and {0, 1, n - 3, n - 2, n - 1} <= set(kept)


def test_reference_mass_of_all_rows_is_one_a_row():
    q, _, _, c, table, starts = ref.batch(1, [40, 9], [7, 9], 4, 2, 64, 16)
    kc, ks = c[:2]
    lse = torch.empty(16, 4, dtype=torch.float64)
    for b, n in ((0, 40), (1, 9)):
        ids = table[b][: -(-n // 16)]
        k = (kc[ids].double() * ks[ids].double()[..., None]).transpose(0, 1).reshape(2, -1, 64)[:, :n]
        for r in range(starts[b], starts[b + 1]):
            see = n - starts[b + 1] + r + 1
            for h in range(4):
                lse[r, h] = torch.logsumexp(k[h // 2, :see] @ q[r, h].double() * 0.125, 0)
    before = torch.rand((2, 2, 48))
    out, added, off = long.mass(q, lse, c, before, table, starts, [40, 9], 0.125)
    assert torch.allclose(added.sum(-1), torch.tensor([[14.0, 14.0], [18.0, 18.0]], dtype=torch.float64))
    assert (off > 0).all() and torch.equal(out[1, :, 9:], before[1, :, 9:].double())
    assert torch.allclose(out[0, :, :33], before[0, :, :33].double() + added[0, :, :33])
    assert torch.equal(out[0, :, 33:40], added[0, :, 33:40])


@pytest.mark.parametrize("seed", range(20))
def test_reference_eviction_leaves_others_pages_alone(seed):
    rng = random.Random(seed)
    page, pages, count = 16, 60, rng.randint(1, 60)
    lengths = [rng.randint(0, 100) for _ in range(6)]
    table = ref.tables(rng, lengths, page, pages, 8)
    for i in range(1, 6, 2):  # prefixes are shared
        k = min(lengths[i], lengths[i - 1]) // page
        table[i][:k] = table[i - 1][:k]
    out, after, missing = long.evict(table, lengths, count, pages, page)
    assert missing == 0
    held = [[p for p in r if p >= 0] for r in out]
    for i, n in enumerate(lengths):
        assert after[i] == min(n, count) and len(held[i]) == -(-after[i] // page)
        if n <= count:
            assert out[i] == table[i]
            continue
        for p in held[i]:  # what is written is nobody else's, before or after
            assert not any(p in o for j, o in enumerate(held) if j != i)
            assert not any(p in table[j] for j in range(6) if j != i)
