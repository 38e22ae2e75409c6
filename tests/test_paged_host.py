"""CPU tests of the paged cache's operators: what they refuse before any device
call (in Python and at the C-ABI), the shapes of their custom ops, and the plain
forms that the GPU tests compare with, pinned against other plain forms."""

import ctypes
import math
import random

import pytest
import torch
from torch.fx.experimental.proxy_tensor import make_fx

import paged_reference as ref
import sparkq

BF = torch.bfloat16


def ints(*shape):
    return torch.zeros(shape, dtype=torch.int32)


def cache(pages=4, hkv=2, page=16, d=64, layers=None):
    lead = (pages,) if layers is None else (layers, pages)
    return tuple(torch.zeros((*lead, hkv, page, d), dtype=torch.int8) if codes else
                 torch.zeros((*lead, hkv, page), dtype=torch.float16) for codes in (1, 0, 1, 0))


def _change(args, i, value):
    return [value if k == i else a for k, a in enumerate(args)]


# --- refusals in Python --------------------------------------------------------

def _norm_args():
    return [torch.zeros((3, 4, 64), dtype=BF), torch.zeros((3, 2, 64), dtype=BF),
            torch.zeros(64, dtype=BF), torch.zeros(64, dtype=BF), ints(3)]


@pytest.mark.parametrize("i,value,error,words", [
    (0, None, TypeError, "tensors"), (0, torch.zeros((3, 64), dtype=BF), ValueError, "queries"),
    (1, torch.zeros((2, 2, 64), dtype=BF), ValueError, "queries"),
    (1, torch.zeros((3, 2, 32), dtype=BF), ValueError, "queries"),
    (0, torch.zeros((3, 0, 64), dtype=BF), ValueError, "queries"),
    (1, torch.zeros((3, 2, 64), dtype=torch.float16), ValueError, "one dtype"),
    (2, torch.zeros(32, dtype=BF), ValueError, "shape"),
    (3, torch.zeros(64), ValueError, "one dtype"),
    (4, ints(2), ValueError, "positions"), (4, torch.zeros(3), ValueError, "positions"),
    (4, ints(3), ValueError, "GPU"),
])
def test_norm_rope_refuses(i, value, error, words):
    with pytest.raises(error, match=words):
        sparkq.qk_norm_rope(*_change(_norm_args(), i, value), dims=64, eps=1e-6)


def test_norm_rope_dims_are_ints():
    with pytest.raises(ValueError, match="dims"):
        sparkq.qk_norm_rope(*_norm_args(), dims=64.0, eps=1e-6)


def _bad_caches():
    c = cache()
    yield "the cache is", c[:3]
    yield "the cache is", (*c[:3], None)
    yield "int8 codes", (c[0].float(), *c[1:])
    yield "int8 codes", (c[0], c[1].float(), *c[2:])
    yield "int8 codes", (c[0], c[1][..., :8], *c[2:])
    yield "int8 codes", (*c[:2], c[2][:, :1], c[3])
    yield "int8 codes", tuple(t[0] for t in c)


def _append_args():
    return [torch.zeros((5, 2, 64), dtype=BF), torch.zeros((5, 2, 64), dtype=BF), cache(),
            ints(3, 2), ints(4), ints(3)]


def test_append_refuses():
    call = sparkq.paged_kv_append
    for words, c in _bad_caches():
        with pytest.raises(ValueError, match=words):
            call(*_change(_append_args(), 2, c))
    for i, value, words in [
            (0, torch.zeros((5, 1, 64), dtype=BF), "like the cache"),
            (0, torch.zeros((5, 128), dtype=BF), "like the cache"),
            (1, torch.zeros((4, 2, 64), dtype=BF), "like the cache"),
            (1, torch.zeros((5, 2, 64)), "both alike"),
            (3, ints(3), "expected page_table"), (3, ints(3, 0), "expected page_table"),
            (3, ints(3, 2).long(), "int32"), (4, ints(3), "starts"), (5, ints(4), "lengths"),
            (5, torch.zeros(3), "lengths"), (3, ints(2, 3).t(), "contiguous"),
            (5, ints(3), "GPU")]:
        with pytest.raises(ValueError, match=words):
            call(*_change(_append_args(), i, value))
    with pytest.raises(ValueError, match="float16, bfloat16 or float32"):
        call(*_change(_change(_append_args(), 0, torch.zeros((5, 2, 64), dtype=torch.float64)), 1,
                      torch.zeros((5, 2, 64), dtype=torch.float64)))


def _sdpa(i=None, value=None, **kw):
    args = [torch.zeros((5, 4, 64), dtype=BF), cache(), ints(3, 2), ints(4), ints(3)]
    return sparkq.paged_quantized_sdpa(*(args if i is None else _change(args, i, value)),
                                       **{"scale": 0.1, "max_new": 2, **kw})


def test_attention_refuses():
    for words, c in _bad_caches():
        with pytest.raises(ValueError, match=words):
            _sdpa(1, c)
    for i, value, words in [
            (0, torch.zeros((5, 3, 64), dtype=BF), "divisible"),
            (0, torch.zeros((5, 0, 64), dtype=BF), "divisible"),
            (0, torch.zeros((5, 4, 32), dtype=BF), "queries"),
            (0, torch.zeros((5, 4, 64)), "float16 or bfloat16"), (2, ints(3), "page_table"),
            (3, ints(5), "starts"), (4, ints(2), "lengths")]:
        with pytest.raises(ValueError, match=words):
            _sdpa(i, value)
    for kw, words in [({"mask": "sliding"}, "mask"), ({"scale": math.inf}, "scale"),
                      ({"scale": "1"}, "scale"), ({"max_new": 0}, "max_new"),
                      ({"max_new": True}, "max_new"), ({"max_new": 1.0}, "max_new"),
                      ({"out_dtype": torch.float16}, "out_dtype"), ({}, "GPU")]:
        with pytest.raises(ValueError, match=words):
            _sdpa(**kw)


def test_page_operators_refuse():
    for words, c in _bad_caches():
        for call in (sparkq.kv_pages_fork, sparkq.kv_pages_compact):
            with pytest.raises(ValueError, match=words):
                call(c, ints(3, 2), ints(3))
    c = cache(layers=3)
    for call in (sparkq.kv_pages_fork, sparkq.kv_pages_compact):
        for args, words in [((ints(3), ints(3)), "page_table"), ((ints(3, 0), ints(3)), "page_table"),
                            ((ints(3, 2), ints(2)), "lengths"), ((ints(3, 2), ints(3)), "GPU")]:
            with pytest.raises(ValueError, match=words):
                call(c, *args)
        with pytest.raises(ValueError, match="contiguous"):
            call(tuple(t.transpose(2, 3) if t.ndim == 5 else t for t in cache(hkv=16, layers=1)),
                 ints(3, 2), ints(3))
    with pytest.raises(ValueError, match="parents"):
        sparkq.kv_pages_fork(c, ints(3, 2), ints(3), ints(3, 1))
    with pytest.raises(ValueError, match="new_tokens"):
        sparkq.kv_pages_fork(c, ints(3, 2), ints(3), ints(5), ints(3))


def test_the_cache_class_refuses():
    make = sparkq.PagedKVCache
    for args, kw, words in [((0, 4, 2, 64), {}, "positive"), ((1, 4, 2, 96), {}, "head_dim"),
                            ((1, 4, 2, 64), {"page_size": 48}, "page_size"),
                            ((1, 4, 2, 64), {"batch": -1}, "positive")]:
        with pytest.raises(ValueError, match=words):
            make(*args, device="cpu", **kw)
    c = make(2, 4, 2, 64, page_size=16, max_pages=3, batch=2, device="cpu")
    assert c.layer(1)[0].shape == (4, 2, 16, 64) and c.page_table.tolist() == [[-1] * 3] * 2
    with pytest.raises(ValueError, match="each of the 2 rows"):
        c.step([1])
    with pytest.raises(ValueError, match="each of the 3 rows"):
        c.step([1, 1], parents=[0, 1, 1])
    with pytest.raises(ValueError, match="negative"):
        c.step([1, -1])


# --- refusals at the C-ABI -------------------------------------------------------

def _rc(name, *args):
    from sparkq import _lib

    rc = getattr(_lib.lib(), name)(*args)
    return rc, _lib.lib().sparkq_last_error().decode()


D = 4096  # a pointer that nothing reads


def _refused(name, good, changes):
    """Each change of one argument is refused with its code and words."""
    for i, value, code, words in changes:
        rc, msg = _rc(name, *_change(good, i, value))
        assert rc == code and words in msg, (i, value, rc, msg)


def i64(*v):
    return (ctypes.c_int64 * len(v))(*v)


def test_abi_norm_rope():
    good = [D, D, D, D, D, 32, D, D, 3, 4, 2, 64, 64, 0, 1e-6, 1e4, 1.0, 2, i64(256, 64, 128, 64), None]
    _refused("sparkq_qk_norm_rope", good, [
        (0, None, -1, "null"), (18, None, -1, "null"), (5, 16, -1, "int32 or int64"),
        (8, -1, -1, "shape"), (9, 0, -1, "shape"), (8, 2 ** 40, -1, "large"), (12, 63, -1, "even"),
        (12, 66, -1, "dims"), (12, 0, -1, "dims"), (14, math.nan, -1, "eps"), (15, 0.0, -1, "base"),
        (16, math.inf, -1, "scale"), (17, 0, -1, "BF16")])


def test_abi_append():
    st = i64(*[2048, 1024, 64, 32, 16, 1] * 2)
    good = [D, D, D, D, D, D, D, D, D, 5, 3, 2, 64, 4, 2, 2, 16, 2, i64(128, 64, 128, 64), st, None]
    _refused("sparkq_paged_kv_append", good, [
        (0, None, -1, "null"), (2, None, -1, "null"), (6, None, -1, "null"), (7, None, -1, "null"),
        (9, -1, -1, "shape"), (12, 96, -2, "head dim"), (13, 0, -1, "shape"), (14, 0, -1, "shape"),
        (15, 1, -1, "overlap"), (16, 48, -1, "page_size"), (16, 8, -1, "page_size"),
        (16, 2048, -1, "page_size"), (14, 2 ** 28, -1, "2^31"), (17, 3, -1, "float"),
        (18, i64(130, 64, 128, 64), -1, "16-byte"), (18, i64(128, 64, -128, 64), -1, "16-byte"),
        (19, i64(*[2040, 1024, 64, 32, 16, 1] * 2), -1, "16 bytes"),
        (19, i64(*[2048, -1024, 64, 32, 16, 1] * 2), -1, "negative"), (0, D + 8, -1, "16-byte"),
        (2, D + 4, -1, "16-byte"), (9, 2 ** 31 - 1, -1, "large")])


def test_abi_attention():
    st = [2048, 1024, 64, 32, 16, 1]
    good = [D, D, D, D, D, D, D, D, D, 5, 3, 4, 2, 64, 4, 2, 2, 16, 2, 1, 2, 2, 0.1, i64(256, 64),
            i64(*st * 2), None, 0, None]
    wide = [2 ** 36 * 16, 1024, 64, 32, 16, 1]
    _refused("sparkq_paged_sdpa", good, [
        (0, None, -1, "null"), (8, None, -1, "null"), (11, 3, -1, "divisible"), (13, 80, -2, "head dim"),
        (17, 24, -1, "page_size"), (18, 0, -1, "max_new"), (20, 0, -1, "float16 or bfloat16"),
        (21, 1, -1, "out dtype"), (22, math.nan, -1, "finite"), (23, i64(260, 64), -1, "16-byte"),
        (24, i64(*st, 2048, 1024, 64, 32, 16, 2), -2, "same strides"),
        (24, i64(*[2048, 1024, 64, 32, 16, 2] * 2), -2, "contiguous"),
        (24, i64(*[2048, 1024, 64, 33, 16, 1] * 2), -2, "multiples of 8"),
        (24, i64(*wide * 2), -2, "32 GiB"), (2, D + 8, -2, "16-byte"), (10, 2 ** 30, -1, "large")])


def test_abi_pages():
    st = i64(8192, 2048, 8192, 2048, 512, 64, 512, 64)
    fork = [D, D, D, D, D, D, D, D, 2, D, D, D, st, 3, 3, 2, 4, 2, 16, 2048, 64, D, 4096, None]
    _refused("sparkq_kv_pages_fork", fork, [
        (0, None, -1, "null"), (4, None, -1, "null"), (9, None, -1, "null"), (11, None, -1, "null"),
        (22, 0, -4, "workspace"), (21, None, -4, "workspace"),
        (18, 100, -1, "page_size"), (19, 2040, -1, "multiples of 16"), (17, 0, -1, "shape"),
        (8, 1, -1, "overlap"), (12, i64(8192, 2040, 8192, 2048, 512, 64, 512, 64), -1, "apart"),
        (12, i64(8192, 1024, 8192, 2048, 512, 64, 512, 64), -1, "apart"), (12, None, -1, "strides"),
        (15, 2 ** 30, -1, "large")])
    rows = _change(_change(fork, 6, None), 14, 4)  # 4 rows of 3 sequences without parents
    assert _rc("sparkq_kv_pages_fork", *rows)[0] == -1
    compact = [D, D, D, D, D, D, 2, D, D, st, 3, 2, 4, 2, 16, 2048, 64, D, 4096, None]
    _refused("sparkq_kv_pages_compact", compact, [
        (3, None, -1, "null"), (5, None, -1, "null"), (8, None, -1, "null"), (18, 8, -4, "workspace"),
        (14, 0, -1, "page_size"), (17, D + 4, -1, "16-byte")])


def test_workspaces():
    from sparkq import _lib

    f = _lib.lib().sparkq_paged_sdpa_workspace_bytes
    assert f(0, 1, 32, 8, 128, 1, 4096) == f(1, 1, 33, 8, 128, 1, 4096) == 0
    assert f(1, 1, 32, 8, 128, 1, 128) == 0  # one part holds it all
    # no more parts than the batch's tokens have, 16 rows each
    assert f(1, 1, 32, 8, 128, 1, 4096) == 8 * 32 * 16 * 130 * 4
    assert 0 < f(4096, 64, 32, 8, 128, 64, 1 << 20) < 1 << 28
    g = _lib.lib().sparkq_kv_pages_workspace_bytes
    assert g(-1, 4) == g(4, 0) == 0 and g(4, 100) >= 4 * (3 * 100 + 3 * 4)


# --- custom ops ------------------------------------------------------------------

def test_fakes_and_a_traced_step():
    m = lambda *shape, dtype=BF: torch.empty(shape, dtype=dtype, device="meta")  # noqa: E731
    c = [m(9, 2, 16, 64, dtype=torch.int8), m(9, 2, 16, dtype=torch.float16)] * 2
    i32 = lambda *shape: m(*shape, dtype=torch.int32)  # noqa: E731

    def step(qkv, w, pos, kc, ks, vc, vs, table, lengths, parents, new, starts):
        ops = torch.ops.sparkq
        table, lengths, missing = ops.kv_pages_fork(kc, ks, vc, vs, table, lengths, parents, new)
        q, k = ops.qk_norm_rope(qkv[:, :4], qkv[:, 4:6], w, w, pos, 64, 1e-6, 1e4, 1.0, False)
        ops.paged_kv_append(k, qkv[:, 6:], kc, ks, vc, vs, table, starts, lengths)
        out = ops.paged_sdpa(q, kc, ks, vc, vs, table, starts, lengths, 0.125, 2, True, torch.float32)
        table, used = ops.kv_pages_compact(kc, ks, vc, vs, table, lengths)
        return out, table, lengths, missing, used

    args = (m(5, 8, 64), m(64), i32(5), *c, i32(3, 7), i32(3), i32(4), i32(4), i32(5))
    out, table, lengths, missing, used = step(*args)
    assert out.shape == (5, 4, 64) and out.dtype == torch.float32
    assert table.shape == (4, 7) and lengths.shape == (4,) and missing.shape == used.shape == (1,)
    graph = make_fx(step, tracing_mode="fake")(*args)
    names = {str(n.target) for n in graph.graph.nodes if n.op == "call_function"}
    for name in ("qk_norm_rope", "paged_kv_append", "paged_sdpa", "kv_pages_fork", "kv_pages_compact"):
        assert f"sparkq.{name}.default" in names


# --- the plain forms ---------------------------------------------------------------

def test_reference_attention_is_softmax_attention():
    q, _, _, cache_, table, starts = ref.batch(1, [40, 9], [7, 9], 4, 2, 64, 16)
    out, mass, _, done, _ = ref.attention(q, cache_, table, starts, [40, 9], 0.125)
    assert done.all() and (mass >= out.abs() - 1e-12).all()
    kc, ks, vc, vs = cache_
    for b, n in ((0, 40), (1, 9)):
        ids = table[b][: -(-n // 16)]
        k, v = ((c[ids].double() * s[ids].double()[..., None]).transpose(0, 1).reshape(2, -1, 64)[:, :n]
                .repeat_interleave(2, 0) for c, s in ((kc, ks), (vc, vs)))
        rows = slice(starts[b], starts[b + 1])
        new = rows.stop - rows.start
        mask = torch.ones((new, n), dtype=torch.bool).tril(n - new)
        want = torch.nn.functional.scaled_dot_product_attention(
            q[rows].double().transpose(0, 1), k, v, attn_mask=mask, scale=0.125)
        assert torch.allclose(out[rows], want.transpose(0, 1), atol=1e-12)


def test_reference_norm_rope_keeps_norms_and_relative_positions():
    x = torch.randn((2, 1, 8), dtype=torch.float64)
    one = torch.ones(8, dtype=torch.float64)
    for kind in (False, True):
        far, _ = ref.norm_rope(x, one, torch.tensor([3, 3]), 8, 0.0, 100.0, traditional=kind)
        near, _ = ref.norm_rope(x, one, torch.tensor([0, 0]), 8, 0.0, 100.0, traditional=kind)
        assert torch.allclose(near, x / x.pow(2).mean(-1, keepdim=True).sqrt())
        assert torch.allclose(far.norm(dim=-1), torch.full((2, 1), 8 ** 0.5, dtype=torch.float64))
        a, _ = ref.norm_rope(x, one, torch.tensor([7, 4]), 8, 0.0, 100.0, traditional=kind)
        b, _ = ref.norm_rope(x, one, torch.tensor([13, 10]), 8, 0.0, 100.0, traditional=kind)
        assert torch.allclose((a[0] * a[1]).sum(), (b[0] * b[1]).sum())


@pytest.mark.parametrize("seed", range(30))
def test_reference_fork_leaves_nobody_anothers_page_to_write(seed):
    rng = random.Random(seed)
    page, pages, b = 16, 60, 6
    table = ref.tables(rng, [rng.randint(0, 60) for _ in range(b)], page, pages, 5)
    lengths = [rng.randint(0, sum(p >= 0 for p in r) * page) for r in table]
    parents = [rng.randrange(-1, b) for _ in range(8)]
    fresh = [rng.randint(0, 20) for _ in range(8)]
    out, after, missing, pairs = ref.fork(table, lengths, parents, fresh, pages, page)
    assert missing == 0
    held = [[p for p in r if p >= 0] for r in out]
    for i, r in enumerate(held):
        assert len(r) == -(-after[i] // page)
        before = lengths[parents[i]] if parents[i] >= 0 else 0
        assert after[i] == min(before + fresh[i], 5 * page)
        if after[i] > before:  # every page it writes is its own
            for p in r[before // page:]:
                assert sum(p in o for o in held) == 1
    copied = dict((new, old) for old, new in pairs)
    for i, r in enumerate(held):  # and its old tokens are there
        before = lengths[parents[i]] if parents[i] >= 0 else 0
        for j in range(-(-before // page)):
            assert copied.get(r[j], r[j]) == table[parents[i]][j]
    got, used, moved = ref.compact(out, after, pages, page)
    new = dict(moved)
    assert sorted({p for r in got for p in r if p >= 0}) == list(range(used))
    assert all(g == new.get(o, o) for a, c in zip(got, out) for g, o in zip(a, c))
