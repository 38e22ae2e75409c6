"""The ways the long-context operators are called: together over steps of a
PagedKVCache, captured and replayed, two graphs at once, on a side stream, as custom
ops, with nothing in the batch, and the calls they refuse on the device."""

import math
import random

import pytest
import torch

import paged_long_reference as long
import paged_reference as ref
import sparkq
from test_gpu_paged_long import check_mass, check_scores, check_sparse
from test_gpu_paged_sdpa import check

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
HQ, HKV, D, PAGE = 8, 2, 64, 16
SCALE = D ** -0.5


def _ints(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


def _cpu(cache, layer):
    return tuple(t[layer].cpu() for t in cache.cache)


def _step(cache, gen, news, parents=None):
    """A step of every layer; the packed rows' starts as a list."""
    cache.step(news, parents)
    assert cache.missing.item() == 0
    kv = [torch.randn((2, sum(news), HKV, D), generator=gen).to(BF).to(cache.mass_or_dev)
          for _ in range(2)]
    for layer, (k, v) in enumerate(kv):
        cache.append(layer, k, v)
    return cache.starts.tolist()


class Cache(sparkq.PagedKVCache):
    @property
    def mass_or_dev(self):
        return self.cache[0].device


def test_pages_attended_over_steps(gpu):
    """Prompts, decode steps, sequences that continue others or end, pages that are
    copied and moved: the bounds are always those of the pages as they are, and the
    scores, pages and outputs follow from them."""
    gen = torch.Generator().manual_seed(1)
    cache = Cache(2, 60, HKV, D, page_size=PAGE, max_pages=12, batch=3, device=gpu, bounds=True)
    plan = [([100, 33, 7], None), ([1, 1, 1], None), ([1, 4, 1, 2], [0, 0, 2, 1]),
            ([1, 0, 3], [3, 0, 1]), "compact", ([1, 1, 1], None), ([20, 1], [2, 0])]
    for item in plan:
        if item == "compact":
            cache.compact()
        else:
            starts = _step(cache, gen, *item)
        table, lengths = cache.page_table.tolist(), cache.lengths.tolist()
        whole = [0]
        for n in lengths:
            whole.append(whole[-1] + n)
        for layer in range(2):
            kv = _cpu(cache, layer)
            got = cache.bounds[layer].cpu()
            want = long.bounds(kv, got, table, whole, lengths)  # every page that is held
            assert torch.equal(got, want)
            q = torch.randn((starts[-1], HQ, D), generator=gen).to(BF)
            batch = cache.page_table, cache.starts, cache.lengths
            kw = {"scale": SCALE, "max_new": cache.max_new}
            scores, seen = sparkq.paged_page_scores(q.to(gpu), cache.bounds[layer], *batch,
                                                    page_size=PAGE, **kw)
            check_scores(scores, seen, q, got, table, starts, lengths, PAGE, SCALE)
            pages = sparkq.select_top(scores, 5, lengths=seen, first=1, last=2).cpu()
            assert torch.equal(pages, long.select(scores.cpu()[None], 5, seen.tolist(), 1, 2)[0])
            out = cache.attend_pages(layer, q.to(gpu), scale=SCALE, count=5)
            check_sparse(out, q, kv, pages, table, starts, lengths, SCALE)
            # with all pages it is the attention
            out = cache.attend_pages(layer, q.to(gpu), scale=SCALE, count=12)
            check(out, q, kv, table, starts, lengths, SCALE)


def test_weights_and_eviction_over_steps(gpu):
    """Mass follows rows through steps; eviction leaves each head the tokens that
    gathered most; the pages it frees are dealt again, shared ones are not written."""
    gen = torch.Generator().manual_seed(2)
    cache = Cache(2, 40, HKV, D, page_size=PAGE, max_pages=10, batch=2, device=gpu, mass=True,
                  bounds=True)
    with pytest.raises(ValueError, match="mass=True"):
        cache.attend_pages(0, torch.zeros((0, HQ, D), dtype=BF, device=gpu), scale=1.0, count=1)
    mass = cache.mass.cpu()
    plan = [([90, 40], None), ([1, 1], None), ([1, 2, 1], [0, 0, 1]), (50, 2, 5), ([1, 1, 1], None),
            ([1, 30, 1, 1], [1, 0, 2, -1]), (40, 0, 40), ([1, 1, 1, 1], None)]
    for item in plan:
        if isinstance(item[0], int):
            table, lengths = cache.page_table.tolist(), cache.lengths.tolist()
            before = [t.cpu() for t in cache.cache]
            keep = long.select(mass, item[0], lengths, *item[1:])
            assert cache.evict(item[0], first=item[1], last=item[2]).item() == 0
            want = long.evict(table, lengths, item[0], 40, PAGE)
            assert cache.page_table.tolist() == want[0] and cache.lengths.tolist() == want[1]
            moved, mass = long.moved(before, mass, keep, table, lengths, *want[:2])
            assert all(torch.equal(a.cpu(), b) for a, b in zip(cache.cache, moved))
            assert torch.equal(cache.mass.cpu(), mass)
            assert cache.starts.tolist() == [0] * len(cache.starts)
            table, lengths = want[:2]
            whole = [0]
            for n in lengths:
                whole.append(whole[-1] + n)
            for layer in range(2):
                got = cache.bounds[layer].cpu()
                assert torch.equal(got, long.bounds(_cpu(cache, layer), got, table, whole, lengths))
            continue
        starts = _step(cache, gen, *item)
        if item[1] is not None:
            mass = mass[:, [max(p, 0) for p in item[1]]]
        table, lengths = cache.page_table.tolist(), cache.lengths.tolist()
        assert torch.equal(cache.mass.cpu(), mass)
        for layer in range(2):
            q = torch.randn((starts[-1], HQ, D), generator=gen).to(BF)
            out = cache.attend(layer, q.to(gpu), scale=SCALE)
            kv = _cpu(cache, layer)
            check(out, q, kv, table, starts, lengths, SCALE)
            _, lse = sparkq.paged_quantized_sdpa(
                q.to(gpu), cache.layer(layer), cache.page_table, cache.starts, cache.lengths,
                scale=SCALE, max_new=cache.max_new, return_lse=True)
            check_mass(cache.mass[layer], q, lse.cpu(), kv, mass[layer], table, starts, lengths, SCALE)
        mass = cache.mass.cpu()


def test_a_short_step_is_taken_back_and_tokens_evicted(gpu):
    gen = torch.Generator().manual_seed(3)
    cache = Cache(1, 10, HKV, D, page_size=PAGE, max_pages=6, batch=2, device=gpu, mass=True)
    cache.step([80, 80])
    k = torch.randn((160, HKV, D), generator=gen).to(BF).to(gpu)
    cache.append(0, k, k)
    cache.attend(0, torch.randn((160, HQ, D), generator=gen).to(BF).to(gpu), scale=SCALE)
    mass = cache.mass.clone()
    cache.step([1, 1], [1, 0])
    assert cache.missing.item() == 2
    cache.undo()
    assert torch.equal(cache.mass, mass)
    assert cache.evict(33, first=1, last=8).item() == 0
    assert cache.lengths.tolist() == [33, 33]
    with pytest.raises(ValueError, match="no step"):
        cache.undo()
    cache.step([40, 1], [0, 0])
    assert cache.missing.item() == 0 and cache.lengths.tolist() == [73, 34]
    # rows that share every page: eviction asks for pages of its own
    cache.step([0, 0, 0], [0, 0, 0])
    assert cache.evict(60).item() == 3 * 4 - 5 and cache.lengths.tolist() == [73] * 3
    cache.step([0], [0])
    assert cache.evict(60).item() == 0 and cache.lengths.tolist() == [60]


class Step:
    """The operators of one decode step and an eviction of four sequences in two
    layers, on tensors that stay where they are."""

    def __init__(self, gpu, seed, new):
        self.gen, self.new = torch.Generator().manual_seed(seed), new
        self.starts = _ints([new * i for i in range(5)], gpu)
        self.pool = [t.to(gpu) for t in ref.pool(self.gen, 90, HKV, PAGE, D, layers=2)]
        self.bounds = torch.zeros((2, 90, HKV, 2, D), dtype=BF, device=gpu)
        self.mass = torch.zeros((2, 4, HKV, 24 * PAGE), device=gpu)
        self.table = torch.full((4, 24), -1, dtype=torch.int32, device=gpu)
        self.lengths = torch.zeros(4, dtype=torch.int32, device=gpu)
        self.q = torch.zeros((4 * new, HQ, D), dtype=BF, device=gpu)
        self.fill(0)

    def fill(self, k):
        lengths = [300 + 7 * k, 80 + k, 33, 200 - 9 * k]
        ids = torch.randperm(85, generator=self.gen).tolist()
        rows = [[ids.pop() for _ in range(-(-n // PAGE))] for n in lengths]
        rows[3][:4] = rows[0][:4]  # a shared prefix
        self.table.copy_(torch.tensor([r + [-1] * (24 - len(r)) for r in rows], dtype=torch.int32))
        self.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        self.q.copy_(torch.randn(self.q.shape, generator=self.gen))
        self.mass.copy_(torch.rand(self.mass.shape, generator=self.gen))
        self.bounds.copy_(torch.randn(self.bounds.shape, generator=self.gen))
        for t, c in zip(self.pool, ref.pool(self.gen, 90, HKV, PAGE, D, layers=2)):
            t.copy_(c)

    def __call__(self):
        out, batch = [], (self.table, self.starts, self.lengths)
        kw = {"scale": SCALE, "max_new": self.new}
        for layer in range(2):
            cache = tuple(t[layer] for t in self.pool)
            sparkq.paged_key_bounds(cache, self.bounds[layer], *batch, max_new=self.new)
            scores, seen = sparkq.paged_page_scores(self.q, self.bounds[layer], *batch,
                                                    page_size=PAGE, **kw)
            pages = sparkq.select_top(scores, 6, lengths=seen, first=1, last=2)
            out += [scores, pages, sparkq.paged_sparse_sdpa(self.q, cache, pages, *batch, **kw)]
            o, lse = sparkq.paged_quantized_sdpa(self.q, cache, *batch, return_lse=True, **kw)
            sparkq.paged_kv_mass(self.q, lse, cache, self.mass[layer], *batch, **kw)
            out += [o, lse]
        keep = sparkq.select_top(self.mass, 70, lengths=self.lengths, first=2, last=5)
        return [*out, keep, *sparkq.kv_pages_evict(self.pool, keep, self.table, self.lengths,
                                                   mass=self.mass)]

    def state(self):
        return [t.clone() for t in (*self.pool, self.bounds, self.mass)]

    def restore(self, state):
        for t, s in zip((*self.pool, self.bounds, self.mass), state):
            t.copy_(s)


def _equal(got, want):
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("new", [1, 5, 40])
def test_a_captured_step(gpu, new):
    """Every replay, on batches that change in between, with eager steps and
    synchronisation between them, is the eager step bit for bit."""
    step = Step(gpu, 4, new)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        outs = step()
    for k in range(4):
        step.fill(k)
        before = step.state()
        want = [t.clone() for t in step()]
        after = step.state()
        step.restore(before)
        junk = torch.randn(1 << 20, device=gpu).sum()
        graph.replay()
        torch.cuda.synchronize()
        assert float(junk) == float(junk)
        _equal(outs, want)
        _equal(step.state(), after)
        assert want[-1].item() == 0


def test_two_graphs_and_a_side_stream(gpu):
    """Graphs of two batches replay on two streams at once, and a step runs on a stream
    of its own: their scratch is their own."""
    steps = [Step(gpu, 5, 1), Step(gpu, 6, 12)]
    torch.cuda.synchronize()
    side, graphs, outs, befores, wants, afters = torch.cuda.Stream(), [], [], [], [], []
    for step in steps:
        befores.append(step.state())
        wants.append([t.clone() for t in step()])
        afters.append(step.state())
        torch.cuda.synchronize()
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=side):
            outs.append(step())
    streams = [torch.cuda.Stream() for _ in steps]
    for _ in range(4):
        for step, before in zip(steps, befores):
            step.restore(before)
        torch.cuda.synchronize()
        for graph, stream in zip(graphs, streams):
            with torch.cuda.stream(stream):
                graph.replay()
        torch.cuda.synchronize()
        for step, out, want, after in zip(steps, outs, wants, afters):
            _equal(out, want)
            _equal(step.state(), after)
    for step, before, want in zip(steps, befores, wants):
        step.restore(before)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = step()
        side.synchronize()
        _equal(got, want)


def test_custom_ops_are_the_operators(gpu):
    ops = torch.ops.sparkq
    utils = ("test_schema", "test_autograd_registration", "test_faketensor")
    step = Step(gpu, 7, 3)
    before = step.state()
    want = [t.clone() for t in step()]
    after = step.state()
    step.restore(before)
    batch, got = (step.table, step.starts, step.lengths), []
    for layer in range(2):
        cache = tuple(t[layer] for t in step.pool)
        ops.paged_key_bounds(*cache, step.bounds[layer], *batch, 3)
        scores, seen = ops.paged_page_scores(step.q, step.bounds[layer], *batch, PAGE, SCALE, 3, True)
        pages = ops.select_top(scores, 6, seen, 1, 2)
        got += [scores, pages, ops.paged_sparse_sdpa(step.q, *cache, pages, *batch, SCALE, 3, True, None)]
        o, lse = ops.paged_sdpa_lse(step.q, *cache, *batch, SCALE, 3, True, None)
        ops.paged_kv_mass(step.q, lse, *cache, step.mass[layer], *batch, SCALE, 3, True)
        got += [o, lse]
    keep = ops.select_top(step.mass, 70, step.lengths, 2, 5)
    got += [keep, *ops.kv_pages_evict(*step.pool, keep, step.table, step.lengths, step.mass)]
    _equal(got, want)
    _equal(step.state(), after)
    step.restore(before)
    for op, args in [
            (ops.paged_key_bounds, (*cache, step.bounds[0].clone(), *batch, 3)),
            (ops.paged_page_scores, (step.q, step.bounds[0], *batch, PAGE, SCALE, 3, False)),
            (ops.select_top, (scores, 6, None, 0, 0)), (ops.select_top, (step.mass, 9, step.lengths, 1, 2)),
            (ops.paged_sparse_sdpa, (step.q, *cache, pages, *batch, SCALE, 3, False, torch.float32)),
            (ops.paged_sdpa_lse, (step.q, *cache, *batch, SCALE, 3, False, torch.float32)),
            (ops.paged_kv_mass, (step.q, lse, *cache, step.mass[0].clone(), *batch, SCALE, 3, False)),
            (ops.kv_pages_evict, (*step.pool, keep, step.table, step.lengths, step.mass)),
            (ops.kv_pages_evict, (*step.pool, keep, step.table, step.lengths, None))]:
        torch.library.opcheck(op.default, args, test_utils=utils)


def test_nothing_in_the_batch(gpu):
    _, _, _, cache, _, _ = ref.batch(1, [40], [1], HQ, HKV, D, PAGE)
    dev = tuple(t.to(gpu) for t in cache)
    bounds = torch.full((cache[0].shape[0], HKV, 2, D), 7.0, dtype=BF, device=gpu)
    for b, t in ((0, 0), (3, 0), (0, 5), (3, 5)):
        table = torch.zeros((b, 2), dtype=torch.int32, device=gpu)
        starts, lengths = _ints([0] * (b + 1), gpu), _ints([20] * b, gpu)
        at, q = (table, starts, lengths), torch.randn((t, HQ, D), device=gpu).to(BF)
        kw = {"scale": 0.1, "max_new": 1}
        sparkq.paged_key_bounds(dev, bounds, *at, max_new=1)
        scores, seen = sparkq.paged_page_scores(q, bounds, *at, page_size=PAGE, **kw)
        assert scores.shape == (t, HKV, 2) and seen.shape == (t,)
        pages = sparkq.select_top(scores, 2, lengths=seen)
        assert pages.shape == (t, HKV, 2)
        out = torch.full(q.shape, 7.0, dtype=BF, device=gpu)
        sparkq.paged_sparse_sdpa(q, dev, pages, *at, out=out, **kw)
        _, lse = sparkq.paged_quantized_sdpa(q, dev, *at, return_lse=True, **kw)
        mass = torch.full((b, HKV, 2 * PAGE), 7.0, device=gpu)
        sparkq.paged_kv_mass(q, lse, dev, mass, *at, **kw)
        assert (out == 7.0).all() and (mass == 7.0).all()
        keep = torch.zeros((b, HKV, 30), dtype=torch.int32, device=gpu)
        got = sparkq.kv_pages_evict(dev, keep, table, lengths, mass=mass)
        assert got[2].item() == 0 and got[1].tolist() == [20] * b
    assert (bounds == 7.0).all()
    for a, c in zip(dev, cache):
        assert torch.equal(a.cpu(), c)


def test_calls_that_are_refused(gpu):
    lengths, news = [40, 9], [1, 1]
    q, _, _, cache, table, starts = ref.batch(8, lengths, news, HQ, HKV, D, PAGE)
    q = q.to(BF).to(gpu)
    dev = tuple(t.to(gpu) for t in cache)
    at = _ints(table, gpu), _ints(starts, gpu), _ints(lengths, gpu)
    pages, m = cache[0].shape[0], len(table[0])
    bounds = torch.zeros((pages, HKV, 2, D), dtype=BF, device=gpu)
    mass = torch.zeros((2, HKV, m * PAGE), device=gpu)
    lse = torch.zeros((2, HQ), device=gpu)
    sel = torch.zeros((2, HKV, 2), dtype=torch.int32, device=gpu)
    kw = {"scale": 0.1, "max_new": 1}
    tables = at[0][:1].expand(2, -1), *at[1:]
    for call in (lambda t: sparkq.paged_key_bounds(dev, bounds, *t, max_new=1),
                 lambda t: sparkq.paged_page_scores(q, bounds, *t, page_size=PAGE, **kw),
                 lambda t: sparkq.paged_sparse_sdpa(q, dev, sel, *t, **kw),
                 lambda t: sparkq.paged_kv_mass(q, lse, dev, mass, *t, **kw),
                 lambda t: sparkq.kv_pages_evict(dev, sel, t[0], t[2])):
        with pytest.raises(ValueError, match="overlap"):
            call(tables)
        with pytest.raises(ValueError, match="device"):
            call((at[0].cpu(), *at[1:]))
    apart = torch.zeros((pages, 2, HKV, 2, D), dtype=BF, device=gpu)
    sparkq.paged_key_bounds(dev, apart[:, 1], *at, max_new=1)
    wide = torch.zeros((pages, HKV, 2, D + 1), dtype=BF, device=gpu)[..., :D]
    with pytest.raises(ValueError, match="contiguous"):
        sparkq.paged_key_bounds(dev, wide, *at, max_new=1)
    odd = torch.zeros(pages * HKV * 2 * D + 4, dtype=BF, device=gpu)[4:].view(bounds.shape)
    with pytest.raises(ValueError, match="16-byte"):
        sparkq.paged_page_scores(q, odd, *at, page_size=PAGE, **kw)
    with pytest.raises(ValueError, match="overlap"):
        sparkq.paged_page_scores(q, bounds[:, :1].expand(-1, HKV, -1, -1), *at, page_size=PAGE, **kw)
    with pytest.raises(ValueError, match="out must be"):
        sparkq.paged_sparse_sdpa(q, dev, sel, *at, out=q[:1], **kw)
    with pytest.raises(ValueError, match="overlap"):
        sparkq.paged_kv_mass(q, lse, dev, mass[:1].expand(2, -1, -1), *at, **kw)
    with pytest.raises(ValueError, match="aligned"):
        sparkq.paged_kv_mass(q, lse, dev, torch.zeros((2, HKV, m * PAGE + 1), device=gpu)[..., :-1], *at, **kw)
    many = torch.zeros((2, 129 * HKV, D), dtype=BF, device=gpu)
    with pytest.raises(ValueError, match="at most 128 query heads"):
        sparkq.paged_kv_mass(many, torch.zeros((2, 129 * HKV), device=gpu), dev, mass, *at, **kw)
    with pytest.raises(ValueError, match="overlap"):
        sparkq.kv_pages_evict(dev, sel, at[0], at[2], mass=mass[:1].expand(2, -1, -1))
    with pytest.raises(ValueError, match="too large"):
        sparkq.select_top(torch.zeros((1, 1, 1), device=gpu).expand(1 << 22, 1, 1), 1)


def test_scores_that_are_nan_are_taken_last(gpu):
    x = torch.tensor([[[math.nan, -math.inf, 1.0, math.nan, -5.0]]], device=gpu)
    assert sparkq.select_top(x, 3).tolist() == [[[0, 2, 4]]]
    assert sparkq.select_top(x, 2).tolist() == [[[2, 4]]]
    assert sparkq.select_top(x, 4, first=0, last=2).tolist() == [[[0, 2, 3, 4]]]


def test_a_wide_table_of_short_rows(gpu):
    """Work is dealt by the lengths on the device, not by what the table has room for."""
    rng, gen = random.Random(4), torch.Generator().manual_seed(4)
    lengths, news = [90, 3, 500], [30, 1, 0]
    q, _, _, cache, _, starts = ref.batch(17, lengths, news, HQ, HKV, D, PAGE)
    table = ref.tables(rng, lengths, PAGE, cache[0].shape[0], 8192)
    q, dev = q.to(BF), tuple(t.to(gpu) for t in cache)
    at = _ints(table, gpu), _ints(starts, gpu), _ints(lengths, gpu)
    _, lse = sparkq.paged_quantized_sdpa(q.to(gpu), dev, *at, scale=SCALE, max_new=30, return_lse=True)
    before = torch.rand((3, HKV, 8192 * PAGE), generator=gen)
    got = before.to(gpu)
    sparkq.paged_kv_mass(q.to(gpu), lse, dev, got, *at, scale=SCALE, max_new=30)
    short = [r[:40] for r in table]
    check_mass(got[..., :40 * PAGE], q, lse.cpu(), cache, before[..., :40 * PAGE], short, starts, lengths,
               SCALE)
    assert torch.equal(got[..., 40 * PAGE:].cpu(), before[..., 40 * PAGE:])
