"""The ways the paged cache's operators are called: captured and replayed, two
graphs at once, on a side stream, as custom ops, with nothing in the batch,
with splits of many sequences, and the calls they refuse on the device."""

import math

import pytest
import torch

import paged_reference as ref
from test_gpu_paged_sdpa import check, run

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
HQ, HKV, D, PAGE = 8, 2, 128, 32


def _ints(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


class Step:
    """A whole step of five rows (one a second continuation of sequence 0) in
    two layers, on tensors that stay where they are."""

    def __init__(self, gpu, seed, news):
        self.news = news
        self.starts = _ints([sum(news[:i]) for i in range(6)], gpu)
        self.fresh = _ints(news, gpu)
        self.parents = _ints([0, 1, 0, 3, 2], gpu)
        self.gen = torch.Generator().manual_seed(seed)
        self.pool = [t.to(gpu) for t in ref.pool(self.gen, 170, HKV, PAGE, D, layers=2)]
        self.table = torch.full((4, 40), -1, dtype=torch.int32, device=gpu)
        self.lengths = torch.zeros(4, dtype=torch.int32, device=gpu)
        t = sum(news)
        self.qkv = torch.zeros((t, HQ + 2 * HKV, D), dtype=BF, device=gpu)
        self.pos = torch.zeros(t, dtype=torch.int32, device=gpu)
        self.w = torch.ones(D, dtype=BF, device=gpu)
        self.fill(0)

    def fill(self, k):
        """Other tokens, pages and lengths in the same tensors."""
        lengths = [700 + 64 * k, 33 + k, 5 + k, 1000 + k]
        ids = torch.randperm(160, generator=self.gen).tolist()
        rows = [[ids.pop() for _ in range(-(-n // PAGE))] for n in lengths]
        self.table.copy_(torch.tensor([r + [-1] * (40 - len(r)) for r in rows], dtype=torch.int32))
        self.lengths.copy_(torch.tensor(lengths, dtype=torch.int32))
        self.qkv.copy_(torch.randn(self.qkv.shape, generator=self.gen))
        self.pos.copy_(torch.randint(0, 4000, self.pos.shape, generator=self.gen, dtype=torch.int32))
        for t, c in zip(self.pool, ref.pool(self.gen, 170, HKV, PAGE, D, layers=2)):
            t.copy_(c)

    def __call__(self):
        import sparkq

        out = []
        table, lengths, missing = sparkq.kv_pages_fork(self.pool, self.table, self.lengths,
                                                       self.parents, self.fresh)
        q, k = sparkq.qk_norm_rope(self.qkv[:, :HQ], self.qkv[:, HQ:HQ + HKV], self.w, self.w,
                                   self.pos, dims=D, eps=1e-6)
        for layer in range(2):
            cache = tuple(t[layer] for t in self.pool)
            sparkq.paged_kv_append(k, self.qkv[:, HQ + HKV:], cache, table, self.starts, lengths)
            out.append(sparkq.paged_quantized_sdpa(q, cache, table, self.starts, lengths,
                                                   scale=D ** -0.5, max_new=max(self.news)))
        table, used = sparkq.kv_pages_compact(self.pool, table, lengths)
        return [*out, table, lengths, missing, used]

    def state(self):
        return [t.clone() for t in self.pool]

    def restore(self, state):
        for t, s in zip(self.pool, state):
            t.copy_(s)


def _equal(got, want):
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("news", [[1, 1, 1, 1, 1], [40, 1, 3, 0, 7]])
def test_a_captured_step(gpu, news):
    """Every replay, on batches that change in between, with eager steps and
    synchronisation between them, is the eager step bit for bit, the pool too."""
    step = Step(gpu, 1, news)
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
        _equal(step.pool, after)
        assert want[4].item() == 0


def test_two_graphs_and_a_side_stream(gpu):
    """Graphs of two batches replay on two streams at once, and a step runs on a
    stream of its own: their scratch is their own."""
    steps = [Step(gpu, 2, [1] * 5), Step(gpu, 3, [20, 1, 1, 30, 2])]
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
            _equal(step.pool, after)
    for step, before, want in zip(steps, befores, wants):
        step.restore(before)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            got = step()
        side.synchronize()
        _equal(got, want)


def test_custom_ops_are_the_operators(gpu):
    import sparkq

    ops = torch.ops.sparkq
    utils = ("test_schema", "test_autograd_registration", "test_faketensor")
    step = Step(gpu, 4, [1, 9, 2, 1, 1])
    before = step.state()
    want = [t.clone() for t in step()]
    step.restore(before)
    table, lengths, missing = ops.kv_pages_fork(*step.pool, step.table, step.lengths, step.parents,
                                                step.fresh)
    q, k = ops.qk_norm_rope(step.qkv[:, :HQ], step.qkv[:, HQ:HQ + HKV], step.w, step.w, step.pos, D,
                            1e-6, 10000.0, 1.0, False)
    got = []
    for layer in range(2):
        cache = [t[layer] for t in step.pool]
        ops.paged_kv_append(k, step.qkv[:, HQ + HKV:], *cache, table, step.starts, lengths)
        got.append(ops.paged_sdpa(q, *cache, table, step.starts, lengths, D ** -0.5, 9, True, None))
    args = (q, *cache, table, step.starts, lengths, D ** -0.5, 9, False, torch.float32)
    torch.library.opcheck(ops.paged_sdpa.default, args, test_utils=utils)
    torch.library.opcheck(ops.qk_norm_rope.default,
                          (step.qkv[:, :HQ], step.qkv[:, HQ:HQ + HKV], step.w, step.w, step.pos, D,
                           1e-6, 10000.0, 1.0, True), test_utils=utils)
    torch.library.opcheck(ops.paged_kv_append.default,
                          (k, step.qkv[:, HQ + HKV:], *cache, table, step.starts, lengths),
                          test_utils=utils)
    both = ops.kv_pages_compact(*step.pool, table, lengths)
    _equal([*got, both[0], lengths, missing, both[1]], want)
    torch.library.opcheck(ops.kv_pages_compact.default, (*step.pool, both[0], lengths),
                          test_utils=utils)
    torch.library.opcheck(ops.kv_pages_fork.default, (*step.pool, both[0], lengths, None, step.fresh),
                          test_utils=utils)


def test_nothing_in_the_batch(gpu):
    import sparkq

    _, _, _, cache, _, _ = ref.batch(1, [40], [1], HQ, HKV, D, PAGE)
    dev = tuple(t.to(gpu) for t in cache)
    for b, t in ((0, 0), (3, 0), (0, 5)):
        table = torch.zeros((b, 2), dtype=torch.int32, device=gpu)
        starts, lengths = _ints([0] * (b + 1), gpu), _ints([40] * b, gpu)
        q, kv = (torch.randn((t, h, D), device=gpu).to(BF) for h in (HQ, HKV))
        sparkq.paged_kv_append(kv, kv, dev, table, starts, lengths)
        out = torch.full(q.shape, 7.0, dtype=BF, device=gpu)
        sparkq.paged_quantized_sdpa(q, dev, table, starts, lengths, scale=0.1, max_new=1, out=out)
        assert (out == 7.0).all()
        w = torch.ones(D, dtype=BF, device=gpu)
        qo, ko = sparkq.qk_norm_rope(q, kv, w, w, torch.zeros(t, dtype=torch.int64, device=gpu),
                                     dims=D, eps=1e-6)
        assert qo.shape == q.shape and ko.shape == kv.shape
        assert sparkq.kv_pages_fork(dev, table, lengths)[2].item() == 0
        assert sparkq.kv_pages_compact(dev, table, lengths)[1].item() == (0 if b == 0 else 1)
    for a, c in zip(dev, cache):
        assert torch.equal(a.cpu(), c)


def test_a_batch_that_starts_empty_and_ends_empty(gpu):
    import sparkq

    cache = sparkq.PagedKVCache(2, 9, HKV, D, page_size=16, max_pages=3, device=gpu)
    assert cache.step([]).tolist() == [0]
    cache.step([20, 0, 48], [-1, -1, -1])
    assert cache.lengths.tolist() == [20, 0, 48] and cache.missing.item() == 0
    assert cache.page_table.tolist() == [[0, 1, -1], [-1] * 3, [2, 3, 4]]
    x = torch.randn((68, HKV, D), device=gpu).to(BF)
    cache.append(1, x, x)
    out = cache.attend(1, x, scale=0.1)
    assert out.isfinite().all() and out.shape == x.shape
    cache.step([], [])
    assert cache.compact().item() == 0
    cache.step([1], [-1])
    assert cache.page_table.tolist() == [[0, -1, -1]] and cache.lengths.tolist() == [1]


@pytest.mark.parametrize("hkv,gqa,d", [(1, 4, 64), (1, 16, 128), (2, 1, 256)])
@pytest.mark.parametrize("new", [1, 24])
def test_long_contexts_among_many_sequences(gpu, hkv, gqa, d, new):
    """Splits beyond the first 64 sequences, with tables wider than the contexts."""
    lengths = [5000 if i in (3, 64, 77) else 30 + i for i in range(80)]
    news = [min(new, n) for n in lengths]
    q, _, _, cache, table, starts = ref.batch(5, lengths, news, hkv * gqa, hkv, d, 64, width=90)
    q = q.to(torch.float16)
    out = run(gpu, q, cache, table, starts, lengths, new)
    assert check(out, q, cache, table, starts, lengths, d ** -0.5).all()


@pytest.mark.parametrize("new", [1, 20])
@pytest.mark.parametrize("scale", [0.0, -0.2, 1, 3.0])
def test_scales(gpu, new, scale):
    import sparkq

    lengths, news = [100, 700], [new, new]
    q, _, _, cache, table, starts = ref.batch(6, lengths, news, HQ, HKV, D, PAGE)
    q = q.to(BF)
    dev = tuple(t.to(gpu) for t in cache)
    out = sparkq.paged_quantized_sdpa(q.to(gpu), dev, _ints(table, gpu), _ints(starts, gpu),
                                      _ints(lengths, gpu), scale=scale, max_new=10 ** 9)
    check(out, q, cache, table, starts, lengths, scale)


@pytest.mark.parametrize("d", [128, 256])
@pytest.mark.parametrize("new", [1, 64])
def test_descending_starts_stay_in_bounds(gpu, new, d):
    """Sequences whose rows overlap are more work than the call's scratch is
    for: the others have their results, and what lies behind is left alone."""
    lengths = [3000] * 12 + [90]
    q, _, _, cache, table, _ = ref.batch(7, lengths, [0] * 12 + [new], HQ, HKV, d, PAGE, extra_rows=70)
    t = q.shape[0]
    q = q.to(BF)
    starts = [0 if i % 2 == 0 else new for i in range(13)] + [new]
    out = torch.full((t + 64, HQ, d), 7.0, dtype=BF, device=gpu)
    run(gpu, q, cache, table, starts, lengths, new, out=out[:t])
    assert (out[new:] == 7.0).all()
    assert out[:new].isfinite().all()


@pytest.mark.parametrize("dtype", [torch.float16, BF, torch.float32])
@pytest.mark.parametrize("d", [64, 128, 256])
def test_append_quantizes_like_kv_quantize_s8(gpu, dtype, d):
    """Rows of every size, and with infinities and NaN: the codes and scales of
    the contiguous cache's quantizer, bit for bit."""
    import sparkq

    gen = torch.Generator().manual_seed(d)
    x = torch.randn((60, 2, d), generator=gen)
    top = 38 if dtype != torch.float16 else 4
    x *= 10.0 ** torch.linspace(-8 if dtype == torch.float16 else -45, top, 60)[:, None, None]
    x = x.to(dtype)
    x[5, 0, 7], x[6, 1, 0], x[7, 0, 3] = math.inf, -math.inf, math.nan
    x[8], x[9, 0] = 0, math.nan
    x = x.to(gpu)
    cache = tuple(torch.zeros((4, 2, 16, *tail), dtype=t, device=gpu)
                  for t, tail in ((torch.int8, (d,)), (torch.float16, ())) * 2)
    sparkq.paged_kv_append(x, x.flip(0), cache, _ints([[2, 0, 3, 1]], gpu), _ints([0, 60], gpu),
                           _ints([60], gpu))
    for y, codes, scales in ((x, *cache[:2]), (x.flip(0), *cache[2:])):
        want, ws = sparkq.kv_quantize_s8(y.transpose(0, 1).contiguous()[None])
        got = codes[[2, 0, 3, 1]].transpose(0, 1).reshape(2, 64, d)[:, :60]
        gs = scales[[2, 0, 3, 1]].transpose(0, 1).reshape(2, 64)[:, :60]
        assert torch.equal(got, want.view(torch.int8).view(2, 60, d))
        assert torch.equal(gs.view(torch.int16), ws.half().view(2, 60).view(torch.int16))


def test_calls_that_are_refused(gpu):
    import sparkq

    lengths, news = [40, 9], [1, 1]
    q, k, _, cache, table, starts = ref.batch(8, lengths, news, HQ, HKV, D, PAGE)
    q, k = q.to(BF).to(gpu), k.to(BF).to(gpu)
    dev = tuple(t.to(gpu) for t in cache)
    at = _ints(table, gpu), _ints(starts, gpu), _ints(lengths, gpu)
    kw = {"scale": 0.1, "max_new": 1}
    apart = torch.zeros((dev[0].shape[0], 2, *dev[0].shape[1:]), dtype=torch.int8, device=gpu)[:, 0]
    with pytest.raises(ValueError, match="same strides"):
        sparkq.paged_quantized_sdpa(q, (*dev[:2], apart, dev[3]), *at, **kw)
    with pytest.raises(ValueError, match="overlap"):
        sparkq.paged_quantized_sdpa(q, dev, at[0][:1].expand(2, -1), *at[1:], **kw)
    with pytest.raises(ValueError, match="one device|cache's device"):
        sparkq.paged_quantized_sdpa(q, dev, at[0].cpu(), *at[1:], **kw)
    with pytest.raises(ValueError, match="device"):
        sparkq.paged_kv_append(k.cpu(), k, dev, *at)
    with pytest.raises(ValueError, match="one device"):
        sparkq.paged_kv_append(k, k, (*dev[:3], dev[3].cpu()), *at)
    with pytest.raises(ValueError, match="out must be"):
        sparkq.paged_quantized_sdpa(q, dev, *at, out=q[:1], **kw)
    wide = (torch.zeros((4, 2, 16, 96), dtype=torch.int8, device=gpu),
            torch.zeros((4, 2, 16), dtype=torch.float16, device=gpu)) * 2
    with pytest.raises(ValueError, match="head dim"):
        sparkq.paged_quantized_sdpa(torch.zeros((2, 4, 96), dtype=BF, device=gpu), wide, *at, **kw)


def test_a_step_that_runs_short_is_taken_back(gpu):
    import sparkq

    cache = sparkq.PagedKVCache(1, 6, 1, 64, page_size=16, max_pages=4, batch=2, device=gpu)
    with pytest.raises(ValueError, match="no step"):
        cache.undo()
    cache.step([30, 16])
    table, lengths = cache.page_table.clone(), cache.lengths.clone()
    assert cache.missing.item() == 0
    cache.step([20, 40], [0, 0])  # row 1 takes a copy and three more: one is missing
    assert cache.missing.item() > 0
    cache.undo()
    assert torch.equal(cache.page_table, table) and torch.equal(cache.lengths, lengths)
    assert cache.starts.tolist() == [0, 30, 46] and cache.max_new == 30
    cache.step([20], [0])
    assert cache.missing.item() == 0 and cache.lengths.tolist() == [50]


# --- what head dims and halves of blocks see differently --------------------------

@pytest.mark.parametrize("hkv,gqa,d", [(4, 4, 256), (2, 8, 128), (2, 16, 64)])
@pytest.mark.parametrize("page", [16, 32, 64])
@pytest.mark.parametrize("scale", [0.06, 1.0, 4.0])
def test_sharp_and_flat_weights_over_long_chunks(gpu, hkv, gqa, d, page, scale):
    """Scores of some hundred, where the running maximum moves from block to block
    and differently in the halves of a block, and the contexts are split."""
    import sparkq

    lengths, news = [900, 130, 31], [70, 130, 31]
    q, _, _, cache, table, starts = ref.batch(20, lengths, news, hkv * gqa, hkv, d, page)
    q = q.to(BF)
    out = sparkq.paged_quantized_sdpa(q.to(gpu), tuple(t.to(gpu) for t in cache), _ints(table, gpu),
                                      _ints(starts, gpu), _ints(lengths, gpu), scale=scale,
                                      max_new=130, out_dtype=torch.float32)
    assert check(out, q, cache, table, starts, lengths, scale).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 100])
def test_value_scales_in_any_order(gpu, d, new):
    """Value scales over fp16's range, growing, falling and shuffled: the largest
    so far decides the unit of a row's weights."""
    lengths, news = [300, 280, 260], [new] * 3
    q, _, _, cache, table, starts = ref.batch(21, lengths, news, 8, 2, d, 32)
    order = torch.randperm(260, generator=torch.Generator().manual_seed(1)).tolist()
    for b, n in enumerate(lengths):
        for pos in range(n):
            k = (pos, n - 1 - pos, order[min(pos, 259)])[b]
            cache[3][table[b][pos // 32], :, pos % 32] = 2.0 ** (-24 + k * 39 / n)
    q = q.to(BF)
    out = run(gpu, q, cache, table, starts, lengths, new, out_dtype=torch.float32)
    check(out, q, cache, table, starts, lengths, d ** -0.5)


@pytest.mark.parametrize("new", [1, 24, 90])
def test_hidden_values_at_head_dim_256(gpu, new):
    """NaN and infinite scales behind each sequence's end and in pages that no
    table names; a visible infinite one (p c inf: infinite, NaN where the code c
    is 0) leaves just the rows that see it without finite values."""
    lengths, news = [150, 97], [min(new, 150), min(new, 97)]
    q, _, _, cache, table, starts = ref.batch(22, lengths, news, 8, 2, 256, 32)
    _, ks, _, vs = cache
    named = {p for r, n in zip(table, lengths) for p in r[: -(-n // 32)]}
    for p in range(ks.shape[0]):
        if p not in named:
            ks[p], vs[p] = math.nan, math.inf
    for r, n in zip(table, lengths):
        if n % 32:
            ks[r[n // 32], :, n % 32:] = math.inf
            vs[r[n // 32], :, n % 32:] = math.nan
    q = q.to(torch.float16)
    check(run(gpu, q, cache, table, starts, lengths, new), q, cache, table, starts, lengths, 1 / 16)
    vs[table[0][149 // 32], 1, 149 % 32] = math.inf  # the last token, of one KV head
    out = run(gpu, q, cache, table, starts, lengths, new).cpu()
    last = starts[1] - 1
    assert not out[last, 4:].isfinite().any() and out[last, :4].isfinite().all()
    assert out[:last].isfinite().all() and out[last + 1:].isfinite().all()


@pytest.mark.parametrize("d", [64, 256])
@pytest.mark.parametrize("page", [16, 32, 128])
def test_absent_pages_inside_a_context(gpu, d, page):
    """Holes of every page size in the middle of the blocks of a chunk, and rows
    whose every token is hidden."""
    lengths, news = [700, 200], [60, 200]
    q, _, _, cache, table, starts = ref.batch(23, lengths, news, 8, 2, d, page)
    for j in range(0, len(table[0]) - 2, 3):
        table[0][j] = -1
    for j in range(0, 64 // page + 1):
        table[1][j] = 10 ** 9
    q = q.to(torch.float16)
    out = run(gpu, q, cache, table, starts, lengths, 200)
    assert check(out, q, cache, table, starts, lengths, d ** -0.5).all()
    assert (out[starts[1]:starts[1] + 64] == 0).all()


@pytest.mark.parametrize("d,hkv", [(256, 4), (128, 8), (64, 2)])
def test_more_tiles_than_the_chip_holds(gpu, d, hkv):
    """Several rounds of workgroups, the second of them dealt in reverse."""
    n = 128 * 40 // 4
    lengths, news = [n] * 3, [n, n - 5, 700]
    q, _, _, cache, table, starts = ref.batch(24, lengths, news, 4 * hkv, hkv, d, 64)
    q = q.to(BF)
    out = run(gpu, q, cache, table, starts, lengths, n)
    pick = torch.randperm(q.shape[0], generator=torch.Generator().manual_seed(2))[:60].sort().values
    assert out.isfinite().all()
    # some rows, each as a sequence of one new token of its own
    seq = torch.bucketize(pick, torch.tensor(starts), right=True) - 1
    own = [lengths[b] - news[b] + int(t) - starts[b] + 1 for b, t in zip(seq.tolist(), pick)]
    check(out[pick.to(gpu)], q[pick], cache, [table[b] for b in seq.tolist()], list(range(61)), own,
          d ** -0.5)
