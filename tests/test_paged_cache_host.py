"""PagedKVCache on the CPU, with the plain forms in the kernels' place: what a
step may not do to rows and pages."""

import random

import pytest
import torch

import paged_reference as ref
import sparkq
from sparkq import paged


def _fork(cache, page_table, lengths, parents=None, new_tokens=None):
    pages, page, width = cache[0].shape[1], cache[0].shape[3], page_table.shape[1]
    rows = page_table.shape[0]
    parents = list(range(rows)) if parents is None else parents.tolist()
    table, after, missing, pairs = ref.fork(page_table.tolist(), lengths.tolist(), parents,
                                            new_tokens.tolist(), pages, page)
    old = [t.clone() for t in cache]
    for a, b in pairs:
        for t, o in zip(cache, old):
            t[:, b] = o[:, a]
    ints = lambda v, *shape: torch.tensor(v, dtype=torch.int32).view(*shape)  # noqa: E731
    return ints(table, -1, width), ints(after, -1), ints([missing], 1)


def _append(keys, values, cache, page_table, starts, lengths):
    for t, new in zip(cache, ref.append(keys, values, cache, page_table.tolist(), starts.tolist(),
                                        lengths.tolist())):
        t.copy_(new)


@pytest.fixture
def make(monkeypatch):
    monkeypatch.setattr(paged, "kv_pages_fork", _fork)
    monkeypatch.setattr(paged, "paged_kv_append", _append)
    return lambda pages, max_pages, batch: sparkq.PagedKVCache(
        1, pages, 1, 64, page_size=16, max_pages=max_pages, batch=batch, device="cpu")


class Told:
    """What each row of a cache has been told, and whether it still holds it."""

    def __init__(self, cache):
        self.cache, self.rows = cache, [[] for _ in range(cache.page_table.shape[0])]
        self.gen = torch.Generator().manual_seed(1)

    def step(self, news, parents=None):
        self.cache.step(news, parents)
        old = self.rows
        self.rows = [list(old[p]) if 0 <= p < len(old) else []
                     for p in (range(len(old)) if parents is None else parents)]
        x = torch.randn((sum(news), 1, 64), generator=self.gen)
        self.cache.append(0, x, x)
        for i, n in enumerate(news):
            at = sum(news[:i])
            self.rows[i] += list(x[at:at + n])

    def check(self):
        codes, scales = self.cache.layer(0)[:2]
        lengths = self.cache.lengths.tolist()
        for row, n, r in zip(self.cache.page_table.tolist(), lengths, self.rows):
            assert n == len(r)
            for pos, x in enumerate(r):
                want, s = ref.quantize(x)
                assert torch.equal(codes[row[pos // 16], :, pos % 16], want), pos
                assert torch.equal(scales[row[pos // 16], :, pos % 16], s), pos


def _unchanged(cache, news, parents=None):
    """The step is short of pages, nothing but undo() follows it, and then the
    cache is what it was."""
    state = lambda: (*cache.cache, cache.page_table, cache.lengths, cache.starts)  # noqa: E731
    before = [t.clone() for t in state()]
    starts = cache.step(news, parents)
    assert cache.missing.item() > 0
    x = torch.ones((sum(news), 1, 64))
    for call in (lambda: cache.append(0, x, x), lambda: cache.attend(0, x, scale=1.0),
                 cache.compact, lambda: cache.step([0] * len(news))):
        with pytest.raises(ValueError, match="max_pages"):
            call()
    # nor do the functions under it find a page to write
    _append(x, x, cache.layer(0), cache.page_table, starts, cache.lengths)
    cache.undo()
    assert all(torch.equal(a, b) for a, b in zip(state(), before))


@pytest.mark.parametrize("held,news", [(32, [1, 1]), (30, [20, 20]), (31, [2, 0]), (0, [33, 1]),
                                       (32, [0, 1])])
def test_a_row_past_its_pages_is_short(make, held, news):
    """Two continuations of one sequence, of whose two pages of 16 no more than
    two tokens are left: tokens without a place would land on shared ones."""
    cache = make(8, 2, 1)
    told = Told(cache)
    told.step([held])
    _unchanged(cache, news, [0, 0])
    told.check()
    told.step([32 - held, 0], [0, 0])  # what there is room for
    told.check()


def test_lengths_that_the_caller_lowers_or_sets(make):
    """The step's count of tokens follows lengths that are lowered in place (a
    draft that was rejected) or set."""
    cache = make(8, 2, 2)
    cache.step([30, 10])
    cache.lengths[0] -= 5
    cache.step([7, 0])
    assert cache.lengths.tolist() == [32, 10]
    cache.lengths = torch.tensor([31, 32], dtype=torch.int32)
    _unchanged(cache, [0, 1])
    cache.step([1, 0])
    assert cache.lengths.tolist() == [32, 32]


@pytest.mark.parametrize("seed", range(20))
def test_random_steps_keep_every_token(make, seed):
    """Steps that fork, drop and extend rows up to the last slot of their pages."""
    rng = random.Random(seed)
    cache = make(60, 3, 3)
    told = Told(cache)
    for _ in range(12):
        n = rng.randint(1, 5)
        parents = [rng.randrange(-1, len(told.rows)) for _ in range(n)]
        left = [48 - (len(told.rows[p]) if p >= 0 else 0) for p in parents]
        news = [rng.choice([0, 1, m, rng.randint(0, m)]) if m else 0 for m in left]
        if rng.random() < 0.3:
            i = rng.randrange(n)
            over = [k if j != i else left[i] + rng.randint(1, 20) for j, k in enumerate(news)]
            _unchanged(cache, over, parents)
        told.step(news, parents)
        assert cache.missing.item() == 0
        told.check()


def test_undo_takes_back_only_what_it_can(make):
    """A step that had its pages may have copied them over those of a sequence
    that it dropped, and what was appended may lie in pages held before."""
    cache = make(4, 2, 2)
    told = Told(cache)
    told.step([20, 16])
    with pytest.raises(ValueError, match="no step"):  # appended to
        cache.undo()
    told.check()
    dropped = cache.page_table[1, 0].item()
    cache.step([1, 1], [0, 0])
    assert cache.missing.item() == 0 and (cache.page_table == dropped).any()
    state = [t.clone() for t in (cache.page_table, cache.lengths, cache.starts)]
    with pytest.raises(ValueError, match="was not short"):
        cache.undo()
    assert all(torch.equal(a, b) for a, b in
               zip((cache.page_table, cache.lengths, cache.starts), state))
    cache.append(0, torch.ones((2, 1, 64)), torch.ones((2, 1, 64)))
    cache.step([11, 11])  # 32 each
    cache.step([0, 0, 0], [0, 1, 1])
    cache.step([16, 0, 16], [-1, 0, -1])  # two pages are held, two free: not short
    with pytest.raises(ValueError, match="was not short"):
        cache.undo()
    cache.step([32, 32, 16], [-1, -1, -1])
    assert cache.missing.item() == 1
    cache.append(0, torch.ones((80, 1, 64)), torch.ones((80, 1, 64)))
    with pytest.raises(ValueError, match="no step"):
        cache.undo()


def test_undo_after_a_refused_append(make, monkeypatch):
    cache = make(3, 2, 2)
    cache.step([16, 16])
    table = cache.page_table.clone()
    cache.step([16, 16])
    assert cache.missing.item() == 1

    def refuse(*args):
        raise ValueError("like the cache")

    monkeypatch.setattr(paged, "paged_kv_append", refuse)
    with pytest.raises(ValueError, match="like the cache"):
        cache.append(0, torch.ones((32, 2, 64)), torch.ones((32, 2, 64)))
    cache.undo()
    assert torch.equal(cache.page_table, table) and cache.lengths.tolist() == [16, 16]
