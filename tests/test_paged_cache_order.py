"""CPU tests of PagedKVCache: what it refuses between a step and the step's first append,
and that a call that fails leaves it as it was."""

import pytest
import torch

import sparkq
from sparkq import paged


@pytest.fixture
def cache(monkeypatch):
    """A cache of two rows of 20 and 9 tokens, on the CPU with stand-ins for the calls that
    a GPU takes; `calls` lists these."""
    calls = []

    def fork(cache, table, lengths, parents=None, new_tokens=None):
        calls.append("fork")
        rows = new_tokens.shape[0]
        before = lengths if parents is None else lengths[parents.clamp(min=0).long()]
        return table.new_zeros((rows, table.shape[1])), before + new_tokens, table.new_zeros(1)

    def evict(cache, keep, table, lengths, mass=None):
        calls.append("evict")
        return table, lengths.clamp(max=keep.shape[-1]), table.new_zeros(1)

    monkeypatch.setattr(paged, "kv_pages_fork", fork)
    monkeypatch.setattr(paged, "kv_pages_evict", evict)
    monkeypatch.setattr(paged, "select_top", lambda x, count, **kw: x.new_zeros((*x.shape[:-1], count)).int())
    monkeypatch.setattr(paged, "paged_kv_append", lambda *a: calls.append("append"))
    monkeypatch.setattr(paged, "paged_quantized_sdpa", lambda *a, **kw: (calls.append("attend"), None))
    monkeypatch.setattr(paged, "paged_kv_mass", lambda *a, **kw: None)
    c = sparkq.PagedKVCache(1, 8, 1, 64, page_size=16, max_pages=4, batch=2, device="cpu", mass=True)
    c.step([20, 9])
    c.append(0, None, None)
    c.attend(0, None, scale=1.0)
    calls.clear()
    c.calls = calls
    return c


def test_eviction_is_refused_while_a_step_has_not_appended(cache):
    """Its tokens have no place yet where it was short of pages, and no weight."""
    cache.step([1, 1])
    table, lengths = cache.page_table, cache.lengths
    with pytest.raises(ValueError, match="append.*undo"):
        cache.evict(5)
    assert cache.calls == ["fork"] and cache.page_table is table and cache.lengths is lengths
    cache.missing = torch.ones(1, dtype=torch.int32)  # (what the device says of a short step)
    cache.undo()
    assert cache.lengths.tolist() == [20, 9]
    cache.evict(8)
    assert cache.calls == ["fork", "evict"] and cache.lengths.tolist() == [8, 8]


def test_eviction_after_what_has_no_new_tokens(cache):
    cache.step([1, 1])
    cache.append(0, None, None)
    cache.evict(8)  # the step's tokens are in the cache
    cache.step([0], [1])  # rows are dropped, nothing is to be appended
    cache.evict(7)
    cache.step([0, 0], [0, 0])
    cache.evict(6)
    assert cache.calls == ["fork", "append", "evict", "fork", "evict", "fork", "evict"]


def test_a_step_that_fails_leaves_the_cache_as_it_was(cache, monkeypatch):
    """Weights of rows that continue others are a tensor of their own, which there may be
    no memory for."""
    def full(self, parents):
        raise torch.OutOfMemoryError("no memory")

    names = ("page_table", "lengths", "missing", "mass", "starts", "max_new", "_last", "_counts")
    before = [getattr(cache, n) for n in names]
    with monkeypatch.context() as m:
        m.setattr(sparkq.PagedKVCache, "_mass_of", full)
        with pytest.raises(torch.OutOfMemoryError):
            cache.step([3, 4, 5], [0, 0, 1])
    assert all(getattr(cache, n) is b for n, b in zip(names, before)) and not cache.calls
    cache.step([3, 4, 5], [0, 0, 1])
    assert cache.lengths.tolist() == [23, 24, 14] and cache.mass.shape[1] == 3
