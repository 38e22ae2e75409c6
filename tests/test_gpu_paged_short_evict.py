"""A step that the pool has too few pages for, and an eviction in its place."""

import pytest
import torch

import sparkq

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
HQ, HKV, D, PAGE = 8, 2, 64, 16


def test_eviction_in_the_place_of_a_short_step(gpu):
    """The step is refused to evict, taken back, and fits after the eviction: nothing of the
    rows is lost in between."""
    gen = torch.Generator().manual_seed(1)
    make = lambda n, h: torch.randn((n, h, D), generator=gen).to(BF).to(gpu)  # noqa: E731
    cache = sparkq.PagedKVCache(2, 10, HKV, D, page_size=PAGE, max_pages=8, batch=2, device=gpu, mass=True)

    def step(news, parents=None):
        cache.step(news, parents)
        if cache.missing.item():
            return False
        for layer in range(2):
            cache.append(layer, make(sum(news), HKV), make(sum(news), HKV))
            cache.attend(layer, make(sum(news), HQ), scale=D ** -0.5)
        return True

    assert step([75, 79])  # all ten pages
    state = [t.clone() for t in (*cache.cache, cache.mass, cache.page_table, cache.lengths)]
    assert not step([4, 4], [0, 1]) and cache.missing.item() == 1
    with pytest.raises(ValueError, match="undo"):
        cache.evict(48)
    cache.undo()
    for a, b in zip((*cache.cache, cache.mass, cache.page_table, cache.lengths), state):
        assert torch.equal(a, b)
    assert cache.evict(48, first=2, last=8).item() == 0
    assert cache.lengths.tolist() == [48, 48] and (cache.page_table >= 0).sum().item() == 6
    assert step([4, 4], [0, 1]) and cache.lengths.tolist() == [52, 52]
