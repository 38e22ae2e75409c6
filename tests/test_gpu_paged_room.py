"""Rows that reach the end of their row of pages: which the fork reports, and
which steps of PagedKVCache are short of pages for."""

import random

import pytest
import torch

import paged_reference as ref

pytestmark = pytest.mark.gpu

BF = torch.bfloat16


def _ints(v, gpu):
    return torch.tensor(v, dtype=torch.int32, device=gpu)


@pytest.mark.parametrize("held,news", [(32, [1, 1]), (30, [20, 20])])
def test_shared_pages_at_the_end_of_a_row(gpu, held, news):
    """A sequence of two pages of 16, continued twice by more than they have room
    for: short of pages, and what both rows hold is the first one's tokens."""
    import sparkq

    cache = sparkq.PagedKVCache(2, 8, 2, 64, page_size=16, max_pages=2, batch=1, device=gpu)
    cache.step([held])
    x = torch.randn((held, 2, 64), generator=torch.Generator().manual_seed(1)).to(BF).to(gpu)
    for layer in range(2):
        cache.append(layer, x, x)
    before = [t.clone() for t in (*cache.cache, cache.page_table, cache.lengths)]
    cache.step(news, [0, 0])
    assert cache.missing.item() > 0
    for layer in range(2):
        with pytest.raises(ValueError, match="max_pages"):
            cache.append(layer, *[torch.ones((sum(news), 2, 64), dtype=BF, device=gpu)] * 2)
    cache.undo()
    assert all(torch.equal(a, b) for a, b in
               zip((*cache.cache, cache.page_table, cache.lengths), before))
    cache.step([32 - held, 0], [0, 0])
    if held < 32:
        cache.append(0, x[:32 - held], x[:32 - held])
    codes, scales = ref.quantize(x.cpu())
    kc, ks = (t.cpu() for t in cache.layer(0)[:2])
    for row in cache.page_table.tolist():
        assert torch.equal(kc[row].transpose(0, 1).reshape(2, 32, 64)[:, :held].transpose(0, 1), codes)
        assert torch.equal(ks[row].transpose(0, 1).reshape(2, 32)[:, :held].t(), scales)


@pytest.mark.parametrize("b,pages", [(1, 8), (60, 400), (1500, 9000), (300, 17000)])
def test_the_fork_counts_rows_without_room(gpu, b, pages):
    import sparkq

    rng = random.Random(b)
    page, width = 16, 3
    lengths = [rng.randint(0, 48) for _ in range(b)]
    table = ref.tables(rng, lengths, page, pages, width)
    lengths[0] = rng.choice([48, 1000])
    parents = [rng.randrange(-1, b + 1) for _ in range(b + 5)]
    fresh = [rng.choice([0, 1, rng.randint(0, 20), -3, 2 ** 31 - 1]) for _ in range(b + 5)]
    before = [lengths[p] if 0 <= p < b else 0 for p in parents]
    want = sum(n + max(k, 0) > page * width for n, k in zip(before, fresh))
    cache = tuple(torch.zeros((1, pages, 1, page, *tail), dtype=t, device=gpu)
                  for t, tail in ((torch.int8, (64,)), (torch.float16, ())) * 2)
    at = _ints(table, gpu), _ints(lengths, gpu), _ints(parents, gpu), _ints(fresh, gpu)
    out = sparkq.kv_pages_fork(cache, *at, return_overfull=True)
    assert len(out) == 4 and out[3].dtype == torch.int32 and out[3].tolist() == [want] != [0]
    for a, c in zip(sparkq.kv_pages_fork(cache, *at), out):
        assert torch.equal(a, c)
    room = [max(0, page * width - n) for n in before]
    fits = _ints([min(max(k, 0), r) for k, r in zip(fresh, room)], gpu)
    lens = _ints([min(n, page * width) for n in lengths], gpu)
    assert sparkq.kv_pages_fork(cache, at[0], lens, at[2], fits,
                                return_overfull=True)[3].tolist() == [0]
