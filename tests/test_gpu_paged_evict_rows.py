"""Eviction in batches whose tables take a launch of their own (more than 128 rounds of 64
entries) and of more rows than the plan takes at a time (1024), with pages that rows
share, in pools whose counters fit on the chip and in ones whose counters do not."""

import random

import pytest
import torch

import paged_reference as ref
from test_gpu_paged_long import _keeps, run_evict

pytestmark = pytest.mark.gpu


def _rows(rng, rows, most, page, width, spare):
    """(lengths, table, pages): every third row continues the full pages of the one before."""
    lengths = [rng.randint(0, most) for _ in range(rows)]
    table, used = [], 0
    for i, n in enumerate(lengths):
        row = table[i - 1][:min(n, lengths[i - 1]) // page] if i % 3 == 1 else []
        while len(row) < -(-n // page):
            row, used = [*row, used], used + 1
        table.append(row)
    names = list(range(used + spare))
    rng.shuffle(names)
    return lengths, [[names[p] for p in r] + [-1] * (width - len(r)) for r in table], used + spare


@pytest.mark.parametrize("rows,most,count,width", [
    (129, 60, 20, 4),      # a launch for the tables
    (150, 100, 37, 70),    # whose rows are more than a wave's 64 entries
    (1100, 40, 17, 3),     # and of which the plan takes 1024 at a time
    (2100, 33, 1, 3)])
@pytest.mark.parametrize("short", [False, True])
def test_evict_of_many_rows(gpu, rows, most, count, width, short):
    rng, gen = random.Random(rows), torch.Generator().manual_seed(rows)
    page, spare = 16, 3 if short else 2 * rows
    lengths, table, pages = _rows(rng, rows, most, page, width, spare)
    pool = ref.pool(gen, pages, 1, page, 64, layers=1)
    mass = torch.rand((1, rows, 1, width * page), generator=gen)
    want = run_evict(gpu, pool, _keeps(rng, lengths, 1, 1, count), table, lengths, mass)
    assert (want[2] > 0) == short
    if not short:  # pages were replaced in rows of every round
        changed = [i for i, n in enumerate(want[1])
                   if any(a != b for a, b in zip(want[0][i], table[i][: -(-n // page)]))]
        assert min(changed) < 64 and max(changed) > rows - 64


@pytest.mark.parametrize("short", [False, True])
def test_evict_of_many_rows_in_a_large_pool(gpu, short):
    """More than 16384 pages: holders are counted in the workspace."""
    rng, gen = random.Random(9), torch.Generator().manual_seed(9)
    page, rows, width = 16, 2400, 20
    lengths, table, pages = _rows(rng, rows, 300, page, width, 8 if short else 6000)
    assert pages > 16384
    pool = ref.pool(gen, pages, 1, page, 64, layers=1)
    want = run_evict(gpu, pool, _keeps(rng, lengths, 1, 1, 10), table, lengths, None)
    assert (want[2] > 0) == short
