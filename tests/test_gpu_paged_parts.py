"""Contexts split into as many parts as there can be (512), in tiles that end in
groups of 16 without rows."""

import pytest
import torch

import paged_reference as ref
from test_gpu_paged_sdpa import check, run

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("gqa,d,new", [(1, 64, 20), (2, 128, 9), (1, 256, 33)])
def test_the_most_parts_of_a_tile_of_few_rows(gpu, gqa, d, new):
    n = 70000
    q, _, _, cache, table, starts = ref.batch(30, [n], [new], gqa, 1, d, 1024)
    q = q.to(torch.float16)
    out = run(gpu, q, cache, table, starts, [n], new, out_dtype=torch.float32)
    assert check(out, q, cache, table, starts, [n], d ** -0.5).all()


@pytest.mark.parametrize("d", [64, 128, 256])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("size,scale", [(2.0 ** -100, 2.0 ** 98), (2.0 ** -122, 2.0 ** 119),
                                        (2.0 ** -126, 0.1), (2.0 ** -130, 2.0 ** 126)])
def test_queries_down_to_the_smallest(gpu, d, new, size, scale):
    """bf16 queries near the end of its range and past it (2^-130: of 4 bits), with
    a scale that makes ordinary scores of them, and one that makes none."""
    import sparkq

    lengths = [300, 90]
    q, _, _, cache, table, starts = ref.batch(31, lengths, [new, new], 4, 1, d, 32)
    q = (q * size).to(torch.bfloat16)
    ints = lambda v: torch.tensor(v, dtype=torch.int32, device=gpu)  # noqa: E731
    out = sparkq.paged_quantized_sdpa(q.to(gpu), tuple(t.to(gpu) for t in cache), ints(table),
                                      ints(starts), ints(lengths), scale=scale, max_new=new)
    assert check(out, q, cache, table, starts, lengths, scale).all()
