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
