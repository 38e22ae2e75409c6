"""PagedKVCache.step beside work that is still under way on the GPU."""

import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_step_does_not_wait_for_the_device(gpu):
    """Steps are enqueued behind products that take some tens of milliseconds, and
    have what they were given although the lists' memory is gone by then."""
    import sparkq

    cache = sparkq.PagedKVCache(1, 200, 1, 64, page_size=16, max_pages=20, batch=4, device=gpu)
    a = torch.randn((8192, 8192), device=gpu)
    b = torch.empty_like(a)
    for _ in range(6):  # (the staging memory and the kernels' first use)
        cache.step([1, 2, 0, 3])
    torch.mm(a, a, out=b)
    torch.cuda.synchronize()
    done = torch.cuda.Event()
    for _ in range(6):
        torch.mm(a, a, out=b)
    done.record()
    starts = [cache.step([i, 1, 5 - i, 0]) for i in range(5)]
    assert not done.query()
    torch.cuda.synchronize()
    assert [s.tolist() for s in starts] == [[0, i, i + 1, 6, 6] for i in range(5)]
    assert cache.lengths.tolist() == [6 + 10, 12 + 5, 15, 18] and cache.missing.item() == 0


def test_a_step_is_not_captured(gpu):
    """Its numbers would be those of the capture in every replay."""
    import sparkq

    cache = sparkq.PagedKVCache(1, 8, 1, 64, page_size=16, max_pages=4, batch=1, device=gpu)
    cache.step([3])
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        kept = cache.lengths + 1
        with pytest.raises(RuntimeError, match="captured"):
            cache.step([1])
    graph.replay()
    torch.cuda.synchronize()
    assert kept.tolist() == [4]
    cache.step([1])
    assert cache.lengths.tolist() == [4]
