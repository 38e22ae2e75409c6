"""Drafted tokens of a cache that gathers weights: what is taken back weighs nothing where
the weights are added once it is known which tokens stay."""

import pytest
import torch

import sparkq

pytestmark = pytest.mark.gpu

BF = torch.bfloat16
HQ, HKV, D, PAGE, SCALE = 8, 2, 64, 16, 0.125


@pytest.mark.parametrize("drafted,kept", [([4, 4, 4], [4, 1, 2]), ([20, 1, 9], [3, 1, 9])])
def test_weights_of_accepted_tokens_alone(gpu, drafted, kept):
    gen = torch.Generator().manual_seed(sum(kept))
    make = lambda n, h: torch.randn((n, h, D), generator=gen).to(BF).to(gpu)  # noqa: E731
    prompt = [50, 7, 33]
    first = [sum(drafted[:b]) for b in range(3)]
    stay = [first[b] + i for b in range(3) for i in range(kept[b])]
    data = {(n, layer): (make(n, HKV), make(n, HKV), make(n, HQ)) for n in (sum(prompt), sum(drafted))
            for layer in range(2)}
    caches = [sparkq.PagedKVCache(2, 30, HKV, D, page_size=PAGE, max_pages=8, batch=3, device=gpu, mass=True)
              for _ in range(2)]
    for c in caches:
        c.step(prompt)
        for layer in range(2):
            k, v, q = data[sum(prompt), layer]
            c.append(layer, k, v)
            c.attend(layer, q, scale=SCALE)
    drafts, plain = caches
    drafts.step(drafted)
    kept_rows = []
    for layer in range(2):
        k, v, q = data[sum(drafted), layer]
        drafts.append(layer, k, v)
        _, lse = sparkq.paged_quantized_sdpa(q, drafts.layer(layer), drafts.page_table, drafts.starts,
                                             drafts.lengths, scale=SCALE, max_new=drafts.max_new, return_lse=True)
        kept_rows.append((q[stay], lse[stay]))
    drafts.lengths.sub_(torch.tensor([a - b for a, b in zip(drafted, kept)], dtype=torch.int32, device=gpu))
    starts = torch.tensor([0, kept[0], kept[0] + kept[1], sum(kept)], dtype=torch.int32, device=gpu)
    for layer, (q, lse) in enumerate(kept_rows):
        sparkq.paged_kv_mass(q, lse, drafts.layer(layer), drafts.mass[layer], drafts.page_table, starts,
                             drafts.lengths, scale=SCALE, max_new=max(kept))
    plain.step(kept)
    for layer in range(2):
        k, v, q = (t[stay] for t in data[sum(drafted), layer])
        plain.append(layer, k, v)
        plain.attend(layer, q, scale=SCALE)
    assert drafts.lengths.tolist() == plain.lengths.tolist() == [a + b for a, b in zip(prompt, kept)]
    for b, n in enumerate(plain.lengths.tolist()):
        # a weight is exp(score - lse), of scores that are off by (D + 8) 2^-24 of scale * sum
        # |q||k| < 16 (2^-14) and logarithms by as much, on either side by another kernel
        assert torch.allclose(drafts.mass[:, b, :, :n], plain.mass[:, b, :, :n], rtol=2.0 ** -12, atol=2.0 ** -24)
        assert abs(plain.mass[:, b, :, :n].sum().item() / (2 * HQ) - n) < 1e-3 * n
