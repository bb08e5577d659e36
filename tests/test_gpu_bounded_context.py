"""The bounded-context example: chunked prompt, decode steps that gather weights, evictions."""

import importlib.util
import os

import pytest
import torch

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def example():
    spec = importlib.util.spec_from_file_location("bounded_context", os.path.join(ROOT, "examples", "bounded_context.py"))
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    return m


def test_stays_within_its_budget():
    x, held = example().run(requests=3, prompt=300, new=60, budget=128, slack=16, window=64, sinks=4, chunk=100)
    torch.cuda.synchronize()
    assert torch.isfinite(x.float()).all() and x.shape == (3, 16, 128)
    assert held[0] == 129 and max(held) == 144 and held[-1] <= 144


def test_sums_follow_the_rows_that_stay():
    m = example()
    cache = m.PagedLayers(1, 2, 4, 2, 64, 200)
    g = torch.Generator(device="cuda").manual_seed(3)
    kv = torch.randn(2 * 150, 1, 2, 2, 64, generator=g, device="cuda").to(torch.bfloat16)
    cache.append(kv, torch.arange(150, device="cuda").repeat(2, 1), 150)
    q = torch.randn(2, 4, 64, generator=g, device="cuda").to(torch.bfloat16)
    from flashmap_b200 import cache_ops
    for _ in range(3):
        cache_ops.paged_decode_attention(q, *cache.views(0), cache.held, cache.table, cache.most, 0.125,
                                         weight_sums=cache.sums[0])
    total = cache.sums[0].sum(-1)
    assert torch.allclose(total, torch.full_like(total, 3 * 2.0), atol=1e-4)  # two query heads a kv head, three steps
    before = cache.sums[0].clone()
    cache.evict(100, 4, 20)
    assert cache.held.tolist() == [100, 100] and cache.most == 100
    kept = cache.sums[0][..., :100]
    assert float(cache.sums[0][..., 100:].abs().sum()) == 0.0
    # the kept sums are the largest ones, the first and the last in any case
    for r in range(2):
        for h in range(2):
            middle = before[r, h, 4:130].sort(descending=True).values[:76].sum()
            want = middle + before[r, h, :4].sum() + before[r, h, 130:150].sum()
            assert torch.allclose(kept[r, h].sum(), want, atol=1e-5)


def test_the_first_eviction_has_weights_to_go_by(monkeypatch):
    """A prompt past the budget is cut before the first new token: the weights of its own last tokens rank it."""
    m = example()
    seen = []
    plain = m.PagedLayers.evict

    def evict(cache, budget, sinks, recent):
        seen.append([s[..., : cache.most].sum(-1) for s in cache.sums])
        plain(cache, budget, sinks, recent)

    monkeypatch.setattr(m.PagedLayers, "evict", evict)
    _, held = m.run(requests=2, prompt=300, new=2, budget=128, slack=16, window=64, sinks=4, chunk=100, look=20)
    assert held == [129, 130] and len(seen) == 1
    for total in seen[0]:  # 20 tokens, 4 query heads to a kv head
        assert torch.allclose(total, torch.full_like(total, 80.0), atol=1e-3)
