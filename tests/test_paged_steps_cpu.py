"""Steps of kvmix_amd.paged that are over are refused: their plans name pages that hold something else by now.  No GPU."""
import pytest
import torch

from kvmix_amd import paged
from test_paged_sharing_cpu import Pools


@pytest.fixture
def pools(monkeypatch):
    p = Pools(monkeypatch, 32, row_pages=64)
    p.calls = []
    monkeypatch.setattr(paged.ops, "paged_append", lambda k, v, rows, plan: p.calls.append(plan))
    monkeypatch.setattr(paged.ops, "paged_attention", lambda q, rows, packed, plan, kb, vb, scale: p.calls.append(plan))
    return p


def use(cache, step):
    x = torch.zeros(1)
    cache.append(0, step, x, x)
    cache.attend(0, step, x)


def over(cache, step):
    with pytest.raises(RuntimeError, match="step is over"):
        cache.append(0, step, torch.zeros(1), torch.zeros(1))
    with pytest.raises(RuntimeError, match="step is over"):
        cache.attend(0, step, torch.zeros(1))


def test_a_step_serves_every_layer_until_the_next_one(pools):
    cache = pools.cache
    a, b = cache.new(), cache.new()
    first = cache.step({a: 40})
    other = cache.step({b: 40})
    for _ in range(3):
        use(cache, first)
        use(cache, other)
    cache.fork(a)
    use(cache, first)
    second = cache.step({a: 1})
    use(cache, second)
    use(cache, other)
    over(cache, first)
    assert pools.calls.count(first.plan) == 8


def test_pages_that_moved(pools):
    cache = pools.cache
    a, b, c = (cache.new() for _ in range(3))
    cache.step({a: 100})
    step = cache.step({b: 50, c: 10})
    assert cache.compact() == 0
    use(cache, step)          # (nothing moved)
    cache.free(a)
    use(cache, step)          # (nothing of the step's)
    assert cache.compact() > 0
    over(cache, step)
    use(cache, cache.step({b: 1}))


def test_sequences_that_ended(pools):
    cache = pools.cache
    a, b = cache.new(), cache.new()
    step = cache.step({a: 3, b: 5})
    cache.free(b)
    over(cache, step)


def test_a_step_of_another_cache(pools, monkeypatch):
    step = pools.cache.step({pools.cache.new(): 3})
    other = Pools(monkeypatch, 32)
    with pytest.raises(RuntimeError, match="another cache"):
        other.cache.attend(0, step, torch.zeros(1))


@pytest.mark.parametrize("heads", [0, -4])
def test_numbers_of_heads_that_are_none(heads):
    with pytest.raises(RuntimeError, match="heads"):
        paged.PagedKVCache([4], [4], heads, 2, 64, row_pages=4, packed_pages=4, device="cpu")
