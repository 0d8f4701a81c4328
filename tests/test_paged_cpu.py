"""The bookkeeping of kvmix_amd.paged that needs no GPU: numbers of pages."""
import random

import pytest

from kvmix_amd.paged import PagedKVCache, _Pages


def test_pages_are_counted_shared_and_compacted():
    rng = random.Random(1)
    pages, held = _Pages(50), []
    for _ in range(2000):
        if held and (rng.random() < 0.5 or not pages.free):
            pages.drop(held.pop(rng.randrange(len(held))))
        elif held and rng.random() < 0.3:
            p = rng.choice(held)
            pages.share(p)
            held.append(p)
        else:
            held.append(pages.take())
        assert [pages.users[p] for p in range(50)] == [held.count(p) for p in range(50)]
        assert sorted(pages.free) == [p for p in range(50) if not pages.users[p]]
        if rng.random() < 0.05:
            moves = pages.compacted()
            assert not set(moves) & set(moves.values())
            held = [moves.get(p, p) for p in held]
            used = len(set(held))
            assert all(pages.users[p] for p in range(used)) and sorted(pages.free) == list(range(used, 50))
            assert pages.compacted() == {}


@pytest.mark.parametrize("how,what", [
    ({"k_bits": [4, 4]}, "one width per layer"),
    ({"v_bits": [5]}, "quantization bits"),
    ({"page_size": 48}, "page_size"),
    ({"head_dim": 96}, "head_dim"),
    ({"heads": 6}, "divisible by KV heads"),
    ({"kv_heads": 0}, "divisible by KV heads"),
    ({"window": -1}, "negative"),
])
def test_refusals(how, what):
    good = dict(k_bits=[4], v_bits=[4], heads=8, kv_heads=4, head_dim=128, row_pages=4, packed_pages=4, device="cpu")
    with pytest.raises(RuntimeError, match=what):
        PagedKVCache(**{**good, **how})
