"""kvmix_amd.paged over stand-ins for the operators that move numbers about instead of keys: what every sequence holds, and what
forks share.  No GPU."""
import random

import pytest
import torch

from kvmix_amd import paged
from kvmix_amd.paged import OutOfPages, PagedKVCache


class Pools:
    """Pages as lists of numbers, one per token; the operators as PagedKVCache calls them."""

    def __init__(self, monkeypatch, page, **how):
        self.P, self.packings = page, 0
        for name in ("paged_quantize", "paged_copy", "paged_plan"):
            monkeypatch.setattr(paged.ops, name, getattr(self, name))
        args = dict(k_bits=[4], v_bits=[4], heads=2, kv_heads=1, head_dim=64, row_pages=40, packed_pages=60, page_size=page, window=2 * page, device="cpu")
        args.update(how)
        self.cache = PagedKVCache(**args)
        self.rows = [[None] * page for _ in range(args["row_pages"])]
        self.packed = [[None] * page for _ in range(args["packed_pages"])]

    def paged_quantize(self, rows, packed, pairs, kb, vb):
        assert len({int(q) for _, q in pairs}) == len(pairs)
        for r, q in pairs.tolist():
            assert None not in self.rows[r]
            self.packed[q] = list(self.rows[r])
            self.packings += 1

    def paged_copy(self, pools, pairs):
        pages = self.rows if pools is self.cache.rows else self.packed
        written, read = {q for _, q in pairs.tolist()}, {r for r, _ in pairs.tolist()}
        assert len(written) == len(pairs) and not written & read
        for r, q in pairs.tolist():
            pages[q] = list(pages[r])

    def paged_plan(self, table, lens, packed, new, *_):
        return table.tolist(), list(lens), list(packed), list(new)

    def append(self, step, numbers):
        """The step's new tokens into their pages; numbers [tokens]"""
        at = 0
        for row, n, p, k in zip(*step.plan):
            for t in range(n - k, n):
                assert t >= p
                self.rows[row[t // self.P]][t % self.P] = numbers[at]
                at += 1

    def read(self, s):
        seq = self.cache._sequence(s)
        pages = [self.packed[p] for p in seq.packed] + [self.rows[p] for p in seq.rows]
        return [x for page in pages for x in page][:seq.length]


@pytest.mark.parametrize("seed", range(6))
def test_forks_hold_the_same_page_once(monkeypatch, seed):
    """Random growth, forks, ends and compactions.  Every token is a number of its own: two packed pages that hold the same numbers
    were made of one fp16 page, and would be one."""
    rng = random.Random(seed)
    pools = Pools(monkeypatch, 32)
    cache, truth, number = pools.cache, {}, 0
    for _ in range(400):
        act = rng.random()
        if not truth or act < 0.1:
            truth[cache.new()] = []
        elif act < 0.3 and len(truth) < 12:
            s = rng.choice(list(truth))
            try:
                for t in cache.fork(s, 2):
                    truth[t] = list(truth[s])
            except OutOfPages:
                pass
        elif act < 0.4:
            s = rng.choice(list(truth))
            cache.free(s)
            del truth[s]
        elif act < 0.5:
            cache.compact()
        if not truth:
            continue
        grow = {s: rng.choice([0, 1, 5, 31, 32, 70]) for s in rng.sample(list(truth), rng.randint(1, len(truth)))}
        try:
            step = cache.step(grow)
        except OutOfPages:
            s = max(truth, key=lambda s: len(truth[s]))
            cache.free(s)
            del truth[s]
            continue
        numbers = list(range(number, number + sum(grow.values())))
        number += len(numbers)
        pools.append(step, numbers)
        for s, span in step.tokens().items():
            truth[s] += numbers[span]
        for s, want in truth.items():
            assert pools.read(s) == want
        used = {p for s in truth for p in cache._sequence(s).packed}
        assert len({tuple(pools.packed[p]) for p in used}) == len(used)
        assert cache.free_pages()[1] == 60 - len(used)
        assert cache.free_pages()[0] == 40 - len({p for s in truth for p in cache._sequence(s).rows})
    for s in list(truth):
        cache.free(s)
    assert cache.free_pages() == (40, 60)


def test_forks_pack_once(monkeypatch):
    """Eight answers from one prompt: the pages that were in the window at the fork are packed once, in one step or one by one."""
    for together in (True, False):
        pools = Pools(monkeypatch, 32, window=64, row_pages=64, packed_pages=16)
        cache = pools.cache
        a = cache.new()
        pools.append(cache.step({a: 320}), list(range(320)))
        all_of_them = [a] + cache.fork(a, 7)
        for i in range(4):
            for part in [all_of_them] if together else [[s] for s in all_of_them]:
                pools.append(cache.step({s: 16 for s in part}), [(i, s) for s in part for _ in range(16)])
        # (the last step begins with 368 tokens each, of which 304 have left the window: nine pages, all of them from before the fork)
        assert pools.packings == 9 and cache.free_pages()[1] == 16 - 9
        for s in all_of_them:
            assert pools.read(s) == list(range(320)) + [(i, s) for i in range(4) for _ in range(16)]


def test_room_for_shared_pages_is_asked_for_once(monkeypatch):
    """Three forks whose page leaves the window in the same step need one packed page, and one is there."""
    pools = Pools(monkeypatch, 32, window=0, row_pages=8, packed_pages=1)
    cache = pools.cache
    a = cache.new()
    pools.append(cache.step({a: 32}), list(range(32)))
    forks = cache.fork(a, 2)
    cache.step({s: 1 for s in [a, *forks]})
    assert cache.free_pages()[1] == 0 and all(pools.read(s)[:32] == list(range(32)) for s in [a, *forks])
