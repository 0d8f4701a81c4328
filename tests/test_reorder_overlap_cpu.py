"""Tensors that are reordered together must have no memory in common: against every byte of theirs.  No GPU."""
import random

import numpy as np
import pytest

from kvmix_amd import _lib
from test_beams_cpu import reorder

APART, OVERLAP = -7, -20  # (with no index, which calls whose tensors are apart get to)


def item(at, row_bytes, batch_stride, outer=1, outer_stride=0, inner=1, inner_stride=0):
    return {"base": (1 << 20) + at, "batch_stride": batch_stride, "outer": outer, "outer_stride": outer_stride, "inner": inner,
            "inner_stride": inner_stride, "row_bytes": row_bytes}


def taken(rows, p):
    starts = (p["base"] + p["batch_stride"] * np.arange(rows)[:, None, None] + p["outer_stride"] * np.arange(p["outer"])[:, None]
              + p["inner_stride"] * np.arange(p["inner"]))
    return starts.reshape(-1, 1) + np.arange(p["row_bytes"])


@pytest.mark.parametrize("items,code", [
    ([item(0, 64, 100), item(0, 64, 100)], OVERLAP),                                        # the same
    ([item(0, 32, 48), item(16, 32, 48)], OVERLAP),                                         # columns [0, 32) and [16, 48) of one tensor
    ([item(0, 16, 48), item(32, 16, 48), item(16, 16, 48)], APART),                         # columns beside one another
    ([item(0, 17, 48), item(32, 16, 48), item(16, 16, 48)], OVERLAP),
    ([item(0, 48, 96), item(48, 48, 96)], APART),                                           # every other entry
    ([item(0, 48, 96), item(96 * 3 + 47, 48, 96)], OVERLAP),                                # that a later entry of the other meets
    ([item(0, 48, 96), item(96 * 4, 48, 96)], APART),                                       # behind the last
    ([item(0, 8, 512, 4, 128, 8, 16), item(8, 8, 512, 4, 128, 8, 16)], APART),              # interleaved in every dimension
    ([item(0, 9, 512, 4, 128, 8, 16), item(8, 8, 512, 4, 128, 8, 16)], OVERLAP),
    ([item(0, 8, 512, 1, 0, 32, 16), item(8, 8, 512, 4, 128, 3, 16)], APART),               # the same with dimensions run together
    ([item(0, 8, 512, 1, 0, 32, 16), item(7, 8, 512, 4, 128, 3, 16)], OVERLAP),
    ([item(0, 4, 64, inner=4, inner_stride=16), item(8, 4, 64, inner=8, inner_stride=8)], OVERLAP),
    ([item(0, 64, 1 << 41), item(1 << 40, 64, 1 << 41)], APART),                            # far from one another
    ([item(0, 64, 1 << 41), item(1 << 42, 64, 1 << 41)], OVERLAP),
    ([item(0, 64, 100), item(0, 64, 100, inner=0)], APART),                                 # an empty one
    ([item(0, 64, 1 << 60)], -9),                                                           # beyond what there can be
    # a million rows at different strides: 7 i and 14 j + 3 never meet, 6 i and 10 j + 4 do
    ([item(0, 1, 1 << 30, inner=1 << 20, inner_stride=7), item(3, 1, 1 << 30, inner=1 << 20, inner_stride=14)], APART),
    ([item(0, 1, 1 << 30, inner=1 << 20, inner_stride=6), item(4, 1, 1 << 30, inner=1 << 20, inner_stride=10)], OVERLAP),
])
def test_layouts(items, code):
    assert reorder(4, *items, index=None) == code and reorder(4, *items[::-1], index=None) == code
    assert reorder(1, *items, index=None) == 0  # (one row is itself)


def test_too_fine_to_tell():
    """A million rows each, at strides that have nothing in common: apart, but refused rather than taken for granted."""
    p, q, n = 4194301, 4194319, 1 << 20
    at = next(a for a in range(2, 100) if not (((np.arange(n) * p - a) % q == 0) & (np.arange(n) * p >= a) & ((np.arange(n) * p - a) // q < n)).any())
    assert reorder(2, item(0, 1, 1 << 45, inner=n, inner_stride=p), item(at, 1, 1 << 45, inner=n, inner_stride=q), index=None) == OVERLAP


def test_any_two(seed=0):
    rng = random.Random(seed)
    seen = {APART: 0, OVERLAP: 0}
    for _ in range(4000):
        rows, pair = rng.randint(2, 4), []
        strides = sorted(rng.choice([3, 5, 8, 12, 16, 24, 40, 64, 100]) for _ in range(3))
        for _ in range(2):
            run = rng.randint(1, strides[0])
            inner_stride, outer_stride, batch = strides if rng.random() < 0.7 else sorted(rng.randint(run, 100) for _ in range(3))
            pair.append(item(rng.randint(0, 150), run, batch, rng.randint(1, 3), outer_stride, rng.randint(1, 3), inner_stride))
            if rng.random() < 0.2:  # the first dimension lies inside
                pair[-1]["batch_stride"], pair[-1]["outer_stride"] = pair[-1]["outer_stride"], pair[-1]["batch_stride"]
        want = OVERLAP if np.intersect1d(taken(rows, pair[0]), taken(rows, pair[1])).size else APART
        assert reorder(rows, *pair, index=None) == want, pair
        seen[want] += 1
    assert min(seen.values()) > 400


def test_many_tensors():
    """Any two of many, in any order."""
    items = [item(48 * i, 48, 48 * 65, inner=3, inner_stride=48 * 65 * 9) for i in range(65)]
    random.Random(1).shuffle(items)
    assert reorder(9, *items, index=None) == APART
    for bad in (item(48 * 65 * 9 * 2 + 48 * 65 * 8 + 48 * 64 + 47, 1, 1 << 20), item(48 * 30 + 20, 48, 1 << 20)):
        assert reorder(9, *items[:40], bad, *items[40:], index=None) == OVERLAP
    assert "overlap" in _lib.strerror(OVERLAP)


def test_any_views_of_one_storage(seed=1):
    """Several of alike strides, some of them in a storage of their own."""
    rng = random.Random(seed)
    seen = {APART: 0, OVERLAP: 0}
    for _ in range(2000):
        rows, items = rng.randint(2, 5), []
        inner_stride = rng.choice([4, 7, 16])
        outer_stride = inner_stride * rng.randint(1, 4) + rng.choice([0, 3])
        batch = outer_stride * rng.randint(1, 4) + rng.choice([0, 5, 40])
        for _ in range(rng.randint(2, 6)):
            p = item(rng.randint(0, batch) + rng.choice([0, 0, 0, 1000, 3 * batch]), rng.randint(1, max(1, inner_stride // 2)), batch, rng.randint(1, max(1, batch // outer_stride)),
                     outer_stride, rng.randint(1, max(1, outer_stride // inner_stride)), inner_stride)
            items.append(p)
        bytes_of = [np.unique(taken(rows, p)) for p in items]
        want = OVERLAP if sum(b.size for b in bytes_of) > np.unique(np.concatenate(bytes_of)).size else APART
        assert reorder(rows, *items, index=None) == want, items
        seen[want] += 1
    assert min(seen.values()) > 200
