"""The plan of a step over a paged cache (kvmix_paged_plan): what its items cover, where new tokens go, what it refuses.  No GPU."""
import random

import pytest

from kvmix_amd import _lib

ITEM = 12


def make(lens, packed, new, heads=8, kv_heads=2, page=64, D=128, seed=0, width=None):
    rng = random.Random(seed)
    width = max([-(-n // page) for n in lens] + [1]) if width is None else width
    free_packed, free_rows = list(range(10000)), list(range(10000))
    rng.shuffle(free_packed), rng.shuffle(free_rows)
    table = []
    for n, p in zip(lens, packed):
        row = [free_packed.pop() if i * page < p else free_rows.pop() for i in range(-(-n // page))]
        table.append(row + [-1] * (width - len(row)))
    return table, _lib.paged_plan(table, lens, packed, new, heads, kv_heads, D, page)


def items(words, at, n):
    return [tuple(words[at + ITEM * i:at + ITEM * i + 6]) for i in range(n)]


CASES = [
    ([1], [0], [1], {}),
    ([40, 64, 1000, 33], [0, 0, 832, 0], [1, 1, 1, 1], {}),
    ([32768, 100, 5000], [32640, 0, 4800], [1, 1, 1], {}),
    ([300, 0, 77, 4100], [128, 0, 0, 1984], [128, 0, 77, 2048], {}),
    ([8192] * 4, [6016] * 4, [2048] * 4, dict(heads=32, kv_heads=32)),
    ([3001, 2500, 2000, 1500, 1001, 999], [2752, 2240, 1728, 1248, 768, 736], [101] * 6, dict(heads=32, kv_heads=8, page=32)),
    ([700, 701, 2000], [512, 512, 1024], [3, 5, 900], dict(heads=8, kv_heads=1, page=128)),
    ([513, 200], [0, 0], [17, 33], dict(heads=4, kv_heads=4, page=1024, D=64)),
    ([50000], [49152], [300], dict(heads=8, kv_heads=1, page=256)),
]


@pytest.mark.parametrize("lens,packed,new,how", CASES)
def test_every_pair_of_row_and_token_is_covered_once(lens, packed, new, how):
    table, (plan, words) = make(lens, packed, new, **how)
    page, G = how.get("page", 64), how.get("heads", 8) // how.get("kv_heads", 2)
    assert plan["tokens"] == sum(new) and len(words) >= plan["words"]
    # sequences, tables and slots
    token = 0
    for s, (n, p, k) in enumerate(zip(lens, packed, new)):
        for at, count in ((plan["few_at"], plan["few"]), (plan["tile_at"], plan["tiles"]), (plan["join_at"], plan["joins"])):
            for i in range(count):
                if words[at + ITEM * i] == s:
                    assert words[at + ITEM * i + 6:at + ITEM * i + 10] == [token, k, n, p]
        at = plan["table_at"] + plan["table_stride"] * s
        assert words[at:at + plan["table_stride"]] == table[s]
        for i in range(k):
            t = n - k + i
            assert words[plan["slots_at"] + token + i] == table[s][t // page] * page + t % page
        token += k
    # blocks of pages that get new tokens: all slots, in order
    slots = words[plan["slots_at"]:plan["slots_at"] + token]
    stored = []
    for i in range(plan["stores"]):
        first, slot, count, _ = words[plan["store_at"] + 4 * i:plan["store_at"] + 4 * i + 4]
        assert first == len(stored) and count > 0 and slot % 32 + count <= 32
        stored += range(slot, slot + count)
    assert stored == slots
    # rows by keys
    few, tiles = items(words, plan["few_at"], plan["few"]), items(words, plan["tile_at"], plan["tiles"])
    joins = items(words, plan["join_at"], plan["joins"])
    done, parts = {}, {}
    for unit, most, these in ((32, plan["few_rows"], few), (64, 128, tiles)):
        for s, row0, rows, begin, end, part in these:
            assert 0 < rows <= most and 0 <= row0 and row0 + rows <= new[s] * G and 0 <= begin < end
            assert end <= -(-lens[s] // unit)
            done.setdefault((s, row0, rows, unit), []).append((begin, end))
            if part >= 0:
                parts.setdefault((s, row0), []).append((part, rows))
                assert part + rows <= plan["part_rows"]
    rows_seen = {}
    for (s, row0, rows, unit), spans in done.items():
        spans.sort()
        assert spans[0][0] == 0 and all(a[1] == b[0] for a, b in zip(spans, spans[1:]))
        last = lens[s] - new[s] + (row0 + rows - 1) // G  # the newest token that the rows see
        assert spans[-1][1] == last // unit + 1
        rows_seen.setdefault(s, []).append((row0, rows))
        assert (len(spans) > 1) == ((s, row0) in parts)
    for s, k in enumerate(new):
        spans = sorted(rows_seen.get(s, []))
        assert sum(n for _, n in spans) == k * G and all(a + n == b for (a, n), (b, _) in zip(spans, spans[1:]))
    # columns share the items of few rows out, to within a unit of four blocks
    dealt, seen = [], []
    for c in range(plan["few_columns"]):
        count, after = words[plan["few_at"] + ITEM * c + 10:plan["few_at"] + ITEM * c + 12]
        mine = [c] + list(range(after, after + count - 1))
        seen += mine
        dealt.append(sum(-(-(few[i][4] - few[i][3]) // 4) for i in mine))
    assert sorted(seen) == list(range(len(few)))
    assert not dealt or max(dealt) - min(dealt) <= 1
    # items of many rows: the longest first
    spans = [i[4] - i[3] for i in tiles]
    assert spans == sorted(spans, reverse=True)
    # joined rows are those in parts, and parts do not overlap
    assert {(j[0], j[1]) for j in joins} == set(parts)
    used = set()
    for s, row0, rows, spans, stride, part in joins:
        assert sorted(parts[(s, row0)]) == [(part + i * stride, rows) for i in range(spans)] and stride >= rows
        for i in range(spans * stride):
            assert part + i not in used
            used.add(part + i)
    assert not used or max(used) < plan["part_rows"]


def test_pages_that_the_pools_must_have():
    _, (plan, _) = make([300, 10], [128, 0], [1, 1], seed=3)
    table, _ = make([300, 10], [128, 0], [1, 1], seed=3)
    assert plan["packed_pages"] == max(table[0][:2]) + 1
    assert plan["row_pages"] == max(table[0][2:5] + table[1][:1]) + 1


def test_empty_batches():
    plan, words = _lib.paged_plan([], [], [], [], 8, 2, 128, 64)
    assert plan["tokens"] == plan["few"] == plan["tiles"] == plan["joins"] == 0
    _, (plan, _) = make([0, 64], [0, 0], [0, 0])
    assert plan["tokens"] == plan["few"] == plan["tiles"] == 0


@pytest.mark.parametrize("lens,packed,new,how,what", [
    ([10], [0], [11], {}, "do not fit"),           # more new tokens than tokens
    ([10], [0], [-1], {}, "do not fit"),
    ([100], [64], [40], {}, "do not fit"),         # a new token in a packed page
    ([100], [32], [1], {}, "do not fit"),          # not whole pages
    ([100], [-64], [1], {}, "do not fit"),
    ([100], [0], [1], {"width": 1}, "do not fit"),  # no page for the last tokens
    ([100], [0], [1], {"heads": 7}, "divisible by KV heads"),
    ([100], [0], [1], {"page": 48}, "not expressible"),
    ([100], [0], [1], {"D": 96}, "not expressible"),
    ([100], [0], [1], {"kv_heads": 0}, "negative size"),
])
def test_refusals(lens, packed, new, how, what):
    with pytest.raises(RuntimeError, match=what):
        page = how.get("page", 64)
        width = how.get("width", max(-(-n // page) for n in lens))
        table = [list(range(width)) for _ in lens]
        _lib.paged_plan(table, lens, packed, new, how.get("heads", 8), how.get("kv_heads", 2), how.get("D", 128), page)


def test_a_page_that_is_none():
    with pytest.raises(RuntimeError, match="page number"):
        _lib.paged_plan([[0, -1]], [100], [0], [1], 8, 2, 128, 64)
