"""Which token goes to which piece of the adapters' work, and what calls are refused before anything is launched.  No GPU."""
import ctypes

import pytest

from kvmix_amd import _lib


@pytest.mark.parametrize("adapters,counts,n", [
    ([], [], 0), ([0], [0], 1), ([0], [1], 1), ([-1], [5], 3), ([2, -1, 2, 0, 2], [1, 70, 64, 130, 3], 4), ([1] * 65, [1] * 65, 2),
    ([i % 40 for i in range(64)], [1] * 64, 40), ([0, 1, -3, 0], [1021, 0, 17, 300], 2),
])
def test_every_token_once(adapters, counts, n):
    plan, words = _lib.adapter_plan(adapters, counts, n)
    tokens = [i for i, m in zip(adapters, counts) for _ in range(m)]
    assert plan["tokens"] == len(tokens) and plan["rows"] == sum(i >= 0 for i in tokens) and plan["words"] == len(words)
    assert plan["adapters"] == max([i + 1 for i, m in zip(adapters, counts) if m and i >= 0] + [0])
    rows = words[plan["rows_at"]:]
    assert sorted(rows) == list(range(len(tokens)))
    seen, at = [], 0
    for t in range(plan["tiles"] + plan["bare"]):
        adapter, first, count, _ = words[4 * t:4 * t + 4]
        assert first == at and 1 <= count <= 64 and (adapter < 0) == (t >= plan["tiles"]) and (adapter < 0 or count <= plan["most"])
        assert all(tokens[r] == adapter or (adapter < 0 and tokens[r] < 0) for r in rows[first:first + count])
        assert rows[first:first + count] == sorted(rows[first:first + count])
        at += count
        seen.append(count)
    assert at == len(tokens)


@pytest.mark.parametrize("adapters,counts,n", [([0], [200], 1), ([0, 1, 0], [3, 2, 70], 2), ([-1, 0, -1], [1, 100, 1], 1), ([0, 1] * 40, [1] * 80, 2)])
def test_pieces_of_tokens_that_follow_one_another(adapters, counts, n):
    """Their first token, by which they are found without the list, or -1."""
    plan, words = _lib.adapter_plan(adapters, counts, n)
    for t in range(plan["tiles"] + plan["bare"]):
        _, first, count, at = words[4 * t:4 * t + 4]
        rows = words[plan["rows_at"] + first:plan["rows_at"] + first + count]
        assert at == (rows[0] if rows == list(range(rows[0], rows[0] + count)) else -1)


@pytest.mark.parametrize("adapters,counts,n,code", [([3], [1], 3, -19), ([0], [-1], 1, -8), ([0, 0], [1 << 30, 1], 1, -9), ([0], [1], -1, -8), ([0], [1], (1 << 20) + 1, -9)])
def test_plans_that_are_refused(adapters, counts, n, code):
    plan = _lib.AdapterPlan()
    m = (ctypes.c_int64 * len(adapters))
    assert _lib.load().kvmix_adapter_plan(m(*adapters), m(*counts), len(adapters), n, None, 0, ctypes.byref(plan)) == code


def call(**kw):
    c = _lib.Adapters()
    for name in ("x", "a", "b", "base", "out"):
        setattr(c, name, 1 << 20)
    c.x_token_stride = c.a_rank_stride = 4096
    c.a_adapter_stride, c.b_adapter_stride, c.b_row_stride = 16 * 4096, 16 * 1024, 16
    c.base_token_stride = c.out_token_stride = 1024
    c.adapters, c.rank, c.k, c.n, c.dtype = 4, 16, 4096, 1024, 0
    for name, value in kw.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("change,code", [
    ({"dtype": 1}, -6), ({"rank": 0}, -8), ({"rank": 20}, -9), ({"rank": 136}, -9), ({"k": 4100}, -9), ({"n": 1 << 25}, -9), ({"adapters": 2}, -19),
    ({"x": (1 << 20) + 2}, -9), ({"x_token_stride": 4097}, -9), ({"b_row_stride": 20}, -9), ({"out_token_stride": 2048, "out": 1 << 20}, -8), ({"x": None}, -7),
    ({"a": None}, -7), ({"out_token_stride": 1016, "out": 1 << 21}, -8), ({"scales": None}, -11),
])
def test_calls_that_are_refused(change, code):
    """With a plan of three adapters and no workspace, which the last one gets to."""
    plan, words = _lib.adapter_plan([0, 2, 1], [1, 5, 70], 3)
    p = _lib.AdapterPlan(**plan)
    c, L = call(**change), _lib.load()
    listed = (ctypes.c_int32 * len(words))(*words)
    assert L.kvmix_add_adapters(ctypes.byref(p), listed, ctypes.byref(c), None, 0, None) == code
    if code not in (-7, -8, -11):
        assert L.kvmix_add_adapters_workspace_bytes(ctypes.byref(p), ctypes.byref(c)) == 0


def test_workspace():
    """Every stretch of k has its sums for every token with an adapter."""
    plan, _ = _lib.adapter_plan([0, -1], [100, 50], 1)
    p = _lib.AdapterPlan(**plan)
    for rank, padded in ((8, 16), (16, 16), (24, 32), (128, 128)):
        need = _lib.load().kvmix_add_adapters_workspace_bytes(ctypes.byref(p), ctypes.byref(call(rank=rank)))
        assert need % (100 * padded * 4) == 0 and 1 <= need // (100 * padded * 4) <= 16
