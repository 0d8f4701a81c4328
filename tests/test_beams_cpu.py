"""Calls of the beams' operators that are refused before anything is launched.  No GPU."""
import ctypes

import pytest

from kvmix_amd import _lib


def select(**kw):
    c = _lib.BeamSelect()
    for name in ("logits", "scores", "out_scores", "parents", "tokens"):
        setattr(c, name, 1 << 20)
    c.row_stride = c.vocab = 1000
    c.dtype, c.requests, c.beams, c.count = 1, 3, 4, 4
    for name, value in kw.items():
        setattr(c, name, value)
    return c


@pytest.mark.parametrize("change,code", [
    ({"dtype": 3}, -6), ({"beams": 0}, -8), ({"beams": 65}, -9), ({"count": 0}, -8), ({"count": 65}, -9), ({"vocab": 3}, -9), ({"vocab": 0}, -8),
    ({"vocab": (1 << 20) + 1}, -9), ({"vocab": 1 << 20, "beams": 33, "count": 33}, -9), ({"requests": -1}, -8), ({"requests": 1 << 24}, -9),
    ({"stay": 1, "count": 8}, -8), ({"done": 1 << 20, "end": 1000}, -8), ({"done": 1 << 20, "end": -1}, -8), ({"row_stride": -1}, -8),
    ({"logits": None}, -7), ({"tokens": None}, -7), ({}, -11), ({"requests": 0}, 0),
])
def test_selections_that_are_refused(change, code):
    """(with no workspace, which the last one gets to)"""
    c = select(**change)
    assert _lib.load().kvmix_beam_select(ctypes.byref(c), None, 0, None) == code


@pytest.mark.parametrize("dtype,per", [(1, 4), (0, 8), (2, 8)])
def test_parts_of_a_row(dtype, per):
    """What the workspace holds says how many parts there are: enough for what a block holds, no more lists than the join takes."""
    L = _lib.load()
    for requests, beams in ((1, 1), (1, 4), (64, 8), (1, 64), (1000, 32)):
        for vocab in (1, 7, 300, 8191, 8192, 8193, 32000, 128003, 1 << 19, 1 << 20):
            if beams * vocab > 1 << 25 or requests * beams * (vocab // 2048 + 1) >= 1 << 24:
                continue
            count = min(4, vocab)
            c = select(requests=requests, beams=beams, vocab=vocab, row_stride=vocab, dtype=dtype, count=count)
            need = L.kvmix_beam_select_workspace_bytes(ctypes.byref(c))
            parts, left = divmod(need, requests * beams * (8 + 8 * count))
            assert left == 0 and -(-vocab // (256 * 8 * per)) <= parts <= max(1, -(-vocab // 8)) and parts * beams <= 4096


def reorder(rows, *items, index=1 << 20):
    made = (_lib.Reorder * max(len(items), 1))()
    for at, kw in zip(made, items):
        at.base, at.batch_stride, at.outer, at.outer_stride, at.inner, at.inner_stride, at.row_bytes = 1 << 20, 4096, 1, 0, 4, 1024, 512
        for name, value in kw.items():
            setattr(at, name, value)
    return _lib.load().kvmix_reorder_rows(made, len(items), index, rows, None)


@pytest.mark.parametrize("change,code", [
    ({"base": None}, -7), ({"row_bytes": -1}, -8), ({"inner_stride": 511}, -8), ({"outer": 2, "outer_stride": 100}, -8), ({"batch_stride": 511}, -8),
    ({"inner": 1 << 32, "inner_stride": 1 << 10}, -9), ({"row_bytes": 1 << 36, "inner": 1, "batch_stride": 1 << 37}, -9), ({"outer": -1}, -8),
])
def test_tensors_that_are_not_reordered(change, code):
    assert reorder(4, {}, change) == code


def test_nothing_to_reorder():
    assert reorder(0) == 0 and reorder(1, {}) == 0 and reorder(5) == 0 and reorder(4, {"inner": 0}, {"row_bytes": 0}) == 0
    assert reorder(-1) == -8 and reorder(1025, {}) == -9 and reorder(4, {}, index=None) == -7
