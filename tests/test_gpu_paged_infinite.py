"""ops.paged_attention where new tokens' values are infinite or NaN: they reach the tokens that see them and no others."""
import math

import pytest
import torch

from paged_helpers import Batch

pytestmark = pytest.mark.gpu


def place(b, s, token, channel, value, heads=slice(None)):
    """sets the value of a token of an fp16 page"""
    view = b.rows[int(b.table[s, token // b.page]), :, 1].view(b.kv_heads, b.page // 32, b.D, 32)
    t = token % b.page
    view[heads, t // 32, channel, t % 32] = value


CASES = [
    # lens, packed, new, heads, kv_heads, D, page, (sequence, token, channel, value) ...
    ([300], [128], [4], 4, 2, 128, 64, [(0, 298, 3, math.inf), (0, 299, 3, -math.inf), (0, 297, 127, math.nan), (0, 299, 0, math.inf)]),
    ([300, 90], [128, 0], [5, 1], 16, 4, 64, 64, [(0, 296, 63, math.inf), (0, 298, 1, math.nan), (1, 89, 5, math.inf)]),          # 20 rows
    ([420], [256], [150], 4, 2, 128, 64, [(0, 271, 1, math.inf), (0, 300, 2, -math.inf), (0, 301, 2, math.inf), (0, 419, 3, math.nan), (0, 320, 64, math.inf)]),
    ([77], [0], [77], 2, 2, 64, 32, [(0, 1, 0, math.inf), (0, 33, 0, -math.inf), (0, 76, 5, math.nan), (0, 40, 63, -math.inf)]),      # a prompt
    ([5000], [4864], [3], 2, 2, 128, 64, [(0, 4999, 7, math.inf), (0, 4998, 8, math.nan)]),                                    # spans that are joined
    ([5000], [4608], [130], 2, 1, 128, 64, [(0, 4999, 7, math.inf), (0, 4900, 8, math.nan), (0, 4880, 9, -math.inf)]),
    ([200, 131], [64, 0], [40, 131], 4, 4, 128, 64, [(0, 100, 4, math.inf), (0, 199, 5, math.inf), (1, 64, 6, math.nan)]),       # token 100 is an old one
    ([260], [0], [2], 2, 2, 128, 128, [(0, 3, 9, math.inf), (0, 259, 10, -math.inf)]),
]


@pytest.mark.parametrize("case", range(len(CASES)))
@pytest.mark.parametrize("bits", [(4, 4), (3, 2)])
def test_later_tokens_do_not_reach_earlier_ones(dev, case, bits):
    from kvmix_amd import ops

    *shape, marks = CASES[case]
    b = Batch(dev, *shape, *bits, seed=case)
    head = b.kv_heads - 1                      # the other heads keep their numbers

    def attend():
        return ops.paged_attention(b.q, b.rows, b.packed, b.plan, *bits)

    for s, token, channel, _ in marks:
        place(b, s, token, channel, 0.0, head)
    want = attend().clone()
    assert torch.isfinite(want).all()
    for s, token, channel, value in marks:
        place(b, s, token, channel, value, head)
    got = attend()
    G, at = b.heads // b.kv_heads, 0
    for s, n in enumerate(b.new):
        for i in range(n):
            mine = {}
            for t, token, channel, value in marks:
                if t == s and token <= b.lens[s] - n + i:
                    mine.setdefault(channel, []).append(value)
            for channel, values in mine.items():
                both = math.nan if math.inf in values and -math.inf in values else sum(values)
                want[at + i, head * G:, channel] = both
        at += n
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.nan_to_num(7.0, 8e4, -8e4), want.nan_to_num(7.0, 8e4, -8e4))
    assert torch.equal(attend().nan_to_num(7.0), got.nan_to_num(7.0))
