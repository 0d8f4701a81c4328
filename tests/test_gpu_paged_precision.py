"""How exact ops.paged_attention is: bounds of its own for what the general tests allow more."""
import math

import pytest
import torch

from paged_helpers import Batch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("packed", [False, True])
@pytest.mark.parametrize("new", [1, 40])
@pytest.mark.parametrize("steps", [75, 79])
def test_many_small_probabilities_add_up(dev, packed, new, steps):
    """100000 tokens, each 2^-25.4 (2^-26.7) of one that is far above them: together they weigh 2.3e-3 (9e-4).  As many heads as
    it takes for one block to have a whole sequence; its pages but for the first are one page of zeros and eights.

    A probability is a half relative to a largest of 2^7 or more, so it is off by 2^-25 / 2^7 = 2^-32 of the largest at most
    where it is below a normal half; the sum takes the same numbers.  Beside that the roundings of the result and of
    the probabilities' own (2^-11 each), and 2^-17 of fp32."""
    from kvmix_amd import ops

    T, P, D, H = 100000, 64, 64, 768
    pages = -(-T // P)
    rows = torch.zeros(3, H, 2, P, D, dtype=torch.float16, device=dev)
    large = 15 * steps / 64                                # (4 bits: code 15, a scale that is a half)
    rows[0, :, 0, 5, 0] = large
    rows[:, :, 1] = 8.0
    rows[0, :, 1].view(H, P // 32, D, 32)[:, 0, :, 5] = 0.0
    pool = torch.zeros(2, H, P // 32 * D * 10, dtype=torch.int32, device=dev)
    ops.paged_quantize(rows, pool, torch.tensor([[0, 0], [1, 1]]), 4, 4)
    table = torch.ones(1, pages, dtype=torch.int32)
    table[0, 0], table[0, -2:] = 0, 2
    plan = ops.paged_plan(table, [T], [(pages - 2) * P if packed else 0], [new], H, H, D, P, dev)
    q = torch.zeros(new, H, D, dtype=torch.float16, device=dev)
    q[..., 0] = 1.0
    got = ops.paged_attention(q, rows, pool, plan, 4, 4, scale=1.0).cpu().double()
    small = (T - new + torch.arange(new)).double()        # tokens beside the large one that each new token sees
    want = (8.0 * small / (small + torch.tensor(large, dtype=torch.float64).exp()))[:, None, None].expand_as(got)
    assert float(want.min()) > 5e-3
    tol = 2 * T * 2.0 ** -32 * 8.0 + (2.0 ** -10 + 2.0 ** -17) * want.abs()
    assert ((got - want).abs() <= tol).all(), (float(got.mean()), float(want.mean()))


@pytest.mark.parametrize("scale", [None, 1.0])
@pytest.mark.parametrize("bits", [(4, 4), (2, 2), (3, 2), (1, 3)])
@pytest.mark.parametrize("new,heads,kv_heads,D", [([1, 1], 4, 4, 128), ([1, 4], 8, 2, 128), ([5, 8], 8, 2, 128), ([3, 4], 16, 2, 64)])
def test_up_to_32_rows_keys_are_not_rounded(dev, new, heads, kv_heads, D, bits, scale):
    """Logits over packed keys are exact but for sums in fp32: with a scale of 1 they are near 30, and keys rounded to fp16 would
    be off by 30 * 2^-11 / sqrt(3) or so, 8e-3 of the result.

    What is left, over the norm: values and probabilities are halves, and so is the result, 2.1e-4 each and independent: 3.7e-4.
    Element by element: a logit is off by D roundings of its absolute sum (2^-23 each, with the second halves of the queries
    times scales 2^-21 once), the rest as in Batch.want."""
    from kvmix_amd import ops

    b = Batch(dev, [700, 450], [512, 256], new, heads, kv_heads, D, 64, *bits, seed=21)
    got = ops.paged_attention(b.q, b.rows, b.packed, b.plan, *bits, scale=scale).cpu().double()
    want, _ = b.want(scale)
    s, G, at, tols = D ** -0.5 if scale is None else scale, heads // kv_heads, 0, []
    for i, n in enumerate(new):
        k, v = b.dense(i)
        T = b.lens[i]
        q = b.q[at:at + n].cpu().double().reshape(n, kv_heads, G, D).permute(1, 2, 0, 3)
        dead = torch.arange(T) > (T - n + torch.arange(n))[:, None]
        p = torch.softmax((q @ k[:, None].transpose(-1, -2) * s).masked_fill(dead, -math.inf), -1)
        e = (q.abs() @ k[:, None].abs().transpose(-1, -2) * s * (D * 2.0 ** -23 + 2.0 ** -21)).masked_fill(dead, 0.0).amax(-1, keepdim=True)
        tol = (torch.exp(2 * e) - 1 + 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -17) * (p @ v[:, None].abs()) + T * 2.0 ** -32 * v.abs().amax(1)[:, None, None]
        tols.append(tol.permute(2, 0, 1, 3).reshape(n, heads, D))
        at += n
    err = (got - want).abs()
    assert (err <= torch.cat(tols) + 2.0 ** -11 * want.abs() + 2.0 ** -24).all()
    assert float(err.norm() / want.norm()) < 5e-4
