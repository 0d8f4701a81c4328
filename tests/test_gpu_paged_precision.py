"""How exact ops.paged_attention is: bounds of its own for what the general tests allow more."""
import pytest
import torch

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
