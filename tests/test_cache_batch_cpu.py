"""The tails of a cache take new tokens of the sequences, heads and widths that they hold, and of no others.  No GPU."""
import pytest
import torch

from kvmix_amd.cache import _Tail


@pytest.mark.parametrize("shape", [(1, 2, 1, 8), (4, 1, 1, 8), (4, 2, 1, 1), (3, 2, 5, 8)])
def test_tokens_of_other_shapes(shape):
    """One sequence, head or channel would otherwise be repeated for all."""
    tail = _Tail()
    tail.append(torch.ones(4, 2, 3, 8), reserve=16)
    with pytest.raises(RuntimeError, match="4 sequences"):
        tail.append(torch.zeros(shape), reserve=16)
    assert tail.len == 3 and torch.equal(tail.view(), torch.ones(4, 2, 3, 8)) and not tail.buf[:, :, 3:].any()
    tail.append(torch.zeros(4, 2, 2, 8), reserve=16)
    assert tail.len == 5
