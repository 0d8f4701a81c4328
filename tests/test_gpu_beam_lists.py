"""Selections from as many parts of rows as there can be: against 64 bits."""
import pytest
import torch

from test_gpu_beam_select import check, plain

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("W,V,count", [(33, 1015809, 5), (48, 699050, 48), (63, 532481, 64), (64, 1 << 19, 3)])
def test_the_most_parts(dev, W, V, count):
    """Up to 66 parts to a beam, 4158 to a request, the last one of a single value; the best ones are in the last parts of the last beams,
    behind the 4096th of them."""
    from kvmix_amd import ops

    g = torch.Generator(device=dev).manual_seed(V)
    logits, scores = torch.randn(1, W, V, generator=g, device=dev) * 3, -8 * torch.rand(1, W, generator=g, device=dev)
    logits[0, -2:, -3:] = 27.0 - torch.arange(6, device=dev).view(2, 3)
    check(ops.beam_select(logits, scores, count), plain(logits, scores, count))
    done = torch.zeros(1, W, dtype=torch.bool)
    done[0, ::5] = True
    check(ops.beam_select(logits, scores, count, done.to(dev), V - 1), plain(logits, scores, count, done, V - 1))
