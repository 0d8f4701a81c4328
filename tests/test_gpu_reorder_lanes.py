"""Tensors of fewer pieces than a wave has lanes, or some more: the lanes without a piece hold sources of rows all the same."""
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("B", [20, 33, 64])
@pytest.mark.parametrize("pieces", [1, 3, 63, 65, 130, 255, 257])
def test_lanes_without_a_piece(dev, B, pieces):
    from kvmix_amd import ops

    g = torch.Generator().manual_seed(B + pieces)
    for index in (torch.arange(B).roll(-1), torch.arange(B).flip(0), torch.where(torch.arange(B) < B // 2, torch.arange(B) + (B + 1) // 2, torch.arange(B)),
                  torch.where(torch.arange(B) < 9, B - 1 - torch.arange(B), torch.arange(B))):
        for cut in (0, 5):  # whole pieces, and a last one of eleven bytes
            t = torch.randint(0, 255, (B, 16 * pieces - cut), generator=g).to(torch.uint8).to(dev)
            want = t[index.to(dev)]
            ops.reorder_rows([t], index.to(dev))
            assert torch.equal(t, want)
