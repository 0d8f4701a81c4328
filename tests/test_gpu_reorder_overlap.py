"""Views of one storage that are reordered together: apart they are as the indexed copy, with memory in common they are refused."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def views(x):
    """x [B, 2, H, T, D]: keys and values, their heads, every other token, and columns, that lie between one another"""
    return [x[:, 0, :2, ::2], x[:, 0, :2, 1::2], x[:, 1, :, :, :24], x[:, 1, :, :, 24:], x[:, 0, 2:]]


@pytest.mark.parametrize("B", [4, 40, 100])
def test_views_of_one_storage(dev, B):
    from kvmix_amd import ops

    x = torch.randn(B, 2, 3, 10, 64, generator=torch.Generator().manual_seed(B)).half().to(dev)
    index = torch.randint(0, B, (B,), generator=torch.Generator().manual_seed(1)).to(dev)
    want = x[index]
    ops.reorder_rows(views(x), index)
    assert torch.equal(x, want)


def test_memory_in_common(dev):
    from kvmix_amd import ops

    x = torch.arange(6 * 640, device=dev).view(6, 640)
    before, index = x.clone(), torch.tensor([1, 2, 3, 4, 5, 0], device=dev)
    for tensors in ([x[:, :8], x[:, 4:]], [x[:, 4:], x[:, :8]], [x, x[:, 639:]], [x[:, ::2], x[:, 638:639]], [x.view(6, 8, 80)[:, :, :41], x.view(6, 8, 80)[:, :, 40:]],
                    [x[:, :8], x[:, 8:16], x[:, 15:17]], [x, x.view(torch.int32)]):
        with pytest.raises(RuntimeError, match="overlap"):
            ops.reorder_rows(tensors, index)
    assert torch.equal(x, before)
