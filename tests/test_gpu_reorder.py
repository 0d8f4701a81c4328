"""Tensors reordered in place: the same bits as a copy of the indexed ones, whatever the index, type, length and strides."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def tensors(B, dev, seed=0):
    """Of many types and layouts, views of larger ones among them: (the tensors, what they are views of)"""
    g = torch.Generator().manual_seed(seed)

    def ints(*shape, kind=torch.int32):
        return torch.randint(-100, 100, shape, generator=g).to(kind).to(dev)

    whole = [ints(B), ints(B, 1, kind=torch.bool), ints(B, 3, kind=torch.uint8), ints(B, 7, kind=torch.int64), ints(B, 4, 37, kind=torch.float16),
             ints(B, 2, 16, 55), ints(B, 3, 70, 64, kind=torch.float16), ints(B, 2, 100, 9), ints(B, 33, 31, kind=torch.int8), ints(5, B, 40, kind=torch.float16),
             ints(B, 6, 10, 8, kind=torch.float64), ints(B, 20000), ints(B, 9, 13, kind=torch.bfloat16), ints(1, kind=torch.int32).expand(1) if B == 1 else ints(B, 1)]
    views = [t for t in whole]
    views[5] = whole[5][..., 3:40]                    # the live part of rows
    views[6] = whole[6][:, :, 5:66]
    views[7] = whole[7][:, 1:, 10:, :5]
    views[9] = whole[9].transpose(0, 1)               # the first dimension lies inside
    views[10] = whole[10].permute(0, 3, 1, 2)
    views[8] = whole[8][:, ::2]
    return views, whole


INDEXES = {
    "nothing": lambda B, g: torch.arange(B),
    "all of one": lambda B, g: torch.full((B,), B // 2),
    "turned": lambda B, g: torch.arange(B).roll(1),
    "swapped": lambda B, g: torch.arange(B).flip(0),
    "random": lambda B, g: torch.randint(0, B, (B,), generator=g),
    "permuted": lambda B, g: torch.randperm(B, generator=g),
    "few": lambda B, g: torch.where(torch.rand(B, generator=g) < 0.2, torch.randint(0, B, (B,), generator=g), torch.arange(B)),
}


@pytest.mark.parametrize("kind", INDEXES)
@pytest.mark.parametrize("B", [1, 2, 4, 9, 33, 200, 1024])
def test_any_index(dev, B, kind):
    from kvmix_amd import ops

    index = INDEXES[kind](B, torch.Generator().manual_seed(B)).to(dev)
    views, whole = tensors(B, dev)
    if B == 1024:
        views, whole = views[:9], whole[:9]
    want = [t.clone() for t in whole]
    made, _ = tensors(B, dev)
    for i, t in enumerate(views):
        # the same view of the copy
        copy = want[i].as_strided(t.shape, t.stride(), t.storage_offset())
        copy.copy_(copy[index].clone())
    ops.reorder_rows(views, index)
    for i, (a, b) in enumerate(zip(whole, want)):
        assert torch.equal(a, b), i


@pytest.mark.parametrize("kind", INDEXES)
@pytest.mark.parametrize("B", [16, 32, 63, 64, 65])
def test_rows_of_a_wave(dev, B, kind):
    """As many as lanes, one more, and as many as registers hold; some of them gone round, some copied, in requests of their own."""
    from kvmix_amd import ops

    index = INDEXES[kind](B, torch.Generator().manual_seed(B + 1))
    eights = (torch.arange(B) // 8 * 8 + index % 8).clamp(max=B - 1)
    for i in (index.to(dev), eights.to(dev)):
        views, _ = tensors(B, dev, seed=1)
        want = [t[i].clone() for t in views]
        ops.reorder_rows(views, i)
        assert all(torch.equal(a, b) for a, b in zip(views, want))


def test_many_tensors_and_large_ones(dev):
    """More than one launch takes, an entry beyond 2^31 bytes from the first, NaN and infinities as they are."""
    from kvmix_amd import ops

    g = torch.Generator().manual_seed(3)
    many = [torch.randn(6, 5, 3 + i, generator=g).to(dev) for i in range(130)]
    many[7][2, 1, 3], many[8][3, 2, 2] = float("nan"), float("inf")
    index = torch.tensor([3, 3, 0, 5, 4, 1], device=dev)
    want = [t[index].view(torch.int32) for t in many]
    ops.reorder_rows(many, index)
    assert all(torch.equal(a.view(torch.int32), b) for a, b in zip(many, want))
    far = torch.empty(4, (1 << 30) + 5, dtype=torch.uint8, device=dev)
    for i in range(4):
        far[i] = i + 1
        far[i, -1] = 100 + i
    ops.reorder_rows([far], torch.tensor([2, 3, 2, 0], device=dev))
    assert [int(far[i, 0]) for i in range(4)] == [3, 4, 3, 1] and [int(far[i, -1]) for i in range(4)] == [102, 103, 102, 100]
    assert all(bool((far[i, :-1] == far[i, 0]).all()) for i in range(4))


def test_an_index_that_is_none(dev):
    from kvmix_amd import ops

    t = torch.arange(50, device=dev).view(5, 10)
    ops.reorder_rows([t], torch.tensor([4, -1, 5, 1 << 40, 0], device=dev))
    assert (t[:, 0] // 10).tolist() == [4, 1, 2, 3, 0]
    ops.reorder_rows([], torch.tensor([0, 1], device=dev))
    ops.reorder_rows([torch.empty(2, 0, 5, device=dev)], torch.tensor([1, 0], device=dev))
    ops.reorder_rows([torch.empty(0, 5, device=dev)], torch.zeros(0, dtype=torch.int64, device=dev))


def test_the_index_among_the_tensors(dev):
    from kvmix_amd import ops

    for B in (40, 300):
        index = torch.randperm(B, generator=torch.Generator().manual_seed(B)).to(dev)
        many = [torch.arange(B, device=dev)[:, None].expand(B, 3000).contiguous(), index, torch.arange(B, device=dev)]
        want = [t[index] for t in many]
        ops.reorder_rows(many, index)
        assert all(torch.equal(a, b) for a, b in zip(many, want))


def test_refusals(dev):
    from kvmix_amd import ops

    t, index = torch.zeros(4, 8, device=dev), torch.zeros(4, dtype=torch.int64, device=dev)
    for ts, i, match in [
        ([t], index[:3], "as many"), ([t], index.int(), "int64"), ([t], index[None], "int64"), ([t.cpu()], index, "GPU|cpu"), ([t], index.cpu(), "GPU|cpu"),
        ([t, t], index, "overlap"), ([torch.zeros(1, 8, device=dev).expand(4, 8)], index, "overlap"), ([torch.zeros(4, 1, device=dev).expand(4, 8)], index, "overlap"),
        ([torch.zeros(20, device=dev).as_strided((4, 8), (2, 1))], index, "overlap"), ([torch.zeros(4, 9, 9, 9, 9, device=dev)[:, ::2, ::2, ::2, ::2]], index, "two dimensions"),
        ([t.clone().requires_grad_()], index, "no derivative"), ([torch.zeros(1025, 2, device=dev)], torch.zeros(1025, dtype=torch.int64, device=dev), "1024"),
        ([torch.tensor(1.0, device=dev)], index, "as many"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            ops.reorder_rows(ts, i)


def test_captured_and_on_another_stream(dev):
    from kvmix_amd import ops

    views, _ = tensors(9, dev)
    index = torch.randint(0, 9, (9,), generator=torch.Generator().manual_seed(1)).to(dev)
    start = [t.clone() for t in views]
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.reorder_rows(views, index)
    side.synchronize()
    assert all(torch.equal(a, b[index]) for a, b in zip(views, start))
    graph, mine = torch.cuda.CUDAGraph(), index.clone()
    with torch.cuda.graph(graph):
        ops.reorder_rows(views, mine)
    for i in range(3):
        for a, b in zip(views, start):
            a.copy_(b)
        mine.copy_(index.roll(i))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b[index.roll(i)]) for a, b in zip(views, start))
