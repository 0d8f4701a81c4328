"""Offsets beyond 32 bits: rows of projections, pages and logits that lie far from the first."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_adapters_of_rows_far_apart(dev):
    """Every 32776 values a row: the last begins beyond 2^31 values, of x, base and out."""
    from kvmix_amd import ops

    T, wide = 66000, 32776
    where = [0, 1, 30000, T - 65, T - 1]
    big = torch.empty(T, wide, dtype=torch.float16, device=dev)
    g = torch.Generator().manual_seed(1)
    x, base = torch.randn(T, 128, generator=g).half().to(dev), torch.randn(T, 64, generator=g).half().to(dev)
    big[:, 8:136], big[:, 136:200], big[:, 200:264] = x, base, 7.0
    a, b = (torch.randn(2, 16, 128, generator=g) / 11).half().to(dev), (torch.randn(2, 64, 16, generator=g) / 4).half().to(dev)
    plan = ops.adapter_plan([1, -1, 0], [T - 100, 30, 70], 2, dev)
    want = ops.add_adapters(base, x, a, b, plan)
    # (a step of the rows by hand: the small tensors are right)
    for t in where:
        i = 1 if t < T - 100 else 0
        y = base[t].double() + b[i].double() @ (a[i].double() @ x[t].double())
        assert torch.allclose(want[t].double(), y, rtol=2.0 ** -10, atol=2.0 ** -12)
    out = big[:, 200:264]
    ops.add_adapters(big[:, 136:200], big[:, 8:136], a, b, plan, out=out)
    assert torch.equal(out, want)
    ops.add_adapters(big[:, 136:200], big[:, 8:136], a, b, plan, out=big[:, 136:200])
    assert torch.equal(big[:, 136:200], want)


def test_pages_far_apart(dev):
    """More than 2^31 values of pages; the new tokens are in the first and the last of them."""
    from kvmix_amd import ops

    H, D, P, pages = 32, 128, 64, 4200
    rows = torch.empty(pages, H, 2, P, D, dtype=torch.float16, device=dev)
    rows[0], rows[-2:] = 0.0, 0.0
    table = torch.tensor([[pages - 1, pages - 2], [0, -1]], dtype=torch.int32)
    near = torch.zeros(3, H, 2, P, D, dtype=torch.float16, device=dev)
    qkv = torch.randn(100 + 3, 3 * H, D, generator=torch.Generator().manual_seed(2)).half().to(dev)
    angle = torch.rand(103, D, generator=torch.Generator().manual_seed(3)).to(dev)
    args = ([100, 30], [0, 0], [100, 3], H, H, D, P, dev)
    q = ops.paged_rope_append(qkv, angle.cos(), angle.sin(), rows, ops.paged_plan(table, *args))
    want = ops.paged_rope_append(qkv, angle.cos(), angle.sin(), near, ops.paged_plan(torch.tensor([[2, 1], [0, -1]], dtype=torch.int32), *args))
    assert torch.equal(q, want) and torch.equal(rows[-2:], near[1:]) and torch.equal(rows[0], near[0])


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_logits_far_apart(dev, dtype):
    from kvmix_amd import ops

    R, wide = 530, (1 << 22) + 3
    big = torch.empty(R, 1, wide, dtype=dtype, device=dev)
    near = torch.randn(R, 1, 3001, generator=torch.Generator().manual_seed(4)).to(dtype).to(dev)
    big[:, :, 5:3006] = near
    scores = torch.linspace(-9, -1, R, device=dev)[:, None].contiguous()
    for a, b in zip(ops.beam_select(big[:, :, 5:3006], scores, 3), ops.beam_select(near, scores, 3)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("kind,as_tensors", [(torch.float32, False), (torch.float16, False), (torch.float16, True)])
def test_a_projection_beyond_the_caches(dev, kind, as_tensors):
    """More than 128 MB of it: as sequence by sequence."""
    from kvmix_amd import ops

    H, KV, D, P, lens = 48, 16, 128, 64, [4000, 1, 3301]
    T = sum(lens)
    qkv = torch.randn(T, H + 2 * KV, D, generator=torch.Generator(device=dev).manual_seed(5), device=dev).half()
    angle = torch.rand(T, D, generator=torch.Generator().manual_seed(6)).to(dev)
    cos, sin = angle.cos().to(kind), angle.sin().to(kind)
    need = [-(-n // P) for n in lens]
    table = torch.full((3, max(need)), -1, dtype=torch.int32)
    ids = torch.randperm(sum(need), generator=torch.Generator().manual_seed(7)).int().split(need)
    for row, i in zip(table, ids):
        row[:len(i)] = i
    rows, apart = (torch.zeros(sum(need), KV, 2, P, D, dtype=torch.float16, device=dev) for _ in range(2))
    q = ops.paged_rope_append(qkv, cos, sin, rows, ops.paged_plan(table, lens, [0] * 3, lens, H, KV, D, P, dev), as_tensors)
    at = 0
    for s, n in enumerate(lens):
        part = slice(at, at + n)
        plan = ops.paged_plan(table[s:s + 1], [n], [0], [n], H, KV, D, P, dev)
        assert torch.equal(ops.paged_rope_append(qkv[part], cos[part], sin[part], apart, plan, as_tensors), q[part])
        at += n
    assert torch.equal(rows, apart)
