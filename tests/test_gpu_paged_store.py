"""ops.paged_append / paged_quantize / paged_read / paged_copy against plain indexing and the operators' own quantizer."""
import pytest
import torch

from helpers import dequantize_torch
from paged_helpers import unpack_pages, unpack_rows

pytestmark = pytest.mark.gpu

POISON = float("nan")


def plan_of(dev, table, lens, new, kv_heads, D, page, packed=None):
    from kvmix_amd import ops

    return ops.paged_plan(torch.tensor(table), lens, packed or [0] * len(lens), new, kv_heads, kv_heads, D, page, dev)


@pytest.mark.parametrize("D,page", [(128, 64), (64, 32), (128, 256)])
@pytest.mark.parametrize("new", [[1, 1, 1], [5, 0, 130], [33, 64, 31]])
def test_append(dev, D, page, new):
    from kvmix_amd import ops

    H, old = 3, [7, 40, 63]
    lens = [a + b for a, b in zip(old, new)]
    width = max(-(-n // page) for n in lens)
    ids = torch.randperm(3 * width + 2, generator=torch.Generator().manual_seed(1)).tolist()
    table = [[ids.pop() if i * page < n else -1 for i in range(width)] for n in lens]
    rows = torch.full((3 * width + 2, H, 2, page, D), POISON, dtype=torch.float16, device=dev)
    n = sum(new)
    k, v = torch.randn(n, H, D, dtype=torch.float16, device=dev), torch.randn(n, H, D, dtype=torch.float16, device=dev)
    ops.paged_append(k, v, rows, plan_of(dev, table, lens, new, H, D, page))
    gk, gv = unpack_rows(rows)
    wk, wv = (torch.full((3 * width + 2, H, page, D), POISON, dtype=torch.float64) for _ in range(2))
    i = 0
    for s, m in enumerate(new):
        for t in range(lens[s] - m, lens[s]):
            wk[table[s][t // page], :, t % page], wv[table[s][t // page], :, t % page] = k[i].cpu().double(), v[i].cpu().double()
            i += 1
    assert torch.equal(gk.nan_to_num(9e9), wk.nan_to_num(9e9)) and torch.equal(gv.nan_to_num(9e9), wv.nan_to_num(9e9))


def test_append_strided_and_unaligned(dev):
    from kvmix_amd import ops

    H, D, page = 4, 128, 64
    qkv = torch.randn(9, 12, D, dtype=torch.float16, device=dev)
    plan = plan_of(dev, [[2], [0]], [5, 20], [5, 4], H, D, page)
    want, got = (torch.zeros(3, H, 2, page, D, dtype=torch.float16, device=dev) for _ in range(2))
    ops.paged_append(qkv[:, 4:8].contiguous(), qkv[:, 8:].contiguous(), want, plan)
    ops.paged_append(qkv[:, 4:8], qkv[:, 8:], got, plan)
    assert torch.equal(got, want)
    odd = torch.zeros(9 * H * D + 1, dtype=torch.float16, device=dev)[1:].view(9, H, D)
    odd.copy_(qkv[:, 4:8])
    got.zero_()
    ops.paged_append(odd, qkv[:, 8:].transpose(0, 1).contiguous().transpose(0, 1), got, plan)
    assert torch.equal(got, want)


def special(rows, seed):
    """Pages with constant groups, a very small and a very large range, signed zeros."""
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows.shape, generator=g)
    x[0, 0, :, :32] = 1.5
    x[0, 1] *= 1e-6
    x[1, 0] *= 3000.0
    x[1, 1, :, ::2] = 0.0
    x[1, 1, :, 1::2] = -0.0
    rows.copy_(x.half())


def quantized_as_the_operator_does(k, v, kb, vb):
    """k, v [n, H, P, D] fp16 -> the values that KVmix's own quantizer's codes stand for, rounded once to fp16"""
    from kvmix_amd import ops

    out = []
    for x, bits, keys in ((k, kb, True), (v, vb, False)):
        t = (x.transpose(2, 3) if keys else x).contiguous()
        code, scale, mn = ops.quantize_pack_dense3(t) if bits == 3 else ops.quantize_pack_last_dim_cuda(t, 32, bits)
        from helpers import unpack_codes_torch

        q = unpack_codes_torch(code, bits, bits == 3).double()
        y = q * scale.double().repeat_interleave(32, -1) + mn.double().repeat_interleave(32, -1)
        out.append((y.transpose(2, 3) if keys else y))
    return out


@pytest.mark.parametrize("kb,vb", [(1, 4), (2, 3), (3, 2), (4, 1)])
@pytest.mark.parametrize("D,page", [(128, 64), (64, 32), (128, 128), (64, 1024)])
def test_quantize_and_read(dev, kb, vb, D, page):
    from kvmix_amd import ops

    H = 2
    rows = torch.empty(4, H, 2, page, D, dtype=torch.float16, device=dev)
    special(rows, kb * 10 + vb)
    packed = torch.full((6, H, page // 32 * D * (kb + vb + 2)), -7, dtype=torch.int32, device=dev)
    pairs = torch.tensor([[0, 5], [1, 0], [3, 2]])
    ops.paged_quantize(rows, packed, pairs, kb, vb)
    assert (packed[[1, 3, 4]] == -7).all()
    k, v = unpack_rows(rows[[0, 1, 3]])
    want = quantized_as_the_operator_does(k.half().to(dev), v.half().to(dev), kb, vb)
    mine = unpack_pages(packed[[5, 0, 2]], D, kb, vb)
    read = ops.paged_read(packed, torch.tensor([5, 0, 2]), kb, vb, D)
    for w, m, r in zip(want, mine, read):
        assert torch.equal(w.cpu(), m)                              # codes, scales and minima
        assert r.shape == (3, page, H, D)
        assert torch.equal(r.cpu(), w.cpu().half().transpose(1, 2))  # their values, rounded once
    back = ops.paged_read(rows, torch.tensor([0, 1, 3]))
    assert torch.equal(back[0].cpu().double(), k.transpose(1, 2)) and torch.equal(back[1].cpu().double(), v.transpose(1, 2))


def test_infinities_and_nan_are_quantized_as_the_operator_does(dev):
    from kvmix_amd import ops

    rows = torch.randn(1, 1, 2, 32, 64, dtype=torch.float16, device=dev)
    rows[0, 0, 0, 3, 5] = float("inf")
    rows[0, 0, 0, 9, 6] = float("-inf")
    rows[0, 0, 0, 4, 7] = float("nan")
    rows[0, 0, 1].view(64, 32)[2, 8] = float("nan")
    packed = torch.zeros(1, 1, 64 * 10, dtype=torch.int32, device=dev)
    ops.paged_quantize(rows, packed, torch.tensor([[0, 0]]), 4, 4)
    k, v = (t.half().to(dev) for t in unpack_rows(rows))
    for want, got in zip(quantized_as_the_operator_does(k, v, 4, 4), unpack_pages(packed, 64, 4, 4)):
        assert torch.equal(want.cpu().nan_to_num(1e30, 2e30, 3e30), got.nan_to_num(1e30, 2e30, 3e30))


def test_many_pages(dev):
    """More pairs than one launch takes."""
    from kvmix_amd import ops

    n, H, D, page = 905, 1, 64, 32
    rows = torch.randn(n, H, 2, page, D, dtype=torch.float16, device=dev)
    packed = torch.zeros(n, H, D * 6, dtype=torch.int32, device=dev)
    to = torch.randperm(n)
    ops.paged_quantize(rows, packed, torch.stack([torch.arange(n), to], 1), 2, 2)
    k, v = ops.paged_read(packed, to, 2, 2, D)
    want = quantized_as_the_operator_does(*(t.half().to(dev) for t in unpack_rows(rows)), 2, 2)
    assert torch.equal(k.cpu(), want[0].cpu().half().transpose(1, 2)) and torch.equal(v.cpu(), want[1].cpu().half().transpose(1, 2))
    again = ops.paged_read(rows, to)
    assert torch.equal(again[0].cpu().double(), unpack_rows(rows)[0][to].transpose(1, 2))
    assert dequantize_torch is not None


@pytest.mark.parametrize("pools,pages,count", [(1, 5, 1), (3, 40, 20), (35, 9, 4), (2, 1000, 450)])
def test_copy(dev, pools, pages, count):
    from kvmix_amd import ops

    g = torch.Generator().manual_seed(pools)
    ids = torch.randperm(pages, generator=g)
    src, dst = ids[:count], ids[count:2 * count]
    src = src[torch.randint(0, count, (count,), generator=g)]  # a page may be copied to several places
    sizes = [(2, 8), (3, 1024), (1, 4), (2, 4096 + 4)]
    kinds = [torch.float16, torch.int32]
    made = []
    for i in range(pools):
        H, n = sizes[i % 4]
        x = torch.randint(-30000, 30000, (pages, H, n), generator=g)
        made.append(x.to(kinds[i % 2]).to(dev))
    want = [x.clone() for x in made]
    for x in want:
        x[dst.to(dev)] = x[src.to(dev)]
    ops.paged_copy(made, torch.stack([src, dst], 1))
    for a, b in zip(made, want):
        assert torch.equal(a, b)


def test_copy_refusals(dev):
    from kvmix_amd import ops

    x = torch.zeros(8, 2, 64, dtype=torch.int32, device=dev)
    for pairs, what in (([[0, 1], [2, 1]], "no order"), ([[0, 1], [1, 2]], "no order"), ([[3, 3]], "no order"), ([[0, 8]], "page number"), ([[-1, 2]], "page number")):
        with pytest.raises(RuntimeError, match=what):
            ops.paged_copy([x], torch.tensor(pairs))
    with pytest.raises(RuntimeError, match="same number of pages"):
        ops.paged_copy([x, x[:4].clone()], torch.tensor([[0, 1]]))
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.paged_copy([x[:, :, :32]], torch.tensor([[0, 1]]))
    with pytest.raises(RuntimeError, match="host memory"):
        ops.paged_copy([x], torch.tensor([[0, 1]], device=dev))
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.paged_copy([x.cpu()], torch.tensor([[0, 1]]))
    with pytest.raises(RuntimeError):
        ops.paged_copy([torch.zeros(8, 3, dtype=torch.int16, device=dev)], torch.tensor([[0, 1]]))  # pages of six bytes
    ops.paged_copy([x], torch.zeros(0, 2, dtype=torch.int32))
    ops.paged_copy([], torch.tensor([[0, 1]]))


def test_store_refusals(dev):
    from kvmix_amd import ops

    rows = torch.zeros(4, 2, 2, 64, 128, dtype=torch.float16, device=dev)
    packed = torch.zeros(3, 2, 2 * 128 * 10, dtype=torch.int32, device=dev)
    one = torch.tensor([[0, 0]])
    with pytest.raises(RuntimeError, match="page number"):
        ops.paged_quantize(rows, packed, torch.tensor([[4, 0]]), 4, 4)
    with pytest.raises(RuntimeError, match="page number"):
        ops.paged_quantize(rows, packed, torch.tensor([[0, 3]]), 4, 4)
    with pytest.raises(RuntimeError, match="written twice"):
        ops.paged_quantize(rows, packed, torch.tensor([[0, 1], [1, 1]]), 4, 4)
    with pytest.raises(RuntimeError, match="packed pages must be"):
        ops.paged_quantize(rows, packed, one, 4, 2)
    with pytest.raises(RuntimeError, match="quantization bits"):
        ops.paged_quantize(rows, packed, one, 4, 0)
    with pytest.raises(RuntimeError, match="Half"):
        ops.paged_quantize(rows.float(), packed, one, 4, 4)
    with pytest.raises(RuntimeError, match="fp16 pages must be"):
        ops.paged_quantize(rows[:, :, 0], packed, one, 4, 4)
    with pytest.raises(RuntimeError, match="page number"):
        ops.paged_read(packed, torch.tensor([3]), 4, 4, 128)
    with pytest.raises(RuntimeError, match="both widths"):
        ops.paged_read(packed, torch.tensor([0]), 4)
    with pytest.raises(RuntimeError):
        ops.paged_read(torch.zeros(1, 1, 2, 48, 128, dtype=torch.float16, device=dev), torch.tensor([0]))
    plan = plan_of(dev, [[9]], [5], [5], 2, 128, 64)
    k = torch.zeros(5, 2, 128, dtype=torch.float16, device=dev)
    with pytest.raises(RuntimeError, match="page number"):
        ops.paged_append(k, k, rows, plan)
    with pytest.raises(RuntimeError, match="keys and values must be"):
        ops.paged_append(k[:4], k[:4], rows, plan)
    with pytest.raises(RuntimeError, match="another size"):
        ops.paged_append(k, k, rows, plan_of(dev, [[1]], [5], [5], 2, 128, 32))
    with pytest.raises(RuntimeError, match="Half"):
        ops.paged_append(k.float(), k, rows, plan)
