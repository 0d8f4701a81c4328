"""Rotated appends to a paged cache: against the rotation in 64 bits, the fp16 tensor expression and the plain append."""
import pytest
import torch

from paged_helpers import unpack_rows

pytestmark = pytest.mark.gpu


def _case(dev, lens, new, heads, kv_heads, D, page, seed=0):
    """Sequences of `lens` tokens of which `new` are new, in fp16 pages: (pages, plan, slots of the new tokens)"""
    from kvmix_amd import ops

    g = torch.Generator().manual_seed(seed)
    counts = [-(-n // page) for n in lens]
    ids, table, at = torch.randperm(sum(counts) + 2, generator=g), torch.full((len(lens), max(counts + [1])), -1, dtype=torch.int32), 0
    slots = []
    for s, (n, c) in enumerate(zip(lens, counts)):
        table[s, :c] = ids[at:at + c]
        at += c
        slots += [(int(table[s, t // page]), t % page) for t in range(n - new[s], n)]
    rows = torch.full((sum(counts) + 2, kv_heads, 2, page, D), 7.0, dtype=torch.float16, device=dev)
    return rows, ops.paged_plan(table, lens, [0] * len(lens), new, heads, kv_heads, D, page, dev), slots


def _tables(tokens, D, dtype, dev, seed=1):
    angle = torch.rand(tokens, D // 2, generator=torch.Generator().manual_seed(seed)) * 6.3
    angle = torch.cat([angle, angle], -1)
    return angle.cos().to(dtype).to(dev), angle.sin().to(dtype).to(dev)


SHAPES = [
    # lens, new, heads, kv heads, D, page
    ([1], [1], 1, 1, 128, 32),
    ([1], [1], 1, 1, 64, 32),
    ([5, 64, 65, 130], [1, 1, 1, 1], 32, 8, 128, 64),
    ([5, 64, 65, 130], [5, 0, 1, 77], 12, 12, 64, 64),
    ([33, 31, 32, 0, 200], [33, 3, 32, 0, 101], 8, 1, 128, 32),
    ([300, 1021], [300, 999], 32, 32, 128, 128),
    ([640] * 4, [640] * 4, 9, 3, 64, 64),
]


@pytest.mark.parametrize("dtype,as_tensors", [(torch.float16, False), (torch.float16, True), (torch.float32, False)])
@pytest.mark.parametrize("lens,new,heads,kv_heads,D,page", SHAPES)
def test_against_64_bits(dev, lens, new, heads, kv_heads, D, page, dtype, as_tensors):
    from kvmix_amd import ops

    rows, plan, slots = _case(dev, lens, new, heads, kv_heads, D, page)
    tokens = sum(new)
    # (every other projection is a view of something wider)
    wide = torch.randn(tokens, heads + 2 * kv_heads + 1, D, generator=torch.Generator().manual_seed(3)).half().to(dev)
    qkv = wide[:, 1:] if heads % 2 else wide[:, :-1].contiguous()
    cos, sin = _tables(tokens, D, dtype, dev)
    before = rows.clone()
    q = ops.paged_rope_append(qkv, cos, sin, rows, plan, as_tensors)
    assert q.shape == (tokens, heads, D) and q.dtype == torch.float16
    x = qkv[:, :heads + kv_heads].double().cpu()
    turned = torch.cat([-x[..., D // 2:], x[..., :D // 2]], -1)
    c, s = cos.double().cpu()[:, None], sin.double().cpu()[:, None]
    want = x * c + turned * s
    # one rounding to fp16 (2^-11 of the value, 2^-25 where it is subnormal) after fp32 arithmetic (two operations of 2^-24 each of
    # the products); rounded as tensors are, each product rounds to fp16 as well, and the sum of what they became
    size = (x * c).abs() + (turned * s).abs()
    tol = 2.0 ** -11 * want.abs() + 2.0 ** -22 * size + 2.0 ** -25
    if as_tensors:
        tol = 2.0 ** -11 * (want.abs() + size * (1 + 2.0 ** -11)) + 2.0 ** -22 * size + 3 * 2.0 ** -25
    assert ((q.double().cpu() - want[:, :heads]).abs() <= tol[:, :heads]).all()
    k, v = unpack_rows(rows)
    seen = torch.zeros(rows.shape[0], page, dtype=torch.bool)
    for t, (p, i) in enumerate(slots):
        assert ((k[p, :, i] - want[t, heads:]).abs() <= tol[t, heads:]).all()
        assert torch.equal(v[p, :, i], qkv[t, heads + kv_heads:].double().cpu())
        seen[p, i] = True
    # nothing else is written
    kb, vb = unpack_rows(before)
    for now, was in ((k, kb), (v, vb)):
        assert torch.equal(now.transpose(1, 2)[~seen], was.transpose(1, 2)[~seen])


@pytest.mark.parametrize("lens,new,heads,kv_heads,D,page", SHAPES)
def test_as_the_tensor_expression_and_the_plain_append(dev, lens, new, heads, kv_heads, D, page):
    """Where it is asked for, the same bits as rotating with tensors and appending, infinities and NaN among them."""
    from kvmix_amd import ops
    from kvmix_amd.decoder import apply_rope

    rows, plan, _ = _case(dev, lens, new, heads, kv_heads, D, page)
    tokens = sum(new)
    qkv = torch.randn(tokens, heads + 2 * kv_heads, D, generator=torch.Generator().manual_seed(4)).half().to(dev)
    qkv.view(-1)[::97] = float("inf")
    qkv.view(-1)[5::131] = float("nan")
    qkv.view(-1)[7::53] = 6e4
    cos, sin = _tables(tokens, D, torch.float16, dev)
    other = rows.clone()
    qk = apply_rope(qkv[:, :heads + kv_heads], cos[:, None], sin[:, None])
    ops.paged_append(qk[:, heads:], qkv[:, heads + kv_heads:], other, plan)
    q = ops.paged_rope_append(qkv, cos, sin, rows, plan, as_tensors=True)
    nan = torch.isnan(qk[:, :heads])
    assert torch.equal(torch.isnan(q), nan) and torch.equal(q[~nan], qk[:, :heads][~nan])
    nan = torch.isnan(other)
    assert torch.equal(torch.isnan(rows), nan) and torch.equal(rows[~nan], other[~nan])


def test_strides_and_one_row_of_tables(dev):
    """Any strides (copied where sixteen bytes do not fit), tables of one row for all tokens, offset pointers."""
    from kvmix_amd import ops

    heads, kv_heads, D, page = 6, 2, 64, 64
    rows, plan, _ = _case(dev, [40, 70], [40, 3], heads, kv_heads, D, page)
    base = torch.randn(43 * 10 * D + 1, generator=torch.Generator().manual_seed(5)).half().to(dev)
    qkv = base[1:].view(43, 10, D)
    cos, sin = _tables(1, D, torch.float32, dev)
    want_rows = rows.clone()
    want = ops.paged_rope_append(qkv.clone(), cos.expand(43, D).contiguous(), sin.expand(43, D).contiguous(), want_rows, plan)
    turned = qkv.transpose(0, 1).contiguous().transpose(0, 1)
    wide = torch.cat([cos, cos], -1)
    for x, c, s in ((qkv, cos[0], sin[0]), (turned, cos, sin), (qkv.transpose(1, 2).contiguous().transpose(1, 2), cos.expand(43, D), wide[:, D:].mul(0) + sin),
                    (qkv, wide.repeat(43, 1)[:, :D], sin.repeat(43, 2)[:, D:])):
        got = rows.clone()
        assert torch.equal(ops.paged_rope_append(x, c, s, got, plan), want) and torch.equal(got, want_rows)


def test_refusals(dev):
    from kvmix_amd import ops

    rows, plan, _ = _case(dev, [5, 64], [1, 2], 4, 2, 128, 64)
    qkv = torch.randn(3, 8, 128, device=dev).half()
    cos, sin = _tables(3, 128, torch.float32, dev)
    before = rows.clone()
    for bad, match in (((qkv[:2], cos, sin, rows, plan), "new tokens"), ((qkv[:, :7], cos, sin, rows, plan), "heads"),
                       ((qkv.float(), cos, sin, rows, plan), "Half"), ((qkv, cos[:2], sin, rows, plan), "one row"),
                       ((qkv, cos[:, :64], sin, rows, plan), "head_dim"), ((qkv, cos, sin.half(), rows, plan), "one type"),
                       ((qkv, cos.double(), sin.double(), rows, plan), "float16 or float32"), ((qkv, cos.cpu(), sin, rows, plan), "device|cpu"),
                       ((qkv.cpu(), cos, sin, rows, plan), "GPU|cpu"), ((qkv, cos, sin, rows[:, :1].contiguous(), plan), "another shape"),
                       ((qkv, cos, sin, rows[:1], plan), "page"), ((qkv.clone().requires_grad_(), cos, sin, rows, plan), "no derivative"),
                       ((qkv, cos, sin, rows, plan, True), "float16 tables")):
        with pytest.raises(RuntimeError, match=match):
            ops.paged_rope_append(*bad)
    assert torch.equal(rows, before)


def test_captured_and_on_another_stream(dev):
    from kvmix_amd import ops

    rows, plan, _ = _case(dev, [5, 64, 200], [1, 1, 90], 8, 2, 128, 64)
    qkv = torch.randn(92, 12, 128, device=dev).half()
    cos, sin = _tables(92, 128, torch.float32, dev)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = rows.clone()
        q = ops.paged_rope_append(qkv, cos, sin, got, plan)
    side.synchronize()
    want = rows.clone()
    assert torch.equal(ops.paged_rope_append(qkv, cos, sin, want, plan), q) and torch.equal(got, want)
    graph, x, into = torch.cuda.CUDAGraph(), qkv.clone(), rows.clone()
    with torch.cuda.graph(graph):
        out = ops.paged_rope_append(x, cos, sin, into, plan)
    for i in range(3):
        x.copy_(qkv * (i + 1) / 4)
        into.copy_(rows)
        graph.replay()
        torch.cuda.synchronize()
        want = rows.clone()
        assert torch.equal(ops.paged_rope_append(x, cos, sin, want, plan), out) and torch.equal(into, want)
