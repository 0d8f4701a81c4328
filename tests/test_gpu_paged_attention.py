"""ops.paged_attention against a plain implementation in 64 bits."""
import math

import pytest
import torch

from paged_helpers import Batch, unpack_pages, unpack_rows

pytestmark = pytest.mark.gpu


def attend(b, **how):
    from kvmix_amd import ops

    return ops.paged_attention(b.q, b.rows, b.packed, b.plan, b.kb, b.vb, **how)


def check(b, got, scale=None):
    want, tol = b.want(scale)
    err = (got.cpu().double() - want).abs()
    assert got.shape == want.shape and torch.isfinite(got).all()
    assert (err <= tol).all(), float((err / tol).max())
    # Roundings are independent: over the whole result they add up to far less than the bound of each.  With four channels
    # ten times larger a logit of a rounded key is off by 2^-11 / sqrt(12) sqrt(sum q^2 k^2 / D) ~ 1.4e-4 * 2.2 = 3e-4 or so;
    # values, probabilities and the result by 2.8e-4 at most each.  Seven times that:
    assert float(err.norm() / want.norm()) < 4e-3


SHAPES = [
    # lens, packed, new, heads, kv_heads, D, page
    ([1], [0], [1], 4, 4, 128, 64),
    ([1], [0], [1], 4, 1, 64, 32),
    ([2, 31, 32, 33], [0, 0, 0, 0], [1, 1, 1, 1], 8, 2, 128, 32),
    ([64, 65, 128, 129], [0, 64, 64, 128], [1, 1, 1, 1], 4, 4, 128, 64),
    ([191, 500, 1001], [0, 256, 768], [1, 2, 3], 8, 8, 64, 128),
    ([700, 60, 1300], [512, 0, 1088], [1, 4, 1], 32, 8, 128, 64),       # 16 rows; a sequence without packed pages
    ([420], [256], [5], 12, 12, 128, 64),
    ([2100, 300], [1920, 64], [2, 5], 16, 4, 128, 64),                  # 8 and 20 rows: 32 rows at a time
    ([260, 900], [64, 640], [33, 8], 4, 4, 128, 64),                    # 33 rows: the other kernel; and 8 beside it
    ([300], [0], [300], 4, 2, 128, 32),                                 # a prompt: nothing packed
    ([640, 130], [256, 0], [129, 130], 2, 2, 128, 64),                  # a row more than a block takes; a prompt
    ([1500], [1024], [77], 8, 1, 64, 256),                              # 616 rows of one kv head
    ([333, 0, 400, 64], [128, 0, 256, 0], [100, 0, 0, 64], 8, 4, 64, 64),  # idle sequences
    ([5000], [4864], [1], 2, 2, 128, 64),                               # one long sequence: many spans
    ([6000], [5632], [300], 2, 1, 128, 512),
]


@pytest.mark.parametrize("shape", range(len(SHAPES)))
@pytest.mark.parametrize("bits", [(4, 4), (2, 2), (3, 2), (1, 3)])
def test_against_64_bits(dev, shape, bits):
    b = Batch(dev, *SHAPES[shape], *bits, seed=shape)
    check(b, attend(b))


@pytest.mark.parametrize("kb", [1, 2, 3, 4])
@pytest.mark.parametrize("vb", [1, 2, 3, 4])
@pytest.mark.parametrize("D", [64, 128])
def test_every_width(dev, kb, vb, D):
    for new in ([1, 1], [40, 3]):
        b = Batch(dev, [200, 333], [128, 192], new, 4, 2, D, 64, kb, vb, seed=kb * 16 + vb)
        check(b, attend(b))


def test_scale(dev):
    b = Batch(dev, [300, 90], [128, 0], [1, 40], 4, 2, 128, 64, 4, 4, seed=5)
    for scale in (1.0, 0.01):
        check(b, attend(b, scale=scale), scale)


@pytest.mark.parametrize("size", [1e-3, 30.0])
def test_small_and_large_values(dev, size):
    b = Batch(dev, [700, 450], [512, 256], [1, 50], 4, 2, 128, 64, 4, 2, seed=6, scale=size)
    got = attend(b)
    want, tol = b.want()
    assert ((got.cpu().double() - want).abs() <= tol).all()


@pytest.mark.parametrize("bits", [(4, 4), (2, 2), (1, 3)])
@pytest.mark.parametrize("q_size, k_size, scale", [(1e-3, 300.0, None), (1e-6, 1000.0, 20.0), (6000.0, 1e-3, 1e-2), (6000.0, 1000.0, 1e-9)])
def test_queries_of_other_sizes(dev, bits, q_size, k_size, scale):
    b = Batch(dev, [700, 450, 300], [512, 256, 128], [1, 50, 5], 4, 2, 128, 64, *bits, seed=17, scale=k_size)
    b.q[0, 1] = 0.0
    b.q *= q_size
    got = attend(b, scale=scale)
    want, tol = b.want(scale)
    assert ((got.cpu().double() - want).abs() <= tol).all()


def test_one_token_takes_all(dev):
    """A key that is far above all others: exactly its value comes back, and nothing overflows."""
    b = Batch(dev, [300, 300], [128, 128], [1, 64], 2, 2, 128, 64, 4, 4, seed=7)
    for s in range(2):
        page = int(b.table[s, 3])
        b.rows[page, :, 0, 7] = 0.0
        b.rows[page, :, 0, 7, 0] = 30000.0     # token 199 of each sequence
    b.q[..., 0] = 8.0
    got = attend(b)
    for s, rows in ((0, slice(0, 1)), (1, slice(1, 65))):
        _, v = b.dense(s)
        assert torch.equal(got[rows].cpu().double(), v[:, 199].expand(rows.stop - rows.start, 2, 128))


def test_new_tokens_see_their_own_past_only(dev):
    """What later tokens of the chunk hold does not reach earlier ones."""
    from kvmix_amd import ops

    b = Batch(dev, [400], [128], [150], 4, 2, 128, 64, 4, 4, seed=8)
    first = attend(b)
    plan = ops.paged_plan(b.table, [300], [128], [50], 4, 2, 128, 64, dev)   # the same pages, a hundred tokens earlier
    again = ops.paged_attention(b.q[:50].contiguous(), b.rows, b.packed, plan, 4, 4)
    assert torch.allclose(first[:50], again, rtol=2e-3, atol=2e-3)
    k, v = b.rows[:, :, 0].clone(), b.rows.clone()
    later = b.table[0, 300 // 64:]
    b.rows[later[1:].long()[later[1:] >= 0]] *= -3.0
    changed = attend(b)
    assert torch.equal(changed[:256 + 64 - 250], first[:256 + 64 - 250])      # tokens 250 .. 319: the pages up to 320 are unchanged
    assert not torch.equal(changed[80:], first[80:])
    del k, v


def test_pages_beyond_32_bit_offsets(dev):
    """Pools whose last pages lie behind 2^31 elements (4.3 GB of fp16 pages, 10.7 GB of packed ones)."""
    from kvmix_amd import ops

    b = Batch(dev, [300, 150], [128, 64], [1, 40], 4, 4, 128, 64, 4, 4, seed=13)
    want = attend(b)
    far = 1 << 15                                     # 65536 halves to a page of 4 heads
    rows = torch.empty(far + b.rows.shape[0], *b.rows.shape[1:], dtype=torch.float16, device=dev)
    rows[far:] = b.rows
    words = b.packed.shape[1] * b.packed.shape[2]     # 10240 to a page
    behind = -(-(1 << 31) // words) + 5
    packed = torch.empty(behind + b.packed.shape[0], *b.packed.shape[1:], dtype=torch.int32, device=dev)
    ids = torch.arange(b.packed.shape[0])
    k, v = ops.paged_read(b.packed, ids, 4, 4, 128)
    packed[behind:] = b.packed
    table = b.table.clone()
    for s, p in enumerate((2, 1)):
        table[s, :p] += behind
        table[s, p:] += far
    plan = ops.paged_plan(table, b.lens, b.packed_lens, b.new, 4, 4, 128, 64, dev)
    assert torch.equal(ops.paged_attention(b.q, rows, packed, plan, 4, 4), want)
    again = ops.paged_read(packed, ids + behind, 4, 4, 128)
    for got, ref in zip(again, (k, v)):               # by their bits: unused pages hold NaN
        assert torch.equal(got.view(torch.int16), ref.view(torch.int16))
    ops.paged_quantize(rows, packed, torch.tensor([[far, behind - 1]]), 4, 4)
    one = torch.zeros_like(b.packed)
    ops.paged_quantize(b.rows, one, torch.tensor([[0, 1]]), 4, 4)
    assert torch.equal(packed[behind - 1], one[1])
    ops.paged_copy([packed], torch.tensor([[behind + 1, 0]]))
    assert torch.equal(packed[0], b.packed[1])
    kv = torch.randn(41, 4, 128, dtype=torch.float16, device=dev)
    ops.paged_append(kv, kv, rows, plan)
    ops.paged_append(kv, kv, b.rows, b.plan)
    assert torch.equal(rows[far:].nan_to_num(9.0), b.rows.nan_to_num(9.0))


def test_strides_and_alignment_of_queries(dev):
    b = Batch(dev, [333, 64], [128, 0], [40, 1], 8, 4, 128, 64, 2, 4, seed=9)
    want = attend(b)
    wide = torch.zeros(41, 12, 128, dtype=torch.float16, device=dev)
    wide[:, 2:10] = b.q
    b.q = wide[:, 2:10]
    assert torch.equal(attend(b), want)
    heads_first = b.q.transpose(0, 1).contiguous().transpose(0, 1)
    b.q = heads_first
    assert torch.equal(attend(b), want)
    shifted = torch.zeros(41 * 8 * 128 + 1, dtype=torch.float16, device=dev)[1:].view(41, 8, 128)
    shifted.copy_(heads_first)
    b.q = shifted
    assert torch.equal(attend(b), want)


def test_another_stream_and_a_graph(dev):
    b = Batch(dev, [2000, 90, 640], [1792, 0, 448], [1, 1, 50], 8, 2, 128, 64, 4, 3, seed=10)
    want = attend(b)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = attend(b)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(got, want)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = attend(b)
    q = b.q.clone()
    for i in range(3):
        b.q.copy_(q * (i + 1))
        graph.replay()
        replayed = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(replayed, attend(b))


def test_results_do_not_change_from_call_to_call(dev):
    b = Batch(dev, [5000, 3000], [4864, 2816], [1, 70], 8, 2, 128, 64, 4, 4, seed=11)
    first = attend(b)
    for _ in range(3):
        assert torch.equal(attend(b), first)


def test_refusals(dev):
    from kvmix_amd import ops

    b = Batch(dev, [100, 64], [0, 0], [1, 1], 4, 2, 128, 64, 4, 4)
    with pytest.raises(RuntimeError, match="Half"):
        ops.paged_attention(b.q.float(), b.rows, b.packed, b.plan, 4, 4)
    with pytest.raises(RuntimeError, match="quantization bits"):
        ops.paged_attention(b.q, b.rows, b.packed, b.plan, 5, 4)
    with pytest.raises(RuntimeError, match="packed pages must be"):
        ops.paged_attention(b.q, b.rows, b.packed, b.plan, 4, 3)
    with pytest.raises(RuntimeError, match="queries must be"):
        ops.paged_attention(b.q[:1], b.rows, b.packed, b.plan, 4, 4)
    with pytest.raises(RuntimeError, match="page number"):
        ops.paged_attention(b.q, b.rows[:1].contiguous(), b.packed, b.plan, 4, 4)
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.paged_attention(b.q, b.rows.transpose(0, 1), b.packed, b.plan, 4, 4)
    with pytest.raises(RuntimeError):
        ops.paged_attention(b.q, b.rows, b.packed, b.plan, 4, 4, scale=-1.0)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.paged_attention(b.q, b.rows.cpu(), b.packed, b.plan, 4, 4)
    with pytest.raises(RuntimeError, match="expected all tensors on"):
        ops.paged_attention(b.q.cpu(), b.rows, b.packed, b.plan, 4, 4)
    with pytest.raises(RuntimeError, match="GPU only"):
        ops.paged_plan(b.table, [100, 64], [0, 0], [1, 1], 4, 2, 128, 64, "cpu")
    with pytest.raises(RuntimeError, match="as many lengths"):
        ops.paged_plan(b.table, [100], [0, 0], [1, 1], 4, 2, 128, 64, dev)
    with pytest.raises(RuntimeError, match="host memory"):
        ops.paged_plan(b.table.to(dev), [100, 64], [0, 0], [1, 1], 4, 2, 128, 64, dev)
    other = ops.paged_plan(b.table, [32, 32], [0, 0], [1, 1], 4, 2, 128, 32, dev)
    with pytest.raises(RuntimeError, match="another shape"):
        ops.paged_attention(b.q, b.rows, b.packed, other, 4, 4)
    nothing = ops.paged_plan(b.table, [100, 64], [0, 0], [0, 0], 4, 2, 128, 64, dev)
    assert ops.paged_attention(b.q[:0], b.rows, b.packed, nothing, 4, 4).shape == (0, 4, 128)


def test_layout_helpers_agree_with_the_rows(dev):
    """The plain reading of a packed page is the fp16 page that it was made of, to within half a step."""
    from kvmix_amd import ops

    g = torch.Generator().manual_seed(1)
    rows = torch.randn(2, 3, 2, 64, 64, generator=g).half().to(dev)
    packed = torch.zeros(2, 3, 2 * 64 * 10, dtype=torch.int32, device=dev)
    ops.paged_quantize(rows, packed, torch.tensor([[0, 1], [1, 0]]), 4, 4)
    for a, b in zip(unpack_pages(packed[[1, 0]], 64, 4, 4), unpack_rows(rows)):
        assert float((a - b).abs().max()) < 0.5 * 8 / 15 + 0.01 and math.isfinite(float(a.sum()))
