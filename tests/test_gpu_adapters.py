"""Low-rank adapters of many requests: against 64 bits, over sizes, masks of sequences without one, strides and types."""
import pytest
import torch

pytestmark = pytest.mark.gpu

HALF_STEP = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def _inputs(dev, counts, n_adapters, rank, k, n, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    tokens = sum(counts)
    x = torch.randn(tokens, k, generator=g) * (1 + 9 * (torch.rand(k, generator=g) < 0.02))
    a = torch.randn(n_adapters, rank, k, generator=g) * k ** -0.5
    b = torch.randn(n_adapters, n, rank, generator=g) * rank ** -0.5
    return [t.to(dtype).to(dev) for t in (torch.randn(tokens, n, generator=g), x, a, b)] + [torch.randn(n_adapters, generator=g).to(dev)]


def _want(base, x, a, b, scales, adapters, counts):
    """(the result in float64, what it may be off by).

    u = A x in fp32: each of the k products is exact, its sum off by 2^-24 of the absolute sum per addition at worst (k of them).  u enters
    the second product to 2^-22 (bf16: 2^-16) of the token's largest; that sum in fp32 as well, then one rounding to the type."""
    dtype = base.dtype
    base, x, a, b = (t.double().cpu() for t in (base, x, a, b))
    out, tol, at = base.clone(), torch.zeros_like(base), 0
    for i, m in zip(adapters, counts):
        if i >= 0 and m:
            s = 1.0 if scales is None else float(scales[i])
            u, size = x[at:at + m] @ a[i].t(), x[at:at + m].abs() @ a[i].abs().t()
            out[at:at + m] += s * u @ b[i].t()
            kept = u.abs().amax(-1, keepdim=True) * (2.0 ** -22 if dtype == torch.float16 else 2.0 ** -16)
            off = x.shape[1] * 2.0 ** -24 * size + kept
            e = (off @ b[i].abs().t() + 2 * a.shape[1] * 2.0 ** -24 * (u.abs() @ b[i].abs().t())) * abs(s)
            tol[at:at + m] = e + HALF_STEP[dtype] * (out[at:at + m].abs() + e) + TINY[dtype] + 2.0 ** -23 * (out[at:at + m].abs() + base[at:at + m].abs())
        at += m
    return out, tol


CASES = [
    # adapters, counts, of how many, rank, k, n
    ([0], [1], 1, 8, 8, 8),
    ([2], [1], 4, 16, 4096, 4096),
    ([0, -1, 1], [1, 1, 1], 2, 24, 520, 40),
    ([i % 5 for i in range(37)], [1] * 37, 5, 16, 1032, 1000),
    ([1, 0, -1, 1], [33, 70, 9, 129], 2, 32, 776, 264),
    ([0, 1, 0, 3, -1], [0, 200, 1, 16, 64], 4, 64, 2048, 512),
    ([0, 2], [48, 100], 3, 128, 4096, 136),
    ([1] * 3, [17, 15, 65], 2, 72, 40, 24),
    ([-1, -1], [5, 100], 1, 16, 64, 72),
    ([0] * 130, [1] * 130, 1, 8, 11008, 96),
    ([0, 1, 2], [20, 31, 17], 3, 8, 136, 136),      # tiles of two sixteens, k a little more than a step
    ([1, 0], [64, 300], 2, 48, 5000, 1160),         # stretches of k that are not alike, the last step cut off
    ([0, 0, 0], [40, 1, 60], 1, 16, 128, 128),
    ([0, 1], [1, 3], 2, 64, 4096, 264),             # few tokens, much to read
    ([0], [5], 1, 8, 11008, 1000),
    ([1, -1, 0], [16, 20, 2], 2, 32, 2048, 2056),   # few tokens and little to read, to the last of it
    ([0, 2, 1], [1, 1, 1], 3, 64, 1024, 520),
    ([0, 1, 0], [3, 1, 2], 2, 8, 4232, 40),
]


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
@pytest.mark.parametrize("adapters,counts,of,rank,k,n", CASES)
def test_against_64_bits(dev, adapters, counts, of, rank, k, n, dtype):
    from kvmix_amd import ops

    base, x, a, b, scales = _inputs(dev, counts, of, rank, k, n, dtype)
    plan = ops.adapter_plan(adapters, counts, of, dev)
    assert plan.tokens == sum(counts)
    for s in (scales, None):
        want, tol = _want(base, x, a, b, s, adapters, counts)
        out = ops.add_adapters(base, x, a, b, plan, s)
        assert out.dtype == dtype and out.shape == base.shape
        assert ((out.double().cpu() - want).abs() <= tol).all()
        # the same into base itself
        mine = base.clone()
        assert ops.add_adapters(mine, x, a, b, plan, s, out=mine) is mine and torch.equal(mine, out)


def test_rows_without_an_adapter_are_left_alone(dev):
    from kvmix_amd import ops

    counts, adapters = [3, 70, 2], [0, -1, 1]
    base, x, a, b, scales = _inputs(dev, counts, 2, 16, 64, 72, torch.float16)
    x[3:73] = float("nan")  # of no concern to anything
    base[5], base[6] = float("inf"), float("nan")
    plan = ops.adapter_plan(adapters, counts, 2, dev)
    out = ops.add_adapters(base, x, a, b, plan, scales)
    assert torch.equal(out[3:73].view(torch.int16), base[3:73].view(torch.int16))
    assert torch.isfinite(out[:3]).all() and torch.isfinite(out[73:]).all()


def test_infinities_and_large_values(dev):
    """u beyond fp16 is no matter; an infinite or missing value of x reaches its own token and no other."""
    from kvmix_amd import ops

    for dtype in (torch.float16, torch.bfloat16):
        counts, adapters = [40], [0]
        base, x, a, b, _ = _inputs(dev, counts, 1, 16, 256, 64, dtype)
        b *= 1e-3
        x[3] = 3e4
        a[0, 0] = 20.0  # u = 1.5e8
        plan = ops.adapter_plan(adapters, counts, 1, dev)
        b[0, :, 0] = 1e-6
        want, tol = _want(base, x, a, b, None, adapters, counts)
        got = ops.add_adapters(base, x, a, b, plan).double().cpu()
        assert ((got - want).abs() <= tol).all()
        clean = ops.add_adapters(base, x, a, b, plan)
        x[7, 5], x[9, 100] = float("inf"), float("nan")
        got = ops.add_adapters(base, x, a, b, plan)
        others = [i for i in range(40) if i not in (7, 9)]
        assert torch.equal(got[others], clean[others])
        assert torch.isnan(got[9]).all() and not torch.isfinite(got[7]).any()
        u = x[7].double().cpu() @ a[0].double().cpu().t()
        plain = (u[None] * b[0].double().cpu()).sum(-1)
        assert torch.equal(torch.isnan(got[7]).cpu(), torch.isnan(plain)) and torch.equal(got[7].double().cpu()[~torch.isnan(plain)], plain[~torch.isnan(plain)])


def test_values_at_the_ends_of_the_types(dev):
    """u as large as fp32 holds and as small as counts, beside weights that bring it back into the type."""
    from kvmix_amd import ops

    big = torch.finfo(torch.bfloat16).max
    for xs, a_s, b_s in ((big / 2, 1.0, 1e-36), (2.0 ** 64, 2.0 ** 62, 2.0 ** -120), (2.0 ** -60, 2.0 ** -60, 2.0 ** 118), (2.0 ** -40, 1.0, 2.0 ** 100)):
        base, x, a, b, _ = _inputs(dev, [20], 1, 8, 8, 16, torch.bfloat16)
        x, a, b = torch.zeros_like(x), torch.zeros_like(a), b.sign() * b_s
        x[:, 0], a[0, :, 0] = xs, torch.linspace(0.5, 1, 8) * a_s
        b, base = b.bfloat16(), base * 0
        plan = ops.adapter_plan([0], [20], 1, dev)
        want, tol = _want(base, x, a, b, None, [0], [20])
        got = ops.add_adapters(base, x, a, b, plan).double().cpu()
        assert torch.isfinite(want).all() and ((got - want).abs() <= tol).all()
    base, x, a, b, _ = _inputs(dev, [20], 1, 8, 8, 16, torch.float16)
    plan = ops.adapter_plan([0], [20], 1, dev)
    for f in (2.0 ** -14, 2.0 ** -20):  # subnormal x and a: products down to 2^-48
        want, tol = _want(base * 0, (x * f).half(), (a * f).half(), b, None, [0], [20])
        got = ops.add_adapters(base * 0, (x * f).half(), (a * f).half(), b, plan).double().cpu()
        assert ((got - want).abs() <= tol).all()


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_results_beyond_the_caches(dev, dtype):
    """More than 32 MB of them, to the last columns and tokens: as in parts, and against 64 bits."""
    from kvmix_amd import ops

    counts, adapters, n = [700, 33, 1, 1400], [0, -1, 1, 0], 8200
    base, x, a, b, scales = _inputs(dev, counts, 2, 24, 72, n, dtype)
    plan = ops.adapter_plan(adapters, counts, 2, dev)
    out = ops.add_adapters(base, x, a, b, plan, scales)
    want, tol = _want(base, x, a, b, scales, adapters, counts)
    assert ((out.double().cpu() - want).abs() <= tol).all()
    for at in (0, 4096):
        part = slice(at, min(at + 4096, n))
        assert torch.equal(ops.add_adapters(base[:, part], x, a, b[:, part], plan, scales), out[:, part])
    assert torch.equal(ops.add_adapters(base, x, a, b, plan, scales, out=base), out)


def test_inputs_beyond_the_caches(dev):
    """More than 64 MB of x, of two adapters' tokens and of none's, against 64 bits."""
    from kvmix_amd import ops

    k, counts, adapters = 11016, [2900, 17, 260], [1, -1, 0]
    g = torch.Generator(device=dev).manual_seed(3)
    x = torch.randn(3177, k, generator=g, device=dev).half()
    a, b = (torch.randn(2, 40, k, generator=g, device=dev) * k ** -0.5).half(), torch.randn(2, 48, 40, generator=g, device=dev).half()
    base = torch.randn(3177, 48, generator=g, device=dev).half()
    out = ops.add_adapters(base, x, a, b, ops.adapter_plan(adapters, counts, 2, dev))
    for at in range(0, 3177, 353):  # (in 64 bits, some rows at a time)
        i = torch.tensor([1 if t < 2900 else 0 for t in range(at, at + 353)], device=dev)
        u = torch.stack([x[at:at + 353].double() @ a[j].double().t() for j in range(2)])[i, torch.arange(353, device=dev)]
        size = torch.stack([x[at:at + 353].double().abs() @ a[j].double().abs().t() for j in range(2)])[i, torch.arange(353, device=dev)]
        y = base[at:at + 353].double() + (u[:, None] * b[i].double()).sum(-1) * torch.tensor([0.0 if 2900 <= t < 2917 else 1.0 for t in range(at, at + 353)], device=dev)[:, None]
        off = k * 2.0 ** -24 * size + u.abs().amax(-1, keepdim=True) * 2.0 ** -22
        e = (off[:, None] * b[i].double().abs()).sum(-1) + 80 * 2.0 ** -24 * (u.abs()[:, None] * b[i].double().abs()).sum(-1)
        assert ((out[at:at + 353].double() - y).abs() <= e + 2.0 ** -11 * (y.abs() + e) + 2.0 ** -25 + 2.0 ** -23 * (y.abs() + base[at:at + 353].double().abs())).all()


def test_strides_and_shapes(dev):
    """Columns of a wider projection in place, three dimensions, weights that are views, rows that sixteen bytes do not fit."""
    from kvmix_amd import ops

    counts, adapters = [1, 20, 1], [1, 0, 1]
    base, x, a, b, scales = _inputs(dev, counts, 2, 16, 128, 64, torch.float16)
    plan = ops.adapter_plan(adapters, counts, 2, dev)
    want = ops.add_adapters(base, x, a, b, plan, scales)
    wide = torch.randn(22, 192, device=dev).half()
    kept = wide.clone()
    wide[:, 64:128] = base
    view = wide[:, 64:128]
    assert ops.add_adapters(view, x, a, b, plan, scales, out=view) is view and torch.equal(view, want)
    assert torch.equal(wide[:, :64], kept[:, :64]) and torch.equal(wide[:, 128:], kept[:, 128:])
    wide[:, :64] = base
    ops.add_adapters(wide[:, :64], x, a, b, plan, scales, out=wide[:, 128:])  # beside one another
    assert torch.equal(wide[:, 128:], want) and torch.equal(wide[:, :64], base)
    got = ops.add_adapters(base[:, None], x[:, None], a.transpose(1, 2).contiguous().transpose(1, 2), torch.cat([b, b], -1)[..., :16], plan, scales)
    assert torch.equal(got[:, 0], want)
    flat = torch.zeros(22 * 128 + 1, device=dev, dtype=torch.float16)
    flat[1:] = x.view(-1)
    assert torch.equal(ops.add_adapters(base, flat[1:].view(22, 128), a, b, plan, scales), want)
    row = torch.randn(64, device=dev).half()
    assert torch.equal(ops.add_adapters(row.expand(22, 64), x, a, b, plan), ops.add_adapters(row.repeat(22, 1), x, a, b, plan))


def test_refusals(dev):
    from kvmix_amd import ops

    counts = [1, 4]
    base, x, a, b, scales = _inputs(dev, counts, 3, 16, 128, 64, torch.float16)
    plan = ops.adapter_plan([2, -1], counts, 3, dev)
    same = torch.zeros(5, 128, device=dev).half()
    for args, kw, match in [
        ((base[:4], x, a, b, plan), {}, "same tokens"), ((base[:4], x[:4], a, b, plan), {}, "another number"), ((base, x.bfloat16(), a, b, plan), {}, "one type"),
        ((base.float(), x, a, b, plan), {}, "float16 or bfloat16"), ((base, x, a[:2], b[:2], plan), {}, "adapter's number"),
        ((base, x, a[:, :12].contiguous(), b[..., :12].contiguous(), plan), {}, "multiples of 8"), ((base, x, a, b[:2], plan), {}, "adapters must be"),
        ((base, x[:, :120], a, b, plan), {}, "adapters must be"), ((base, x, a, b, plan, scales[:2]), {}, "scales"), ((base, x, a, b, plan, scales.half()), {}, "scales"),
        ((base, x.cpu(), a, b, plan), {}, "device|cpu"), ((base, x, a, b, plan), {"out": torch.empty(5, 72, device=dev).half()}, "like base"),
        ((same[:, :64], x, a, b, plan), {"out": same[:, 8:72]}, "overlap"), ((base, same, a, b, plan), {"out": same[:, :64]}, "overlap"),
        ((base, x, a, b, plan), {"out": torch.empty(1, 64, device=dev).half().expand(5, 64)}, "rows"),
        ((base, x, a, b, plan), {"out": torch.empty(64, 5, device=dev).half().t()}, "rows"),
        ((base, x.clone().requires_grad_(), a, b, plan), {}, "no derivative"), ((base, x, a, b.clone().requires_grad_(), plan), {}, "no derivative"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            ops.add_adapters(*args, **kw)
    for args, match in [(([0], [1, 2], 1), "as many"), (([1], [1], 1), "adapter's number"), (([0], [-1], 1), "negative")]:
        with pytest.raises(RuntimeError, match=match):
            ops.adapter_plan(*args)
    with pytest.raises(RuntimeError, match="GPU"):
        ops.adapter_plan([0], [1], 1, "cpu")


def test_captured_and_on_another_stream(dev):
    from kvmix_amd import ops

    counts, adapters = [1] * 9 + [50], [0, 1, -1, 2, 2, 2, 0, 1, 1, 0]
    base, x, a, b, scales = _inputs(dev, counts, 3, 16, 1024, 256, torch.float16)
    plan = ops.adapter_plan(adapters, counts, 3, dev)
    want = ops.add_adapters(base, x, a, b, plan, scales)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = ops.add_adapters(base, x, a, b, plan, scales)
    side.synchronize()
    assert torch.equal(got, want)
    graphs = []
    for _ in range(2):  # two graphs with workspaces of their own
        graph, mine = torch.cuda.CUDAGraph(), x.clone()
        with torch.cuda.graph(graph):
            out = ops.add_adapters(base, mine, a, b, plan, scales)
        graphs.append((graph, mine, out))
    for i in range(3):
        for j, (graph, mine, out) in enumerate(graphs):
            mine.copy_(x * (i + j + 1))
            graph.replay()
        torch.cuda.synchronize()
        for j, (graph, mine, out) in enumerate(graphs):
            assert torch.equal(out, ops.add_adapters(base, x * (i + j + 1), a, b, plan, scales))
    with pytest.raises(RuntimeError, match="captured"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            ops.adapter_plan([0], [1], 1, dev)
