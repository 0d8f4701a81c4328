"""What the paged operators and the likelihoods promise beside their results: calls that they refuse, streams, numbers of pages."""
import pytest
import torch

from paged_helpers import Batch

pytestmark = pytest.mark.gpu


def test_derivatives_are_refused_where_there_are_none(dev):
    """No call gives a result from which a derivative of its inputs is missing without a word."""
    import torch.autograd.forward_ad as fwd

    from kvmix_amd import ops

    b = Batch(dev, [100, 64], [64, 0], [1, 1], 4, 2, 128, 64, 4, 4)
    kv = torch.randn(2, 2, 128, dtype=torch.float16, device=dev)
    rows = torch.zeros_like(b.rows)
    calls = [("paged_attention", b.q, lambda t: ops.paged_attention(t, b.rows, b.packed, b.plan, 4, 4)),
             ("paged_attention", b.rows, lambda t: ops.paged_attention(b.q, t, b.packed, b.plan, 4, 4)),
             ("paged_append", kv, lambda t: ops.paged_append(t, kv, rows, b.plan)),
             ("paged_append", kv, lambda t: ops.paged_append(kv, t, rows, b.plan)),
             ("paged_quantize", b.rows, lambda t: ops.paged_quantize(t, b.packed.clone(), torch.tensor([[0, 0]]), 4, 4)),
             ("paged_read", b.rows, lambda t: ops.paged_read(t, torch.tensor([0]))),
             ("paged_copy", rows, lambda t: ops.paged_copy([t], torch.tensor([[0, 1]])))]
    for name, x, call in calls:
        call(x)
        leaf = x.clone().requires_grad_()
        with pytest.raises(RuntimeError, match=name + ".*no derivative"):
            call(leaf)
        with torch.no_grad():
            call(leaf)
        with fwd.dual_level():
            with pytest.raises(RuntimeError, match=name + ".*no derivative"):
                call(fwd.make_dual(x.clone(), torch.ones_like(x)))
            call(x)
    x, t = torch.randn(3, 50, device=dev), torch.tensor([1, 2, 3], device=dev)
    with fwd.dual_level():
        for y in (x, x.clone().requires_grad_()):
            with pytest.raises((RuntimeError, NotImplementedError)):
                ops.token_logprobs(fwd.make_dual(y, torch.ones_like(x)), t)
        assert torch.isfinite(ops.token_logprobs(x, t)[0]).all()


def test_a_trace_is_refused(dev):
    """A trace would keep the results of its example as constants."""
    from kvmix_amd import ops

    x, t = torch.randn(3, 50, device=dev), torch.tensor([1, 2, 3], device=dev)
    b = Batch(dev, [64], [0], [1], 4, 2, 128, 64, 4, 4)
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda y: ops.token_logprobs(y, t)[0], (x,), check_trace=False)
    with pytest.raises(RuntimeError, match="trace"):
        torch.jit.trace(lambda q: ops.paged_attention(q, b.rows, b.packed, b.plan, 4, 4), (b.q,), check_trace=False)


def test_a_function_mode_is_no_derivative(dev):
    from kvmix_amd import ops

    x, t = torch.randn(3, 50, device=dev), torch.tensor([1, 2, 3], device=dev)
    want = ops.token_logprobs(x, t)
    with torch.device(dev), torch.autocast("cuda"):
        for a, b in zip(ops.token_logprobs(x, t), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("far", [1 << 32, (1 << 32) + 1, -(1 << 32), 1 << 31, (1 << 63) - 1, -(1 << 63) + 1])
def test_page_numbers_that_are_none(dev, far):
    """64-bit numbers beyond 32 bits are no pages, whatever their low bits are."""
    from kvmix_amd import ops

    rows = torch.zeros(4, 2, 2, 64, 128, dtype=torch.float16, device=dev)
    packed = torch.zeros(4, 2, 2 * 128 * 10, dtype=torch.int32, device=dev)
    for pair in ([far, 1], [1, far]):
        with pytest.raises(RuntimeError, match="page number"):
            ops.paged_quantize(rows, packed, torch.tensor([[0, 0], pair]), 4, 4)
        with pytest.raises(RuntimeError, match="page number"):
            ops.paged_copy([rows], torch.tensor([pair]))
    with pytest.raises(RuntimeError, match="page number"):
        ops.paged_read(rows, torch.tensor([0, far]))
    with pytest.raises(RuntimeError, match="page number"):
        ops.paged_plan(torch.tensor([[0, far]]), [100], [0], [1], 4, 2, 128, 64, dev)
    assert ops.paged_plan(torch.tensor([[0, far]]), [64], [0], [1], 4, 2, 128, 64, dev).tokens == 1  # (a cell that no token needs)


def test_a_plan_made_on_another_stream(dev):
    """A plan can be used on any stream: its list is waited for, and not given to others while it is read."""
    from kvmix_amd import ops

    b = Batch(dev, [700, 60, 300], [512, 0, 128], [1, 40, 3], 8, 2, 128, 64, 4, 4, seed=3)
    kv = torch.randn(44, 2, 128, dtype=torch.float16, device=dev)
    want_rows = b.rows.clone()
    ops.paged_append(kv, kv, want_rows, b.plan)
    want = ops.paged_attention(b.q, want_rows, b.packed, b.plan, 4, 4)
    rows, other_rows = b.rows.clone(), b.rows.clone()
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    # made behind other work, used at once
    torch.cuda._sleep(200_000_000)
    plan = ops.paged_plan(b.table, b.lens, b.packed_lens, b.new, 8, 2, 128, 64, dev)
    with torch.cuda.stream(side):
        ops.paged_append(kv, kv, rows, plan)
        got = ops.paged_attention(b.q, rows, b.packed, plan, 4, 4)
    side.synchronize()
    assert torch.equal(got, want)
    # dropped while it is still to be read
    with torch.cuda.stream(side):
        torch.cuda._sleep(200_000_000)
        ops.paged_append(kv, kv, other_rows, plan)
        got = ops.paged_attention(b.q, other_rows, b.packed, plan, 4, 4)
    words = plan.slots.untyped_storage().nbytes() // 4
    del plan
    others = [torch.zeros(words, dtype=torch.int32, device=dev) for _ in range(4)]
    torch.cuda.synchronize()
    assert torch.equal(got, want) and not any(t.any() for t in others)


def test_plans_are_made_outside_of_captures(dev):
    from kvmix_amd import ops

    table = torch.tensor([[0, 1]])
    x = torch.zeros(4, device=dev)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x += 1
        with pytest.raises(RuntimeError, match="captured"):
            ops.paged_plan(table, [100], [0], [1], 4, 2, 128, 64, dev)
    graph.replay()
    assert ops.paged_plan(table, [100], [0], [1], 4, 2, 128, 64, dev).tokens == 1 and float(x[0]) == 1.0


def test_steps_are_taken_outside_of_captures(dev):
    """A step that is refused leaves the cache as it was."""
    from kvmix_amd.paged import PagedKVCache

    c = PagedKVCache([4], [4], 4, 2, 64, row_pages=16, packed_pages=16, page_size=32, window=32)
    a = c.new()
    step = c.step({a: 200})
    kv = torch.randn(200, 2, 64, dtype=torch.float16, device=dev)
    c.append(0, step, kv, kv)
    q = torch.randn(200, 4, 64, dtype=torch.float16, device=dev)
    want, state = c.attend(0, step, q), (c.length(a), c.free_pages())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        q += 0
        with pytest.raises(RuntimeError, match="captured"):
            c.step({a: 3})
    assert (c.length(a), c.free_pages()) == state
    assert torch.equal(c.attend(0, step, q), want)
