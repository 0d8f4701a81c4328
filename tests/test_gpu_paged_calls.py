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
