"""ops.token_logprobs and its gradient against the formulas in 64 bits and against differences."""
import pytest
import torch

pytestmark = pytest.mark.gpu

KINDS = [torch.float16, torch.bfloat16, torch.float32]


def wanted(x, t):
    x = x.double()
    x = x - x.amax(-1, keepdim=True)  # (a sum of exponentials is lost beside a logit of 3e38, in 64 bits too)
    lp = x - torch.logsumexp(x, -1, keepdim=True)
    p = lp.exp()
    H = -torch.where(p > 0, p * lp, torch.zeros_like(p)).sum(-1)
    return lp.gather(-1, t.clamp(min=0)[..., None])[..., 0].masked_fill(t < 0, 0.0), H, lp


def best_of(x, n):
    """indexes of the n largest, equal ones by index"""
    order = torch.sort(x.double(), dim=-1, descending=True, stable=True).indices
    return order[..., :n]


def close(got, want, size):
    """Statistics in fp32: exponentials and sums of 1e5 terms are good to 2^-18 of the sum, a log probability takes a rounding of
    its own size on top (2^-22)."""
    got, want = got.cpu().double(), want.cpu()
    tol = 2.0 ** -17 * (1 + size) + 2.0 ** -22 * want.abs()
    same = got == want  # (two infinities)
    assert (((got - want).abs() <= tol) | same).all(), float(((got - want).abs() / tol).max())


def check(x, t, top):
    from kvmix_amd import ops

    out = ops.token_logprobs(x, t, top=top)
    lp, H, every = wanted(x, t)
    close(out[0], lp, 0)
    close(out[1], H, H.cpu().abs())
    if top:
        best = best_of(x, top)
        assert torch.equal(out[3], best)
        close(out[2], every.gather(-1, best), 0)


def logits(dev, rows, vocab, kind, seed=0, size=2.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = (torch.randn(rows, vocab, generator=g, device=dev) * size).to(kind)
    return x, torch.randint(0, vocab, (rows,), generator=g, device=dev)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab,top", [(1, 1, 1), (3, 2, 2), (5, 7, 3), (1, 64, 64), (2, 255, 20), (4, 257, 64), (600, 1000, 5), (1, 32000, 5), (7, 32001, 20),
                                            (513, 4099, 1), (2, 131071, 64), (700, 8192, 0), (1, 250007, 0)])
def test_against_64_bits(dev, kind, rows, vocab, top):
    check(*logits(dev, rows, vocab, kind, seed=vocab), top)


@pytest.mark.parametrize("kind", KINDS)
def test_strided_rows(dev, kind):
    x, t = logits(dev, 9, 1031, kind, seed=3)
    wide = torch.full((9, 1100), float("nan"), dtype=kind, device=dev)
    for shift in (0, 1, 3, 8):
        wide[:, shift:shift + 1031] = x
        check(wide[:, shift:shift + 1031], t, 7)
        wide.fill_(float("nan"))
    check(x.t().contiguous().t(), t, 7)
    check(x[::2], t[::2], 7)
    check(x.view(3, 3, 1031), t.view(3, 3), 7)
    check(x[:1].expand(9, 1031), t, 7)


@pytest.mark.parametrize("rows", [1, 600])
def test_equal_logits_come_by_index(dev, rows):
    from kvmix_amd import ops

    t = torch.zeros(rows, dtype=torch.long, device=dev)
    for vocab in (100, 5000, 40000):
        x = torch.full((rows, vocab), 0.25, dtype=torch.float16, device=dev)
        out = ops.token_logprobs(x, t, top=33)
        assert torch.equal(out[3], torch.arange(33, device=dev).expand(rows, 33))
        check(x, t, 33)
        x = (torch.arange(vocab, device=dev) % 3).half().expand(rows, vocab).contiguous()  # a third of the row is the largest
        check(x, t, 33)
        x[:, vocab // 2] = 9.0
        x[:, 1], x[:, 2] = 0.0, -0.0
        check(x, t, 33)


@pytest.mark.parametrize("kind", KINDS)
def test_masked_tokens(dev, kind):
    """-inf and the type's lowest value in masked places."""
    for fill in (float("-inf"), torch.finfo(kind).min):
        for rows, vocab in ((3, 3000), (600, 1025)):
            x, t = logits(dev, rows, vocab, kind, seed=11)
            keep = torch.rand(rows, vocab, device=dev) < 0.01
            keep.scatter_(1, t[:, None], True)
            x = x.masked_fill(~keep, fill)
            check(x, t, 4)
    x, t = logits(dev, 4, 5000, kind, seed=12)
    x[:, :4096] = float("-inf")        # whole pieces of a row
    check(x, t.clamp(min=4096), 3)
    x = torch.full((2, 700), torch.finfo(kind).min, dtype=kind, device=dev)   # a row of them only: all alike
    check(x, t[:2] % 700, 5)


@pytest.mark.parametrize("rows", [2, 600])
def test_rows_that_have_no_likelihood(dev, rows):
    from kvmix_amd import ops

    for bad in (float("nan"), float("inf")):
        x, t = logits(dev, rows, 5001, torch.float32, seed=13)
        x[1, 4000] = bad
        lp, H, top_lp, top_id = ops.token_logprobs(x, t, top=3)
        assert lp[1].isnan() and H[1].isnan() and top_id[1, 0] == 4000
        assert torch.isfinite(lp[0]) and torch.isfinite(H[0]) and torch.isfinite(top_lp[0]).all()
    x[1] = float("-inf")
    lp, H, _, top_id = ops.token_logprobs(x, t, top=3)
    assert lp[1].isnan() and H[1].isnan() and top_id[1].tolist() == [0, 1, 2]


def test_targets_that_are_none(dev):
    from kvmix_amd import ops

    x, t = logits(dev, 5, 900, torch.float16, seed=14)
    t[1], t[3] = -100, 900
    lp, H = ops.token_logprobs(x, t)
    want = wanted(x, t.clamp(max=899))
    assert lp[1] == 0 and lp[3].isnan()
    close(lp[[0, 2, 4]], want[0][[0, 2, 4]], 0)
    close(H, want[1], want[1].cpu())


@pytest.mark.parametrize("offset", [1e4, -3e4])
def test_logits_far_from_zero_lose_nothing(dev, offset):
    x, t = logits(dev, 3, 7000, torch.float32, seed=15)
    check(x + offset, t, 5)


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab", [(1, 1), (3, 33), (5, 1031), (2, 32000), (40, 20001)])
def test_gradient_against_the_formula(dev, kind, rows, vocab):
    from kvmix_amd import ops

    x, t = logits(dev, rows, vocab, kind, seed=vocab + 1)
    if rows > 2:
        t[1] = -1
    x.requires_grad_()
    a, b = torch.randn(rows, device=dev), torch.randn(rows, device=dev)
    lp, H = ops.token_logprobs(x, t)
    for ga, gb in ((a, b), (a, None), (None, b)):
        outs, grads = zip(*[(o, g) for o, g in ((lp, ga), (H, gb)) if g is not None])
        (got,) = torch.autograd.grad(outs, x, grads, retain_graph=True)
        _, h, logp = wanted(x.detach(), t)
        p = logp.exp()
        hit = (torch.arange(vocab, device=dev) == t[:, None]).double()
        da, db = (torch.zeros(rows, device=dev, dtype=torch.float64) if g is None else g.double() for g in (ga, gb))
        da = da.masked_fill(t < 0, 0.0)
        want = da[:, None] * (hit - p) - db[:, None] * p * (logp + h[:, None])
        # probabilities are good to 2^-17, log probability plus entropy to 2^-16 of what it is; the result rounds to its type
        size = p * (da.abs()[:, None] + db.abs()[:, None] * (1 + logp.abs() + h.abs()[:, None])) + da.abs()[:, None] * hit
        tol = 2.0 ** -15 * size + torch.finfo(kind).eps / 2 * want.abs() + (2.0 ** -25 if kind == torch.float16 else 0.0)
        assert got.dtype == kind and got.shape == x.shape
        assert ((got.double() - want).abs() <= tol).all(), float(((got.double() - want).abs() / tol).max())


def test_gradient_against_differences(dev):
    from kvmix_amd import ops

    x, t = logits(dev, 4, 50, torch.float32, seed=20, size=1.0)
    a, b = torch.randn(4, device=dev), torch.randn(4, device=dev)
    x.requires_grad_()
    lp, H = ops.token_logprobs(x, t)
    (got,) = torch.autograd.grad((a * lp + b * H).sum(), x)

    def value(y):
        l, h, _ = wanted(y, t)
        return (a.double() * l + b.double() * h).sum(-1)

    base, eps = x.detach().double(), 1e-5
    for i in range(50):
        up, down = base.clone(), base.clone()
        up[:, i] += eps
        down[:, i] -= eps
        for r in range(4):
            diff = (a[r].double() * (wanted(up, t)[0][r] - wanted(down, t)[0][r]) + b[r].double() * (wanted(up, t)[1][r] - wanted(down, t)[1][r])) / (2 * eps)
            assert abs(float(diff) - float(got[r, i])) < 1e-4
    assert torch.isfinite(value(base))


def test_gradient_of_masked_rows_and_views(dev):
    from kvmix_amd import ops

    x, t = logits(dev, 6, 777, torch.float32, seed=21)
    dead = torch.rand(6, 777, device=dev) < 0.5
    dead.scatter_(1, t[:, None], False)
    leaf = x.clone().requires_grad_()
    lp, H = ops.token_logprobs(leaf.masked_fill(dead, float("-inf")), t)
    (lp.sum() + 0.5 * H.sum()).backward()
    assert torch.isfinite(leaf.grad).all() and (leaf.grad[dead] == 0).all()
    shared = x[:1].clone().requires_grad_()          # one row for several targets: its gradient is the sum
    lp, _ = ops.token_logprobs(shared.expand(6, 777), t)
    lp.sum().backward()
    p = torch.softmax(x[:1].double(), -1)
    want = -6 * p
    want.scatter_add_(1, t[None], torch.ones(1, 6, device=dev, dtype=torch.float64))
    assert torch.allclose(shared.grad.double(), want, atol=1e-5)
    twice = x.clone().requires_grad_()
    lp, _, top_lp, top_id = ops.token_logprobs(twice.view(2, 3, 777), t.view(2, 3), top=2)
    assert not top_lp.requires_grad and lp.shape == (2, 3) and top_id.shape == (2, 3, 2)
    lp.sum().backward()
    assert twice.grad.shape == (6, 777)


def test_refusals(dev):
    from kvmix_amd import ops

    x, t = logits(dev, 4, 100, torch.float32)
    for args, what in (((x.cpu(), t), "GPU only"), ((x, t.cpu()), "expected all tensors"), ((x.double(), t), "float16, bfloat16 or float32"),
                       ((x, t.int()), "int64"), ((x, t[:3]), "shape of the logits"), ((x[:, :0], t), "must not be empty")):
        with pytest.raises(RuntimeError, match=what):
            ops.token_logprobs(*args)
    for top in (-1, 65, 101):
        with pytest.raises(RuntimeError, match="top must be"):
            ops.token_logprobs(x, t, top=top)
    lp, H = ops.token_logprobs(x[:0], t[:0])
    assert lp.shape == (0,) and H.shape == (0,)


def test_another_stream_and_a_graph(dev):
    from kvmix_amd import ops

    for rows, vocab in ((2, 32000), (600, 3000)):
        x, t = logits(dev, rows, vocab, torch.float16, seed=30)
        want = ops.token_logprobs(x, t, top=5)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = ops.token_logprobs(x, t, top=5)
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = ops.token_logprobs(x, t, top=5)
        for i in range(3):
            x.add_(0.5 * torch.randn_like(x))
            graph.replay()
            replayed = [o.clone() for o in out]
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(replayed, ops.token_logprobs(x, t, top=5)))
