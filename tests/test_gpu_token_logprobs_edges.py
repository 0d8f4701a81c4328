"""ops.token_logprobs where its sizes and values have their edges."""
import pytest
import torch

from test_gpu_token_logprobs import KINDS, best_of, check, close, logits, wanted

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("vocab", [65528, 65529, 65532, 65533, 131053, 131057, 131061, 131063, 131064, 131065, 196585, 196595, 262113])
def test_ends_of_chunks(dev, kind, vocab):
    """Vocabularies of nearly as many values as whole blocks hold: the largest logit and the target among the last values that
    a block takes, in rows of every alignment."""
    x, t = logits(dev, 5, vocab, kind, seed=vocab)
    for at in (65533, 65534, 65535, 131071, vocab - 1):
        if at < vocab:
            y = x.clone()
            y[:, at] = 30.0
            check(y, torch.full_like(t, at), 3)
    wide = torch.zeros(3, vocab + 4, dtype=kind, device=dev)
    wide[:, 1:1 + vocab] = x[:3]
    check(wide[:, 1:1 + vocab], t[:3], 20)


@pytest.mark.parametrize("vocab", [131061, 196595])
def test_gradient_at_ends_of_chunks(dev, vocab):
    from kvmix_amd import ops

    x, t = logits(dev, 3, vocab, torch.float32, seed=1)
    t[:] = torch.tensor([65535, 65534, 65533])
    x.scatter_(1, t[:, None], 20.0)
    x.requires_grad_()
    lp, _ = ops.token_logprobs(x, t)
    lp.sum().backward()
    want = -torch.softmax(x.detach().double(), -1)
    want.scatter_add_(1, t[:, None], torch.ones(3, 1, device=dev, dtype=torch.float64))
    # (a probability is good to 2^-17, one minus it to that of one)
    assert ((x.grad.double() - want).abs() <= 2.0 ** -15).all()


@pytest.mark.parametrize("kind", KINDS)
@pytest.mark.parametrize("rows,vocab", [(5, 3001), (600, 3001), (5, 40007), (5, 196585), (5, 262144)])
def test_one_token_takes_nearly_all(dev, kind, rows, vocab):
    """Entropies near zero, with the largest logit anywhere in the row."""
    x, t = logits(dev, rows, vocab, kind, seed=vocab)
    for at in (0, 1500, 65533, 65534, 131071, vocab - 1):
        if at < vocab:
            for size in (17.0, 30.0):
                y = x.clone()
                y[:, at] = size
                check(y, torch.full_like(t, at), 3)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows", [4, 600])
@pytest.mark.parametrize("size", [1e4, 1e7, 3e8, 1e10, 1e20, 1e36])
def test_logits_of_any_size(dev, kind, rows, size):
    x, t = logits(dev, rows, 5001, kind, seed=50)
    check((x.float() * size).to(kind), t, 4)
    x = torch.full((rows, 3000), size, dtype=kind, device=dev)  # all alike but for a few
    x[:, ::7] = 0.0
    x[:, 1::7] = -size
    check(x, t % 3000, 4)


@pytest.mark.parametrize("kind", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("rows,vocab,most", [(2, 15000, 15.0), (600, 15000, 15.0), (2, 60000, 19.5)])
def test_a_huge_logit_behind_many_ordinary_ones(dev, kind, rows, vocab, most):
    """Ordinary logits that sum up to much, and then one beside which they are nothing."""
    x = torch.zeros(rows, vocab, dtype=kind, device=dev)
    x[:, 4096:] = most
    for at in (vocab - 1, vocab - 1000, 5000):
        for size in (1e30, 1e37, 3e38):
            y = x.clone()
            y[:, at] = size
            check(y, torch.full((rows,), at, device=dev), 2)
            check(y, torch.full((rows,), 7, device=dev), 0)


@pytest.mark.parametrize("kind", KINDS)
def test_large_gradients_of_masked_tokens(dev, kind):
    """Gradients of the entropy that are large: a token without probability gets exactly zero."""
    from kvmix_amd import ops

    x, t = logits(dev, 3, 5000, kind, seed=40)
    dead = torch.rand(3, 5000, device=dev) < 0.5
    dead.scatter_(1, t[:, None], False)
    x = x.masked_fill(dead, float("-inf")).requires_grad_()
    lp, H = ops.token_logprobs(x, t)
    for size in (1.0, 1e9, 1e30):
        (got,) = torch.autograd.grad((lp, H), x, (torch.full_like(lp, size), torch.full_like(H, size)), retain_graph=True)
        assert (got[dead] == 0).all() and not got.isnan().any()


def test_more_rows_than_a_launch_has_blocks(dev):
    """2^24 rows and a few: with 256 threads to a row more than a launch's 2^32."""
    from kvmix_amd import ops

    rows = (1 << 24) + 5
    x = (torch.arange(rows, device=dev)[:, None] % 11 * torch.tensor([0.5, 1.0, -0.25, 0.125], device=dev)).half().requires_grad_()
    t = torch.arange(rows, device=dev) % 4
    lp, H, top_lp, top_id = ops.token_logprobs(x, t, top=2)
    (got,) = torch.autograd.grad(lp.sum() + H.sum(), x)
    for part in (slice(0, 44), slice(rows // 2, rows // 2 + 44), slice(rows - 44, rows)):
        y = x.detach()[part]
        want, entropy, every = wanted(y, t[part])
        close(lp[part], want, 0)
        close(H[part], entropy, entropy.cpu().abs())
        best = best_of(y, 2)
        assert torch.equal(top_id[part], best)
        close(top_lp[part], every.gather(-1, best), 0)
        p = every.exp()
        hit = (torch.arange(4, device=dev) == t[part][:, None]).double()
        grad = hit - p - p * (every + entropy[:, None])
        # (as test_gradient_against_the_formula)
        size = p * (2 + every.abs() + entropy.abs()[:, None]) + hit
        assert ((got[part].double() - grad).abs() <= 2.0 ** -15 * size + 2.0 ** -11 * grad.abs() + 2.0 ** -25).all()
