"""ops.token_logprobs where its sizes and values have their edges."""
import pytest
import torch

from test_gpu_token_logprobs import logits

pytestmark = pytest.mark.gpu


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
