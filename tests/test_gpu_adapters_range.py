"""Adapters in bf16 whose products reach both ends of the type: whatever is finite in the formula is finite, and as near to it as anywhere."""
import pytest
import torch

from test_gpu_adapters import _want

pytestmark = pytest.mark.gpu

MOST = float(torch.finfo(torch.bfloat16).max)  # (2 - 2^-7) 2^127


@pytest.mark.parametrize("tokens", [1, 20, 40])
@pytest.mark.parametrize("rank", [8, 128])
@pytest.mark.parametrize("x0,a0,b0", [
    (2.0 ** -30, 1.9 * 2.0 ** -30, MOST),                 # u of about 2^-60: times the largest weight far inside of the type
    (2.0 ** -4, 2.0 ** -4, MOST / 2),                     # u up to 2^-8, sums of up to 2^126
    (2.0 ** -5, 1.9 * 2.0 ** -4, MOST / 2),
    (2.0 ** -40, 2.0 ** -40, MOST),
    (2.0 ** -60, 2.0 ** -56, MOST),                       # below where u is kept
    (1.0, 1.0, MOST / 256),
    (2.0 ** 63, 1.99 * 2.0 ** 63, 2.0 ** -125),           # u up to 2^127
    (MOST, 1.0, 2.0 ** -60),
    (2.0 ** 50, 2.0 ** 50, 2.0 ** -120),
    (1.0, 2.0 ** -7, 2.0 ** -119),                        # results of 2^-126 and less
    (1.0, 2.0 ** -3, 2.0 ** -125),
    (2.0 ** -10, 2.0 ** -10, 2.0 ** -104),
])
def test_products_at_both_ends(dev, tokens, rank, x0, a0, b0):
    from kvmix_amd import ops

    g = torch.Generator().manual_seed(rank)
    x, a = torch.zeros(tokens, 16), torch.zeros(1, rank, 16)
    x[:, 3], a[0, :, 3] = x0 * torch.linspace(0.5, 1, tokens), a0 * torch.linspace(0.5, 1, rank)
    # (signs that leave less than half of the sum's terms over: partial sums stay inside of the type as well)
    b = b0 * (0.5 + 0.5 * torch.rand(1, 24, rank, generator=g, dtype=torch.float64)) * (1 - 2 * (torch.arange(rank) % 2)).double()
    base, x, a, b = torch.zeros(tokens, 24, dtype=torch.bfloat16, device=dev), x.bfloat16().to(dev), a.bfloat16().to(dev), b.bfloat16().to(dev)
    assert torch.isfinite(b).all() and torch.isfinite(a).all()
    want, tol = _want(base, x, a, b, None, [0], [tokens])
    assert (want.abs() < MOST / 2).all()
    got = ops.add_adapters(base, x, a, b, ops.adapter_plan([0], [tokens], 1, dev)).double().cpu()
    assert ((got - want).abs() <= tol).all(), (got, want)
