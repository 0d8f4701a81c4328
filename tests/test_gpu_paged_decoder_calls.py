"""The edges of PagedDecoder's calls."""
import pytest
import torch

from test_gpu_paged_cache import small

pytestmark = pytest.mark.gpu


@pytest.fixture
def model(dev):
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg, w = small(dev, 2)
    return PagedDecoder(cfg, w, [4] * 3, [4] * 3, page_size=32, window=32)


def test_one_token_and_none(dev, model):
    a = model.add()
    first = model.forward({a: torch.arange(20, device=dev)})[a].argmax().reshape(1)
    b = model.fork(a)
    two = first.expand(2)
    assert torch.equal(model.generate([a, b], two, 1), two[:, None])
    ids, lp, best = model.generate([a, b], two, 1, alternatives=3)
    assert torch.equal(ids, two[:, None]) and lp.shape == best.shape == (2, 0, 3)
    assert lp.dtype == torch.float32 and best.dtype == torch.int64 and lp.device == best.device == ids.device
    assert model.generate([a, b], two, 0).shape == (2, 0)
    assert model.cache.length(a) == 20                       # nothing was read
    ids, lp, best = model.generate([a, b], two, 2, alternatives=3)
    assert ids.shape == (2, 2) and lp.shape == best.shape == (2, 1, 3)
    assert model.generate([], first[:0], 3).shape == (0, 3)


def test_calls_that_are_refused(dev, model):
    a = model.add()
    model.forward({a: torch.arange(5, device=dev)})
    one = torch.zeros(1, dtype=torch.long, device=dev)
    for sequences, first, n in (([a], one, -1), ([a, a], one.expand(2), 3), ([a], one.expand(2), 3), ([a], one[:0], 3)):
        with pytest.raises(RuntimeError, match="generate"):
            model.generate(sequences, first, n)
    with pytest.raises(RuntimeError, match="no sequence"):
        model.generate([a + 7], one, 3)
    for chunk in (0, -3):
        with pytest.raises(RuntimeError, match="chunk"):
            model.score(torch.arange(9), chunk=chunk)
    assert model.cache.length(a) == 5 and len(model.cache._sequences) == 1
    assert model.score(torch.arange(0))[0].shape == (0,)
