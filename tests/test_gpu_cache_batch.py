"""A decoder that is used again after its caches held the beams of a search, or another batch."""
import pytest
import torch

from test_gpu_paged_cache import small

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
def test_generate_after_a_beam_search(dev, graph):
    """Reset, a decoder generates as a new one does, for the batch the beams were made of, for one prompt and for as many as there were beams."""
    from kvmix_amd.decoder import Decoder, GraphDecoder, kvmix_layers

    cfg, w = small(dev, 2)
    prompts = torch.randint(0, cfg.vocab_size, (6, 90), generator=torch.Generator().manual_seed(8)).to(dev)
    kind = GraphDecoder if graph else Decoder
    new = lambda: kind(cfg, w, *kvmix_layers(cfg, [4, 2, 3], [2, 4, 4], residual_length=40, capacity=64))
    used = new()
    for rows, beams, again in ((1, 3, 1), (2, 3, 2), (2, 3, 6), (2, 2, 1)):
        for search in (True, False):
            if search:
                got, want = (d.beam_search(prompts[:rows], beams, 6)[0] for d in (used, new()))
            else:
                got, want = (d.generate(prompts[:again], 9) for d in (used, new()))
                assert all(c.as_tuple()[1].shape[0] == again for c in used.caches)
            assert torch.equal(got, want)
            for c in used.caches:
                c.reset()
            used.position = 0


def test_tokens_of_another_batch(dev):
    """A cache that has tokens takes no more of another batch; what it has stays."""
    from kvmix_amd.cache import PackedKVCache

    cache = PackedKVCache(4, 2, residual_length=40)
    k, v = (torch.randn(3, 2, 100, 128, device=dev).half() for _ in range(2))
    cache.append(k, v, prompt=True)
    before = [t.clone() for t in cache.as_tuple() if torch.is_tensor(t)]
    for b in (1, 2, 6):
        with pytest.raises(RuntimeError, match="3 sequences"):
            cache.append(k[:1, :, :1].repeat(b, 1, 1, 1), v[:1, :, :1].repeat(b, 1, 1, 1))
    assert cache.kv_seq_len == 100 and all(torch.equal(a, b) for a, b in zip([t for t in cache.as_tuple() if torch.is_tensor(t)], before))
    cache.reset()
    cache.append(k[:1], v[:1], prompt=True)
    assert cache.as_tuple()[1].shape[0] == 1
    assert all(torch.equal(a, b[:1]) for a, b in zip([t for t in cache.as_tuple() if torch.is_tensor(t)], before))
