"""Beam searches and batch operators as the documents allow them beside the usual: caches that grow by concatenation, the reference's flush
rule, prompts of one token, nothing at all."""
import pytest
import torch

from test_gpu_beam_search import off_by
from test_gpu_paged_cache import small

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("graph", [False, True])
@pytest.mark.parametrize("Q", [1, 45])
def test_the_ratio_rule(dev, graph, Q):
    """Tails that flush every few tokens, in layers of different widths: the caches end with every beam's tokens, and scores are likelihoods
    (of four bits per value, as a paged cache holds them: within what other splits of a prompt are held to)."""
    from kvmix_amd.decoder import Decoder, GraphDecoder, kvmix_layers
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg, w = small(dev, 2)
    prompt = torch.randint(0, cfg.vocab_size, (2, Q), generator=torch.Generator().manual_seed(3)).to(dev)
    model = (GraphDecoder if graph else Decoder)(cfg, w, *kvmix_layers(cfg, [4] * 3, [4] * 3, residual_length=None, capacity=64))
    ids, scores = model.beam_search(prompt, 3, 40)
    # (of 40 tokens 12 stay in fp16, the 28 others are less than a group of 32)
    assert ids.shape == (2, 3, 40) and all(c.kv_seq_len == Q + 39 and (c.k_tokens > 0) == (Q > 1) for c in model.caches)
    exact = PagedDecoder(cfg, w, [4] * 3, [4] * 3, window=4096)
    for r in range(2):
        assert len({tuple(b) for b in ids[r].tolist()}) == 3
        lp, tol = off_by(exact, prompt[r], ids[r])
        assert float((lp - scores[r].double()).abs().max()) <= tol


def test_caches_that_grow_by_concatenation(dev):
    """The reference's tuples instead of caches in place: the same search, bit for bit."""
    from kvmix_amd.decoder import Decoder, kvmix_layers

    cfg, w = small(dev, 2)
    prompt = torch.randint(0, cfg.vocab_size, (2, 70), generator=torch.Generator().manual_seed(3)).to(dev)
    attention, caches = kvmix_layers(cfg, [4, 2, 1], [4, 2, 1], residual_length=40, capacity=64)
    want = Decoder(cfg, w, attention, caches).beam_search(prompt, 4, 30, 5)
    got = Decoder(cfg, w, kvmix_layers(cfg, [4, 2, 1], [4, 2, 1], residual_length=40)[0]).beam_search(prompt, 4, 30, 5)
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_no_tokens(dev):
    from kvmix_amd import ops

    g = torch.Generator().manual_seed(1)
    a, b = torch.randn(2, 8, 64, generator=g).half().to(dev), torch.randn(2, 40, 8, generator=g).half().to(dev)
    for plan in (ops.adapter_plan([], [], 2, dev), ops.adapter_plan([1, -1], [0, 0], 2, dev), ops.adapter_plan([], [], 0, dev)):
        assert plan.tokens == 0
        for shape in ((0,), (0, 1), (3, 0)):
            base, x = torch.zeros(*shape, 40, device=dev).half(), torch.zeros(*shape, 64, device=dev).half()
            assert ops.add_adapters(base, x, a, b, plan).shape == base.shape and ops.add_adapters(base, x, a, b, plan, out=base) is base
    rows = torch.zeros(2, 2, 2, 32, 64, device=dev).half()
    plan = ops.paged_plan(torch.tensor([[0], [1]], dtype=torch.int32), [5, 0], [0, 0], [0, 0], 4, 2, 64, 32, dev)
    table = torch.zeros(0, 64, device=dev)
    assert ops.paged_rope_append(torch.zeros(0, 8, 64, device=dev).half(), table, table, rows, plan).shape == (0, 4, 64)
    assert not rows.any()
