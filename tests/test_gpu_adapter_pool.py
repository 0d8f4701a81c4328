"""Sequences with adapters of their own in one batch, beside sequences without: the decoder against merged weights, and the pool's calls."""
import pytest
import torch

from test_gpu_paged_cache import small

pytestmark = pytest.mark.gpu


def adapters(cfg, rank, targets, seed, dev):
    g = torch.Generator().manual_seed(seed)
    h, i = cfg.hidden_size, cfg.intermediate_size
    shapes = {"wqkv": ((cfg.num_heads + 2 * cfg.num_kv_heads) * cfg.head_dim, h), "wo": (h, h), "w_gate_up": (2 * i, h), "w_down": (h, i)}
    return {(layer, t): ((torch.randn(rank, shapes[t][1], generator=g) * shapes[t][1] ** -0.5).half().to(dev),
                         (torch.randn(shapes[t][0], rank, generator=g) * 0.3).half().to(dev))
            for layer in range(cfg.num_layers) for t in targets}


def merged(w, weights, scale):
    out = dict(w)
    out["layers"] = [dict(lw) for lw in w["layers"]]
    for (layer, t), (a, b) in weights.items():
        old = w["layers"][layer][t]
        out["layers"][layer][t] = (old.float() + scale * b.float() @ a.float()).to(old.dtype)
    return out


def test_against_merged_weights(dev):
    """Chunks and single tokens of sequences with two adapters and without one in the same steps; forks keep their adapter."""
    from kvmix_amd.adapters import TARGETS, AdapterPool
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg, w = small(dev, 2)
    pool = AdapterPool(cfg, 3, 24, device=dev)
    sets = [(0, adapters(cfg, 24, TARGETS, 1, dev), 0.02), (2, adapters(cfg, 5, ("wqkv", "w_down"), 2, dev), -0.05)]
    for i, weights, scale in sets:
        pool.load(i, weights, scale)
    bits = ([4] * 3, [4] * 3)
    model = PagedDecoder(cfg, w, *bits, window=4096, adapters=pool)
    plain = {None: PagedDecoder(cfg, w, *bits, window=4096)}
    plain.update({i: PagedDecoder(cfg, merged(w, weights, scale), *bits, window=4096) for i, weights, scale in sets})
    plain[1] = plain[None]  # an adapter that was never loaded
    of = [None, 0, 2, 1, 0]
    seqs, alone = [model.add(i) for i in of], [plain[i].add() for i in of]
    g = torch.Generator().manual_seed(4)

    def step(counts):
        ids = [torch.randint(0, cfg.vocab_size, (n,), generator=g).to(dev) for n in counts]
        got = model.forward({s: x for s, x in zip(seqs, ids) if x.numel()})
        for s, t, i, x in zip(seqs, alone, of, ids):
            if not x.numel():
                continue
            want = plain[i].forward({t: x})[t]
            # (other splits of a step round elsewhere in fp16; what the adapters do is far more)
            assert float((got[s] - want).abs().max()) < 0.05 * float(want.std()), (i, counts)
        return got

    step([70, 5, 33, 1, 100])
    step([1, 1, 1, 1, 1])
    step([0, 64, 1, 0, 7])
    last = step([1, 1, 1, 2, 1])
    sizes = [float((last[seqs[1]] - last[seqs[0]]).std()), float(last[seqs[0]].std())]
    assert sizes[0] > 0.2 * sizes[1]  # (they are no small change)
    twin = model.fork(seqs[1])
    x = torch.tensor([5], device=dev)
    assert torch.allclose(model.forward({twin: x})[twin], model.forward({seqs[1]: x})[seqs[1]], rtol=0, atol=0.05 * sizes[1])
    two = model.fork(seqs[2], 2)
    assert [model._adapter_of.get(s) for s in (twin, *two)] == [0, 2, 2]
    for s in (twin, *two, *seqs):
        model.free(s)
    assert not model._adapter_of


def test_a_server_with_all_of_it(dev):
    """Chunked prompts of sequences with adapters, answers, beams from an adapter's sequence, likelihoods; pages come back."""
    from kvmix_amd.adapters import AdapterPool
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg, w = small(dev, 2)
    pool = AdapterPool(cfg, 2, 8, targets=("wo", "w_gate_up"), device=dev)
    pool.load(1, adapters(cfg, 8, ("wo", "w_gate_up"), 3, dev), 0.1)
    model = PagedDecoder(cfg, w, [4, 2, 3], [2, 4, 4], page_size=32, window=32, adapters=pool)
    free = model.cache.free_pages()
    a, b = model.add(), model.add(adapter=1)
    prompt = torch.randint(0, cfg.vocab_size, (150,), generator=torch.Generator().manual_seed(1)).to(dev)
    for at in range(0, 150, 64):
        last = model.forward({s: prompt[at:at + 64] for s in (a, b)})
    logits = torch.stack([last[a], last[b]])
    ids, scores = model.beam_search([a, b], logits, 3, 6)
    assert torch.isfinite(scores).all() and not torch.equal(ids[0], ids[1])
    # b's beams were b's adapter's: their scores are the likelihoods under it
    for r, s in enumerate((a, b)):
        twin = model.fork(s)
        after = torch.cat([logits[r][None], model.forward({twin: ids[r, 0, :-1]}, every=True)[twin]])
        lp = torch.log_softmax(after.double(), -1).gather(-1, ids[r, 0][:, None]).sum()
        # (six tokens; packed pages are read by other kernels in a chunk, where packed keys are fp16 numbers)
        assert abs(float(lp - scores[r, 0].double())) <= 6 * 2 * 0.05 * float(after.std())
        model.free(twin)
    out = model.generate([a, b], logits.argmax(-1), 40)
    assert out.shape == (2, 40)
    model.free(a)
    model.free(b)
    assert model.cache.free_pages() == free and not model._adapter_of


def test_the_pool(dev):
    from kvmix_amd.adapters import AdapterPool
    from kvmix_amd.paged_decoder import PagedDecoder
    from kvmix_amd import ops

    cfg, w = small(dev, 2)
    pool = AdapterPool(cfg, 2, 16, targets=("wo",), device=dev)
    first = adapters(cfg, 16, ("wo",), 1, dev)
    pool.load(1, first, 2.0)
    less = {(0, "wo"): tuple(t[:3] if j == 0 else t[:, :3] for j, t in enumerate(first[0, "wo"]))}
    base, x = torch.randn(4, 512, device=dev).half(), torch.randn(4, 512, device=dev).half()
    plan = ops.adapter_plan([1, -1], [3, 1], 2, dev)
    a, b = first[0, "wo"]

    def check(add):
        want = base.double()
        want[:3] += add
        got = pool.add(base.clone(), x, 0, "wo", plan)
        # three roundings to fp16 at most beside fp32 sums of 512 terms (below 2^-9 of their absolute sum)
        assert torch.allclose(got.double(), want, rtol=2.0 ** -10, atol=2.0 ** -8)
        return got

    check(2.0 * x[:3].double() @ a.double().t() @ b.double().t())
    pool.load(1, less, 0.5)  # what was there before is gone
    check(0.5 * x[:3].double() @ a[:3].double().t() @ b[:, :3].double().t())
    assert torch.equal(pool.add(base.clone(), x, 1, "wo", plan), base)  # (zero in the other layers)
    assert pool.add(base, x, 0, "wqkv", plan) is base
    for call in (lambda: AdapterPool(cfg, 0, 16), lambda: AdapterPool(cfg, 1, 12), lambda: AdapterPool(cfg, 1, 136), lambda: AdapterPool(cfg, 1, 8, targets=()),
                 lambda: AdapterPool(cfg, 1, 8, targets=("embed",)), lambda: pool.load(2, first), lambda: pool.load(-1, first), lambda: pool.load(0, {(0, "wqkv"): first[0, "wo"]}),
                 lambda: pool.load(0, {(7, "wo"): first[0, "wo"]}), lambda: pool.load(0, {(0, "wo"): (a, b.t()[:, :5])}), lambda: pool.load(0, {(0, "wo"): (a[:8], b)}),
                 lambda: pool.load(0, adapters(cfg, 24, ("wo",), 1, dev))):
        with pytest.raises(RuntimeError):
            call()
    model = PagedDecoder(cfg, w, [4] * 3, [4] * 3, adapters=pool)
    for i in (2, -1):
        with pytest.raises(RuntimeError, match="no adapter"):
            model.add(adapter=i)
    with pytest.raises(RuntimeError, match="no adapter"):
        PagedDecoder(cfg, w, [4] * 3, [4] * 3).add(adapter=0)
