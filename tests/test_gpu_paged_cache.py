"""kvmix_amd.paged and kvmix_amd.paged_decoder: sequences that grow, fork, end and move, and a model over them."""
import random

import pytest
import torch

pytestmark = pytest.mark.gpu


def reference(q, k, v, new):
    """q [n, heads, D], k, v [T, kv_heads, D] in float64 -> [n, heads, D]"""
    T, H, D = k.shape
    G = q.shape[1] // H
    k, v = k.repeat_interleave(G, 1), v.repeat_interleave(G, 1)
    x = torch.einsum("nhd,thd->hnt", q, k) * D ** -0.5
    dead = torch.arange(T, device=q.device) > (T - new + torch.arange(new, device=q.device))[:, None]
    return torch.einsum("hnt,thd->nhd", torch.softmax(x.masked_fill(dead, float("-inf")), -1), v)


@pytest.mark.parametrize("page,window,bits", [(64, 128, [(4, 4), (2, 3)]), (32, 0, [(3, 2)]), (128, 70, [(4, 1), (1, 4)])])
def test_a_server_of_sequences(dev, page, window, bits):
    """Random growth, forks, ends and compactions; what every sequence reads back and attends to is what was put in."""
    from kvmix_amd.paged import OutOfPages, PagedKVCache

    rng = random.Random(page + window)
    g = torch.Generator(device=dev).manual_seed(3)
    H, nh, D, L = 2, 4, 128, len(bits)
    c = PagedKVCache([b[0] for b in bits], [b[1] for b in bits], nh, H, D, row_pages=4096 // page, packed_pages=8192 // page, page_size=page, window=window)
    truth = {}  # sequence -> per layer (k, v) as stored in fp16
    for turn in range(60):
        act = rng.random()
        if not truth or act < 0.2:
            s = c.new()
            truth[s] = [tuple(torch.zeros(0, H, D, dtype=torch.float16, device=dev) for _ in range(2)) for _ in range(L)]
        elif act < 0.3:
            s = rng.choice(list(truth))
            count = rng.choice([1, 2])
            made = c.fork(s, count)
            for t in [made] if count == 1 else made:
                truth[t] = list(truth[s])
        elif act < 0.38 and len(truth) > 1:
            s = rng.choice(list(truth))
            c.free(s)
            del truth[s]
        elif act < 0.45:
            c.compact()
        grow = {s: rng.choice([0, 1, 1, 1, 5, 70, 200]) for s in rng.sample(list(truth), rng.randint(1, min(4, len(truth))))}
        before = {s: c.length(s) for s in truth}
        try:
            step = c.step(grow)
        except OutOfPages:
            assert {s: c.length(s) for s in truth} == before
            victim = max(truth, key=lambda s: c.length(s))
            c.free(victim)
            del truth[victim]
            continue
        n = sum(grow.values())
        for layer in range(L):
            k, v = (torch.randn(n, H, D, generator=g, device=dev, dtype=torch.float16) for _ in range(2))
            q = torch.randn(n, nh, D, generator=g, device=dev, dtype=torch.float16)
            c.append(layer, step, k, v)
            out = c.attend(layer, step, q)
            for s, span in step.tokens().items():
                truth[s][layer] = tuple(torch.cat([a, b[span]]) for a, b in zip(truth[s][layer], (k, v)))
                if grow[s]:
                    rk, rv = c.read(layer, s)
                    want = reference(q[span].double(), rk.double(), rv.double(), grow[s])
                    assert torch.allclose(out[span].double(), want, rtol=4e-3, atol=4e-3)
    for s, layers in truth.items():
        assert c.length(s) == layers[0][0].shape[0]
        packed = len(c._sequences[s].packed) * page
        assert packed <= max(0, c.length(s) - window)
        for layer, (k, v) in enumerate(layers):
            rk, rv = c.read(layer, s)
            assert torch.equal(rk[packed:], k[packed:]) and torch.equal(rv[packed:], v[packed:])
            for got, want, b in ((rk, k, bits[layer][0]), (rv, v, bits[layer][1])):
                if packed:  # codes: half a step of the group's range (at most 12 sigma), and the roundings to fp16
                    assert float((got[:packed] - want[:packed]).abs().max()) < 0.5 * 12 / (2 ** b - 1) + 0.02
    for s in list(truth):
        c.free(s)
    assert c.free_pages() == (4096 // page, 8192 // page)


def test_forks_share_and_diverge(dev):
    from kvmix_amd.paged import PagedKVCache

    c = PagedKVCache([4], [4], 2, 2, 64, row_pages=16, packed_pages=16, page_size=64, window=64)

    def put(s, n, value):
        step = c.step({s: n})
        x = torch.full((n, 2, 64), value, dtype=torch.float16, device=dev)
        c.append(0, step, x, x)

    a = c.new()
    put(a, 300, 1.0)
    put(a, 20, 2.0)          # 320 tokens: five full pages, three of them packed by now
    assert c.free_pages() == (14, 13)
    b, d = c.fork(a, 2)      # nothing to copy
    assert c.free_pages() == (14, 13)
    put(b, 1, 3.0)
    e = c.fork(b)
    put(d, 2, 4.0)
    put(e, 1, 5.0)
    values = {s: c.read(0, s)[0][:, 0, 0].tolist() for s in (a, b, d, e)}
    start = [1.0] * 300 + [2.0] * 20
    assert values == {a: start, b: start + [3.0], d: start + [4.0] * 2, e: start + [3.0, 5.0]}
    for s in (a, b, d):
        c.free(s)
    moved = c.compact()
    assert moved > 0 and c.read(0, e)[1][:, 1, 63].tolist() == start + [3.0, 5.0]
    c.free(e)
    assert c.free_pages() == (16, 16)
    with pytest.raises(RuntimeError, match="no sequence"):
        c.length(e)


def small(dev, kv_heads=4):
    from kvmix_amd.decoder import DecoderConfig, init_weights

    cfg = DecoderConfig(hidden_size=512, num_layers=3, num_heads=4, num_kv_heads=kv_heads, intermediate_size=704, vocab_size=1000)
    return cfg, init_weights(cfg, dev)


@pytest.mark.parametrize("kv_heads", [4, 2])
def test_chunks_of_a_prompt_are_the_prompt(dev, kv_heads):
    """With everything in fp16 the chunks' logits are those of the dense prompt, up to roundings of the stack in fp16."""
    from kvmix_amd.decoder import Decoder, kvmix_layers
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg, w = small(dev, kv_heads)
    ids = torch.randint(0, cfg.vocab_size, (1, 300), device=dev)
    dense = Decoder(cfg, w, *kvmix_layers(cfg, [4] * 3, [4] * 3, residual_length=4096))
    want = dense.forward(ids)[0]
    m = PagedDecoder(cfg, w, [4] * 3, [4] * 3, window=4096)
    s, other = m.add(), m.add()
    m.forward({s: ids[0, :100]})
    m.forward({s: ids[0, 100:101], other: ids[0, :7]})
    got = m.forward({other: ids[0, 7:9], s: ids[0, 101:]})[s]
    size = float(want.std())
    assert float((got - want).abs().max()) < 0.05 * size
    # one token at a time, next to another sequence
    nxt = want.argmax().reshape(1)
    a = dense.forward(nxt[None])[0]
    b = m.forward({s: nxt, other: nxt})[s]
    assert float((a - b).abs().max()) < 0.05 * size


def test_generation_and_likelihoods(dev):
    from kvmix_amd import ops
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg, w = small(dev, 2)
    m = PagedDecoder(cfg, w, [4, 3, 4], [4, 2, 4], page_size=32, window=32)
    prompt = torch.randint(0, cfg.vocab_size, (200,), device=dev)
    a = m.add()
    first = m.forward({a: prompt})[a].argmax().reshape(1)
    b = m.fork(a)
    ids, top_lp, top_id = m.generate([a, b], first.expand(2), 40, alternatives=3)
    assert ids.shape == (2, 40) and top_id.shape == (2, 39, 3) and torch.equal(ids[0], ids[1])  # two forks that do the same
    assert torch.equal(ids[:, 1:], top_id[..., 0]) and (top_lp.diff(dim=-1) <= 0).all()
    assert m.cache.length(a) == 239
    # a text's likelihoods, in chunks, against the logits of the same chunks
    text = torch.cat([prompt, ids[0]])
    lp, entropy = m.score(text, chunk=64)
    assert lp.shape == entropy.shape == (239,) and (lp <= 0).all() and (entropy >= 0).all()
    s = m.add()
    want = []
    for at in range(0, 239, 64):
        logits = m.forward({s: text[at:min(at + 64, 239)]}, every=True)[s]
        want.append(torch.log_softmax(logits.double(), -1).gather(-1, text[at + 1:at + 1 + logits.shape[0], None])[:, 0])
    assert torch.allclose(lp.double(), torch.cat(want), atol=1e-4)
    assert ops.token_logprobs(logits, text[-logits.shape[0]:])[0].shape == (logits.shape[0],)
    free = m.cache.free_pages()
    for s in (a, b, s):
        m.free(s)
    assert m.cache.free_pages()[0] > free[0]
    assert m.forward({}) == {} and m.score(text[:1])[0].shape == (0,)
