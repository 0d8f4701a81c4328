"""Beam search of the decoders: choices, states that move with them, ends, sequences that share pages."""
import itertools

import pytest
import torch

from test_gpu_paged_cache import small

pytestmark = pytest.mark.gpu


def search(logits_of, prompts, beams, steps, end=None):
    """By the definition, in float64 on the CPU: [(ids, score)] per prompt, the best first; logits_of(ids) -> [vocab]"""
    out = []
    for prompt in prompts:
        found = [([], 0.0, False)]
        for _ in range(steps):
            more = []
            for w, (ids, score, over) in enumerate(found):
                if over:
                    more.append((score, w, end, ids + [end], True))
                    continue
                lp = torch.log_softmax(logits_of(prompt + ids).double(), -1)
                more += [(score + float(lp[v]), w, v, ids + [v], v == end) for v in range(lp.numel())]
            more.sort(key=lambda c: (-c[0], c[1], c[2]))
            found = [(ids, score, over) for score, _, _, ids, over in more[:beams]]
        out.append([(ids, score) for ids, score, _ in found])
    return out


def table_decoder(dev, vocab, graph=False):
    """A Decoder whose logits depend on all tokens so far in a way of their own, and whose `cache` is those tokens."""
    from kvmix_amd.decoder import Decoder, DecoderConfig

    table = torch.randn(499, vocab, generator=torch.Generator().manual_seed(7)).mul(3).float()

    def place(ids):
        h = 1
        for i in ids:
            h = (h * 31 + int(i) * 7 + 3) % 499
        return h

    class Table(Decoder):
        def forward(self, ids):
            seen = ids if self.position == 0 else torch.cat([self.caches[0][0], ids], 1)
            self.position = seen.shape[1]
            self.caches = [(seen.contiguous(), None, 5)]
            return table[[place(row) for row in seen.tolist()]].to(dev)

    cfg = DecoderConfig(hidden_size=64, num_layers=1, num_heads=1, num_kv_heads=1, intermediate_size=64, vocab_size=vocab)
    return Table(cfg, {}, [None]), lambda ids: table[place(ids)]


@pytest.mark.parametrize("vocab,beams,steps,end", [(11, 1, 4, None), (11, 4, 6, None), (11, 4, 9, 3), (64, 8, 5, 1), (9, 9, 7, 0), (300, 3, 4, None)])
def test_choices_and_states(dev, vocab, beams, steps, end):
    """The tokens seen so far move with their beams: the same sequences as from the definition, equal scores among them impossible."""
    model, logits_of = table_decoder(dev, vocab)
    prompts = [[1, 2, 3], [4, 0, 5], [8, 8, 8]]
    ids, scores = model.beam_search(torch.tensor(prompts, device=dev), beams, steps, end)
    want = search(logits_of, prompts, beams, steps, end)
    assert ids.shape == (3, beams, steps) and scores.shape == (3, beams)
    for r in range(3):
        assert ids[r].tolist() == [i for i, _ in want[r]]
        # a score is rounded to fp32 in every step, after an error of 64 half steps of 1 in the sum
        tol = sum(2.0 ** -24 * abs(want[r][-1][1]) + 64 * 2.0 ** -23 for _ in range(steps))
        assert max(abs(float(a) - b) for a, (_, b) in zip(scores[r], want[r])) <= tol


def off_by(model, ids, sequences):
    """Log probabilities of every token of `sequences` [n, steps] after the prompt `ids` [Q], by the model fed with all of them as prompts;
    and four times what its logits may be off by in each: 0.05 of their spread, which other splits of a prompt are held to."""
    lp, tol = [], 0.0
    for row in sequences:
        s = model.add()
        logits = model.forward({s: torch.cat([ids, row])[:-1]}, every=True)[s][ids.numel() - 1:].double()
        model.free(s)
        lp.append(torch.log_softmax(logits, -1).gather(-1, row[:, None])[:, 0].sum())
        tol = max(tol, 4 * 0.05 * float(logits.std()) * row.numel())
    return torch.stack(lp), tol


def test_beams_of_the_decoders(dev):
    """Eager, replayed and paged: a beam's score is its tokens' likelihood, one beam is the greedy choice, the order is that of scores."""
    from kvmix_amd.decoder import Decoder, GraphDecoder, kvmix_layers
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg, w = small(dev, 2)
    prompt = torch.randint(0, cfg.vocab_size, (2, 70), generator=torch.Generator().manual_seed(3)).to(dev)
    paged = PagedDecoder(cfg, w, [4] * 3, [4] * 3, window=4096)
    exact = PagedDecoder(cfg, w, [4] * 3, [4] * 3, window=4096)
    made = []
    for kind in (Decoder, GraphDecoder):
        model = kind(cfg, w, *kvmix_layers(cfg, [4] * 3, [4] * 3, residual_length=4096, capacity=128))
        made.append(model.beam_search(prompt, 4, 12))
    seqs = [paged.add() for _ in range(2)]
    first = paged.forward(dict(zip(seqs, prompt)))
    logits = torch.stack([first[s] for s in seqs])
    free = paged.cache.free_pages()
    made.append(paged.beam_search(seqs, logits, 4, 12))
    assert paged.cache.free_pages() == free and [paged.cache.length(s) for s in seqs] == [70, 70]
    for ids, scores in made:
        assert ids.shape == (2, 4, 12) and (scores.diff(dim=-1) <= 0).all()
        for r in range(2):
            assert len({tuple(b) for b in ids[r].tolist()}) == 4
            lp, tol = off_by(exact, prompt[r], ids[r])
            assert float((lp - scores[r].double()).abs().max()) <= tol
    one, score = paged.beam_search(seqs, logits, 1, 9)
    greedy = paged.generate([paged.fork(s) for s in seqs], logits.argmax(-1), 9)
    assert torch.equal(one[:, 0], greedy)


def test_one_decoder_again_and_again(dev):
    """A decoder whose caches are reset searches as a new one does, with as many prompts and beams as it likes, and generates."""
    from kvmix_amd.decoder import Decoder, GraphDecoder, kvmix_layers

    cfg, w = small(dev, 2)
    prompts = torch.randint(0, cfg.vocab_size, (3, 90), generator=torch.Generator().manual_seed(5)).to(dev)
    for kind in (Decoder, GraphDecoder):
        new = lambda: kind(cfg, w, *kvmix_layers(cfg, [4, 2, 3], [2, 4, 4], residual_length=40, capacity=64))
        used = new()
        for rows, beams, steps in ((2, 3, 9), (1, 4, 50), (3, 1, 5), (2, 3, 9)):
            assert used.position == 0
            got, want = (d.beam_search(prompts[:rows], beams, steps) for d in (used, new()))
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
            assert all(c.kv_seq_len == 90 + steps - 1 and c.as_tuple()[1].shape[0] == rows * beams for c in used.caches)
            for c in used.caches:
                c.reset()
            used.position = 0
        for c in used.caches:
            c.fit(3)
        assert torch.equal(used.generate(prompts, 7), new().generate(prompts, 7))


@pytest.mark.parametrize("window", [32, 4096])
def test_every_continuation(dev, window):
    """With as many beams as there are continuations of all but the last token, the best one of all is found."""
    from kvmix_amd.decoder import DecoderConfig, init_weights
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg = DecoderConfig(hidden_size=512, num_layers=2, num_heads=4, num_kv_heads=2, intermediate_size=704, vocab_size=7)
    w = init_weights(cfg, dev)
    model = PagedDecoder(cfg, w, [4] * 2, [4] * 2, page_size=32, window=window)
    s = model.add()
    prompt = torch.randint(0, 7, (75,), generator=torch.Generator().manual_seed(1)).to(dev)
    logits = model.forward({s: prompt})[s]
    with pytest.raises(RuntimeError, match="64 beams"):
        model.beam_search([s], logits[None], 49, 3)  # (not more than there are tokens)
    ids, scores = model.beam_search([s], logits[None], 7, 2)
    every = torch.tensor(list(itertools.product(range(7), repeat=2)), device=dev)
    lp = []
    for row in every:
        twin = model.fork(s)
        after = model.forward({twin: row[:1]})[twin]
        lp.append(torch.log_softmax(logits.double(), -1)[row[0]] + torch.log_softmax(after.double(), -1)[row[1]])
        model.free(twin)
    lp = torch.stack(lp)
    best = lp.sort(descending=True).values[:7]
    # (one token of seven forks together and one of each fork alone: other splits of the same sums in fp16)
    tol = 2 * 0.05 * float(after.std())
    assert float((best - scores[0].double()).abs().max()) <= tol
    found = torch.stack([lp[(every == row).all(-1)][0] for row in ids[0]])
    assert float((found - scores[0].double()).abs().max()) <= tol


def test_ends_and_pages(dev):
    """Beams that have ended fill up with that token; a pool without room for the beams leaves nothing behind."""
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg, w = small(dev, 2)
    model = PagedDecoder(cfg, w, [4] * 3, [4] * 3, row_pages=12, packed_pages=64, page_size=32, window=32)
    s = model.add()
    logits = model.forward({s: torch.arange(60, device=dev)})[s]
    ids, _ = model.beam_search([s], logits[None], 3, 5)
    end = int(ids[0, 0, 1])
    ids, scores = model.beam_search([s], logits[None], 3, 8, end)
    assert torch.isfinite(scores).all()
    for row in ids[0].tolist():
        if end in row:
            assert set(row[row.index(end):]) == {end}
    free = model.cache.free_pages()
    with pytest.raises(RuntimeError):
        model.beam_search([s], logits[None], 20, 70)
    assert model.cache.free_pages() == free and len(model.cache._sequences) == 1
    assert model.beam_search([s], logits[None], 3, 5)[0].shape == (1, 3, 5)


def test_refusals(dev):
    from kvmix_amd.decoder import Decoder, kvmix_layers
    from kvmix_amd.paged_decoder import PagedDecoder

    cfg, w = small(dev, 2)
    model = PagedDecoder(cfg, w, [4] * 3, [4] * 3, page_size=32, window=32)
    a = model.add()
    logits = model.forward({a: torch.arange(9, device=dev)})[a][None]
    for args, match in [(([a], logits, 0, 3), "beams"), (([a], logits, 65, 3), "beams"), (([a], logits, 2, 0), "new token"), (([a, a], logits.expand(2, -1), 2, 3), "different"),
                        (([a], logits[0], 2, 3), "row"), (([a], logits, 2, 3, 1000), "vocabulary"), (([a], logits, 2, 3, -1), "vocabulary"), (([a + 5], logits, 2, 3), "no sequence")]:
        with pytest.raises(RuntimeError, match=match):
            model.beam_search(*args)
    many = [model.add() for _ in range(20)]
    with pytest.raises(RuntimeError, match="1024 beams"):
        model.beam_search(many, logits.expand(20, -1), 64, 2)
    assert model.beam_search([], logits[:0], 2, 3)[0].shape == (0, 2, 3) and model.cache.length(a) == 9
    dense = Decoder(cfg, w, *kvmix_layers(cfg, [4] * 3, [4] * 3, residual_length=64))
    for args in ((torch.arange(5, device=dev)[None], 2, 0), (torch.zeros(1, 0, dtype=torch.long, device=dev), 2, 3), (torch.arange(5, device=dev)[None], 65, 3),
                 (torch.zeros(17, 5, dtype=torch.long, device=dev), 64, 3)):
        with pytest.raises(RuntimeError, match="beam_search"):
            dense.beam_search(*args)
    dense.forward(torch.arange(5, device=dev)[None])
    with pytest.raises(RuntimeError, match="nothing is cached"):
        dense.beam_search(torch.arange(5, device=dev)[None], 2, 3)


@pytest.mark.parametrize("in_place", [True, False])
def test_caches_that_are_reordered(dev, in_place):
    """Every entry of every layer, through the cache's own call and for all layers at once, and steps afterwards."""
    from kvmix_amd.cache import PackedKVCache, reorder_caches, repeat_caches

    g = torch.Generator().manual_seed(2)
    caches = [PackedKVCache(b, c, residual_length=40) for b, c in ((4, 2), (1, 4))]
    for c in caches:
        c.append(*(torch.randn(6, 2, 200, 128, generator=g).half().to(dev) for _ in range(2)))
        c.append(*(torch.randn(6, 2, 1, 128, generator=g).half().to(dev) for _ in range(2)))
    before = [[t.clone() for t in c.as_tuple() if torch.is_tensor(t)] for c in caches]
    index = torch.tensor([1, 1, 0, 5, 4, 4], device=dev)
    if in_place:
        for c in caches:
            c.reorder(index)
    else:
        reorder_caches([None, *caches], index)
    for c, was in zip(caches, before):
        for a, b in zip([t for t in c.as_tuple() if torch.is_tensor(t)], was):
            assert torch.equal(a, b[index])
    twice = [[t.clone() for t in c.as_tuple() if torch.is_tensor(t)] for c in caches]
    more = [torch.randn(6, 2, 1, 128, generator=g).half().to(dev) for _ in range(2)]
    caches[0].append(*more)
    tail = caches[0].as_tuple()[1]  # of the keys: the new token behind what is left of the others
    n = tail.shape[2] - 1
    assert n > 0 and torch.equal(tail[:, :, n:], more[0]) and torch.equal(tail[:, :, :n], before[0][1][index][:, :, -n:])
    # and repeated, the second cache, which has had no more tokens
    assert repeat_caches([None, caches[1], (more[0], None, 7)], 3)[2][0].shape[0] == 18
    for a, b in zip([t for t in caches[1].as_tuple() if torch.is_tensor(t)], twice[1]):
        assert torch.equal(a, b.repeat_interleave(3, 0))
    caches[1].append(*(t.repeat_interleave(3, 0) for t in more))
    assert torch.equal(caches[1].as_tuple()[5][:, :, -1:], more[1].repeat_interleave(3, 0))
