"""The best continuations of beams: against 64 bits, over types, sizes and rows that ask for care."""
import math

import pytest
import torch

pytestmark = pytest.mark.gpu

INF = float("inf")


def plain(logits, scores, count, done=None, end=None, stay=False):
    """In float64 on the CPU, candidate by candidate: (scores, parents, tokens)"""
    R, W, V = logits.shape
    x, scores = logits.double().cpu(), scores.double().cpu()
    out = []
    for r in range(R):
        found = []
        for w in range(W):
            base = float(scores[r, w])
            lse = torch.logsumexp(x[r, w], -1)
            if done is not None and done[r, w]:
                found += [(base if i == 0 and math.isfinite(base) else -INF, w, i, end) for i in range(count)]
            elif not math.isfinite(base) or not torch.isfinite(lse):
                found += [(-INF, w, i, i) for i in range(count)]
            else:
                # (stable: equal logits in the order of their indexes)
                best, at = (base + (x[r, w] - lse)).sort(descending=True, stable=True)
                found += [(float(best[i]), w, int(at[i]), int(at[i])) for i in range(count)]
        best = sorted(found, key=lambda c: (-c[0], c[1], c[2]))[:count]
        if stay:
            placed, free = [None] * count, [w for w in range(W) if all(c[1] != w for c in best)]
            for c in best:
                placed[c[1] if placed[c[1]] is None else free.pop(0)] = c
            best = placed
        out.append(best)
    pick = lambda i, kind: torch.tensor([[c[i] for c in row] for row in out], dtype=kind).reshape(R, count)
    return pick(0, torch.float64), pick(1, torch.int64), pick(3, torch.int64)


def check(got, want):
    """Scores are off by the rounding to fp32 (2^-24) and by lse's error: every term's exponent is rounded twice (2^-24 of up to 24 bits
    that matter, each), the exponential once (2^-23), a thread adds up to 64 terms and the block eight sums more, all of them relative
    to the sum: 2 * 24 * 0.7 * 2^-24 + 2^-23 + 72 * 2^-24 < 64 * 2^-23.  Choices are the same wherever no two scores are closer."""
    (score, parent, token), (s, p, t) = [x.cpu() for x in got], want
    assert score.dtype == torch.float32 and parent.dtype == token.dtype == torch.int64 and score.shape == s.shape
    dead = s == -INF
    assert torch.equal(score == -INF, dead)
    assert ((score.double() - s).abs()[~dead] <= (2.0 ** -23 * s.abs() + 64 * 2.0 ** -23)[~dead]).all()
    assert torch.equal(parent, p) and torch.equal(token, t)


def random(R, W, V, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed)
    logits = (torch.randn(R, W, V, generator=g) * 3).to(dtype).to(dev)
    return logits, (-8 * torch.rand(R, W, generator=g)).to(dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("R,W,V,count", [
    (1, 1, 1, 1), (1, 4, 4, 4), (3, 2, 5, 5), (2, 5, 301, 10), (1, 4, 32000, 4), (4, 3, 32001, 6), (2, 16, 1009, 32), (1, 64, 500, 64), (5, 1, 70003, 64),
    (40, 8, 9000, 8),
])
def test_against_64_bits(dev, R, W, V, count, dtype):
    from kvmix_amd import ops

    logits, scores = random(R, W, V, dtype, dev, seed=V + W)
    check(ops.beam_select(logits, scores, count), plain(logits, scores, count))
    done = torch.rand(R, W, generator=torch.Generator().manual_seed(2)) < 0.4
    for stay in (False, True) if count == W else (False,):
        check(ops.beam_select(logits, scores, count, done.to(dev), V // 2, stay), plain(logits, scores, count, done, V // 2, stay))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("V", [257, 4099, 33333])
def test_equal_rows_are_equal(dev, V, dtype):
    """The same logits at other alignments, at equal scores: ties go to the lower beam, token by token, down to the last bit."""
    from kvmix_amd import ops

    one, _ = random(1, 1, V, dtype, dev)
    logits, scores = one.expand(2, 6, V).contiguous(), torch.full((2, 6), -1.5, device=dev)
    score, parent, token = ops.beam_select(logits, scores, 12)
    check((score, parent, token), plain(logits, scores, 12))
    assert parent[0].tolist() == list(range(6)) + list(range(6))
    assert torch.equal(score[:, :1].expand(2, 6), score[:, :6])


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
def test_rows_that_ask_for_care(dev, dtype):
    """Constant rows, masks (of -inf and of the type's lowest value) that leave little or nothing, infinities, NaN, lost scores."""
    from kvmix_amd import ops

    V, low = 20000, torch.finfo(dtype).min
    logits, scores = random(4, 12, V, dtype, dev, seed=5)
    rows = logits.view(-1, V)
    rows[0] = 1.25                                        # all alike
    rows[1] = -INF                                        # nothing
    rows[2, 3:] = -INF                                    # three tokens
    rows[3] = low                                         # all alike, as low as can be
    rows[4, :19990] = low
    rows[5, 777] = float("nan")
    rows[6, 778] = INF
    rows[7, 1:] = -INF                                    # one token, sure
    rows[8, :] = 0.0
    rows[8, 10000:] = -0.0                                # all alike
    rows[9, :] = -INF
    rows[9, 19999] = float("nan")                         # in a part that has nothing else
    rows[10, 0] = torch.finfo(dtype).max                  # one token, very sure
    rows[24:36] = -INF                                    # a request of which nothing can be computed
    scores.view(-1)[11], scores.view(-1)[12], scores.view(-1)[13] = -INF, float("nan"), INF
    for count in (1, 12, 40, 64):
        check(ops.beam_select(logits, scores, count), plain(logits, scores, count))
    check(ops.beam_select(logits, scores, 12, stay=True), plain(logits, scores, 12, stay=True))
    done = torch.zeros(4, 12, dtype=torch.bool)
    done[0, 1], done[0, 5], done[1, 0], done[2, :], done[3, ::2] = True, True, True, True, True
    for count in (3, 12, 64):
        check(ops.beam_select(logits, scores, count, done.to(dev), 9), plain(logits, scores, count, done, 9))


def test_the_first_step(dev):
    """One beam of each request counts: all children are its own, the best one in its place."""
    from kvmix_amd import ops

    logits, scores = random(3, 5, 3001, torch.float32, dev)
    scores[:] = -INF
    scores[:, 2] = 0.0
    got = ops.beam_select(logits, scores, stay=True)
    check(got, plain(logits, scores, 5, stay=True))
    assert (got[1] == 2).all() and (got[0][:, 2:3] >= got[0]).all()


def test_strides(dev):
    from kvmix_amd import ops

    logits, scores = random(4, 3, 1001, torch.float16, dev)
    want = ops.beam_select(logits, scores, 6)
    wide = torch.zeros(4, 3, 1100, device=dev).half()
    wide[..., 50:1051] = logits
    two = torch.stack([scores, scores], -1)
    for x, s in ((wide[..., 50:1051], scores), (logits.transpose(0, 1).contiguous().transpose(0, 1), two[..., 0]),
                 (logits.permute(2, 0, 1).contiguous().permute(1, 2, 0), scores)):
        for a, b in zip(ops.beam_select(x, s, 6), want):
            assert torch.equal(a, b)
    same = logits[:, :1].expand(4, 3, 1001)
    for a, b in zip(ops.beam_select(same, scores), ops.beam_select(same.contiguous(), scores)):
        assert torch.equal(a, b)
    assert [t.shape for t in ops.beam_select(logits[:0], scores[:0], 2)] == [(0, 2)] * 3


def test_refusals(dev):
    from kvmix_amd import ops

    logits, scores = random(2, 3, 50, torch.float32, dev)
    done = torch.zeros(2, 3, dtype=torch.bool, device=dev)
    for args, match in [
        ((logits[0], scores), "requests"), ((logits.double(), scores), "float16"), ((logits, scores.half()), "float32"), ((logits, scores[:, :2]), "scores"),
        ((logits, scores, 0), "count"), ((logits, scores, 51), "count"), ((logits, scores, 65), "count"), ((logits[:, :0], scores[:, :0]), "beam"),
        ((logits, scores, 4, None, None, True), "places"), ((logits, scores, 3, done), "ends them"), ((logits, scores, 3, done, 50), "ends them"),
        ((logits, scores, 3, done, -1), "ends them"), ((logits, scores, 3, done.int(), 1), "bool"), ((logits, scores, 3, done[:1], 1), "bool"),
        ((logits, scores.cpu()), "cpu"), ((logits.clone().requires_grad_(), scores), "no derivative"), ((logits, scores.clone().requires_grad_()), "no derivative"),
        ((logits.expand(2, 3, 50)[:, :1].expand(2, 65, 50), scores[:, :1].expand(2, 65)), "64 beams"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            ops.beam_select(*args)


def test_captured_and_on_another_stream(dev):
    from kvmix_amd import ops

    logits, scores = random(3, 4, 40000, torch.float32, dev)
    want = ops.beam_select(logits, scores, stay=True)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        got = ops.beam_select(logits, scores, stay=True)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))
    graphs = []
    for _ in range(2):
        graph, x = torch.cuda.CUDAGraph(), logits.clone()
        with torch.cuda.graph(graph):
            out = ops.beam_select(x, scores, stay=True)
        graphs.append((graph, x, out))
    for i in range(3):
        for j, (graph, x, _) in enumerate(graphs):
            x.copy_(logits.roll(17 * i + j, -1) * (1 + j))
            graph.replay()
        torch.cuda.synchronize()
        for j, (_, x, out) in enumerate(graphs):
            assert all(torch.equal(a, b) for a, b in zip(out, ops.beam_select(x, scores, stay=True)))


@pytest.mark.parametrize("R,W,V,count,dtype", [
    (1, 20, 40000, 20, torch.float32),          # some hundred parts of a request, more than a block reads at once
    (2, 3, 40000, 2, torch.float32),            # few of them, and more than are compared by all threads
    (1, 64, 33000, 3, torch.float16),
    (1, 2, 1 << 20, 5, torch.float32),          # more parts to a beam than lanes
    (1, 32, 1 << 20, 2, torch.bfloat16),        # the largest
    (1, 3, 5000, 1, torch.float16),
])
def test_many_parts(dev, R, W, V, count, dtype):
    from kvmix_amd import ops

    logits, scores = random(R, W, V, dtype, dev, seed=V)
    logits[:, :, V // 3:V // 3 + 5] = 25.0  # the best ones are equal, and in one part
    scores[:, 1:] = scores[:, :1]
    done = torch.rand(R, W, generator=torch.Generator().manual_seed(3)) < 0.3
    check(ops.beam_select(logits, scores, count), plain(logits, scores, count))
    check(ops.beam_select(logits, scores, count, done.to(dev), 7), plain(logits, scores, count, done, 7))


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16])
def test_logits_beyond_the_caches(dev, dtype):
    """More than 32 MB of them, at odd offsets."""
    from kvmix_amd import ops

    R, W, V = 70, 8, 32003
    logits, scores = random(R, W, V, dtype, dev, seed=8)
    got = ops.beam_select(logits, scores, 10)
    for r in (*range(0, R, 9), R - 1):
        check([x[r:r + 1] for x in got], plain(logits[r:r + 1], scores[r:r + 1], 10))
