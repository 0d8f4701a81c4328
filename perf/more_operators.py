"""The operators between a decoder's projections and its cache when many requests are served at once, as cases with sizes, for
measuring them.

Four kinds of calls, through the public entry points only:

* ``rope``     the fused projection of a step's new tokens: queries and keys are rotated, keys and values go into their fp16
               pages (``ops.paged_rope_append``);
* ``adapt``    the low-rank adapters of the requests of a batch, added to a projection that they share (``ops.add_adapters``);
* ``beam``     the best continuations over the beams of every request and the vocabulary (``ops.beam_select``);
* ``reorder``  the states of all layers moved to the beams that go on, in place (``ops.reorder_rows``).

Without `own` the operators are computed with elementary torch operations in 32 bits (beams' scores in 64: they decide an order).
"""
from __future__ import annotations

import math

import torch

own = False

DEV = "cuda"
TAIL = 70  # tokens that a contiguous cache holds in fp16


# ---------------------------------------------------------------------------------------------------------------------
# the cases

def listed():
    return [
        # one user, one token: bound by latency
        {"name": "rope_b1_n1_h32", "kind": "rope", "batch": 1, "new": 1, "heads": 32, "kv_heads": 32, "head_dim": 128, "page": 64,
         "tables": "float16"},
        # a step of a running batch with grouped-query heads, positions far out
        {"name": "rope_b64_n1_h32_kv8", "kind": "rope", "batch": 64, "new": 1, "heads": 32, "kv_heads": 8, "head_dim": 128, "page": 64,
         "tables": "float32"},
        # chunks of prompts of odd length
        {"name": "rope_b8_n1021_h32", "kind": "rope", "batch": 8, "new": 1021, "heads": 32, "kv_heads": 32, "head_dim": 128, "page": 64,
         "tables": "float32"},
        # one request's token with its small adapter: bound by latency
        {"name": "adapt_b1_r8_k4096_n4096", "kind": "adapt", "singles": 1, "chunks": 0, "chunk": 0, "adapters": 4, "rank": 8, "k": 4096,
         "n": 4096, "bare": False, "dtype": "float16"},
        # a step of 64 requests of 40 tenants, beside the fused query, key and value projection
        {"name": "adapt_b64_r16_k4096_n12288", "kind": "adapt", "singles": 64, "chunks": 0, "chunk": 0, "adapters": 40, "rank": 16,
         "k": 4096, "n": 12288, "bare": False, "dtype": "float16"},
        # chunks of prompts beside single tokens, some requests without an adapter, beside the projection down from the wide layer
        {"name": "adapt_b40_c3x509_r32_k11008_n4096", "kind": "adapt", "singles": 40, "chunks": 3, "chunk": 509, "adapters": 9, "rank": 32,
         "k": 11008, "n": 4096, "bare": True, "dtype": "float16"},
        # long prompts' chunks with wide adapters
        {"name": "adapt_c8x1021_r64_k4096_n4096_bf16", "kind": "adapt", "singles": 0, "chunks": 8, "chunk": 1021, "adapters": 6, "rank": 64,
         "k": 4096, "n": 4096, "bare": False, "dtype": "bfloat16"},
        # one request of four beams
        {"name": "beam_b1_w4_v32000", "kind": "beam", "requests": 1, "beams": 4, "count": 4, "vocab": 32000, "dtype": "float32",
         "ended": False, "stay": True},
        # a batch of requests, some of whose beams have ended, twice as many candidates as beams
        {"name": "beam_b16_w5_v32000_c10", "kind": "beam", "requests": 16, "beams": 5, "count": 10, "vocab": 32000, "dtype": "float16",
         "ended": True, "stay": False},
        # many requests of eight beams
        {"name": "beam_b64_w8_v32000", "kind": "beam", "requests": 64, "beams": 8, "count": 8, "vocab": 32000, "dtype": "float32",
         "ended": True, "stay": True},
        # four beams at a short context, two layers: bound by the launch
        {"name": "reorder_b1_w4_l2_t300", "kind": "reorder", "requests": 1, "beams": 4, "layers": 2, "tokens": 300, "kv_heads": 8,
         "head_dim": 128, "k_bits": 4, "v_bits": 4},
        # the caches of eight layers (a shallow model's, or a stage's) of eight requests at a long context
        {"name": "reorder_b8_w4_l8_t8190", "kind": "reorder", "requests": 8, "beams": 4, "layers": 8, "tokens": 8190, "kv_heads": 8,
         "head_dim": 128, "k_bits": 4, "v_bits": 2},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["rope", "rope", "adapt", "adapt", "adapt", "beam", "beam", "reorder"])
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 8), (16, 4), (12, 12), (8, 1)])
    dim = 128 if rng.random() < 0.8 else 64
    if kind == "rope":
        new = 1 if rng.random() < 0.4 else _log_int(rng, 2, 1021)
        return {"kind": kind, "batch": max(1, min(_log_int(rng, 1, 128), 8168 * 96 // (new * (heads + 2 * kv_heads)))), "new": new,
                "heads": heads, "kv_heads": kv_heads, "head_dim": dim, "page": rng.choice([32, 64, 64, 128]),
                "tables": rng.choice(["float16", "float32"])}
    if kind == "adapt":
        singles = _log_int(rng, 1, 128)
        chunks = 0 if rng.random() < 0.5 else rng.randint(1, 8)
        return {"kind": kind, "singles": singles, "chunks": chunks, "chunk": _log_int(rng, 2, 800) if chunks else 0,
                "adapters": _log_int(rng, 1, 60), "rank": rng.choice([8, 16, 16, 24, 32, 64]), "k": 8 * _log_int(rng, 64, 1376) if rng.random() < 0.5 else 4096,
                "n": 8 * _log_int(rng, 64, 1500) if rng.random() < 0.5 else 4096, "bare": rng.random() < 0.3,
                "dtype": rng.choice(["float16", "float16", "bfloat16"])}
    if kind == "beam":
        vocab = 32000 if rng.random() < 0.5 else _log_int(rng, 300, 130000)
        beams = _log_int(rng, 1, 16)
        count = beams if rng.random() < 0.6 else 2 * beams
        return {"kind": kind, "requests": max(1, min(_log_int(rng, 1, 64), 512 * 32000 // (vocab * beams) // 2)), "beams": beams, "count": count,
                "vocab": vocab, "dtype": rng.choice(["float32", "float32", "float16", "bfloat16"]), "ended": rng.random() < 0.5,
                "stay": count == beams and rng.random() < 0.5}
    beams, layers = rng.randint(2, 12), rng.randint(1, 8)
    return {"kind": kind, "requests": rng.randint(1, 8), "beams": beams, "layers": layers, "kv_heads": min(kv_heads, 8), "head_dim": dim,
            "tokens": 32 * _log_int(rng, 1, max(1, 64 * 32 * 32 // (96 * layers))) + rng.randint(1, 31), "k_bits": rng.choice([1, 2, 4]), "v_bits": rng.choice([1, 2, 4])}


def _sequences(case):
    """(tokens, adapter or -1) of each sequence: chunks of prompts, each a little shorter than the one before, then single tokens."""
    counts = [max(1, case["chunk"] - 7 * i) for i in range(case["chunks"])] + [1] * case["singles"]
    return [(n, -1 if case["bare"] and i % 4 == 3 else (5 * i + 2) % case["adapters"]) for i, n in enumerate(counts)]


def _size(case):
    return {"float16": 2, "bfloat16": 2, "float32": 4}[case["dtype"]]


def _runs(case):
    """(rows, bytes of a run, bytes from one to the next) of a sequence in each buffer of a layer's cache: codes, scales and minima of
    the keys (per channel) and the values (per token), and the tails."""
    H, D, T = case["kv_heads"], case["head_dim"], case["tokens"] // 32 * 32
    cap = -(-max(T, 1) // 352) * 352
    kw, vw = case["k_bits"], D * case["v_bits"] // 32
    return [(H * D, T // 32 * kw * 4, cap // 32 * kw * 4), (H * D, T // 32 * 2, cap // 32 * 2), (H * D, T // 32 * 2, cap // 32 * 2),
            (H, T * vw * 4, cap * vw * 4), (H, T * D // 32 * 2, cap * D // 32 * 2), (H, T * D // 32 * 2, cap * D // 32 * 2),
            (H, TAIL * D * 2, 2 * TAIL * D * 2), (H, TAIL * D * 2, 2 * TAIL * D * 2)]


def work(case):
    if case["kind"] == "rope":
        D, tokens = case["head_dim"], case["batch"] * case["new"]
        moved = tokens * (case["heads"] + 2 * case["kv_heads"]) * D * 2
        return {"bytes": 2 * moved + 2 * tokens * D * (2 if case["tables"] == "float16" else 4),
                "flops": 3 * tokens * (case["heads"] + case["kv_heads"]) * D}
    if case["kind"] == "adapt":
        seqs = _sequences(case)
        tokens, adapted = sum(n for n, _ in seqs), sum(n for n, a in seqs if a >= 0)
        used = len({a for _, a in seqs if a >= 0})
        return {"bytes": 2 * (2 * tokens * case["n"] + adapted * case["k"] + used * case["rank"] * (case["k"] + case["n"])),
                "flops": 2 * adapted * case["rank"] * (case["k"] + case["n"])}
    if case["kind"] == "beam":
        rows = case["requests"] * case["beams"]
        return {"bytes": rows * (case["vocab"] * _size(case) + 5) + case["requests"] * case["count"] * 20, "flops": 4 * rows * case["vocab"]}
    dead = case["beams"] - (case["beams"] + 1) // 2
    one = case["layers"] * sum(rows * run for rows, run, _ in _runs(case))
    return {"bytes": case["requests"] * 2 * dead * one, "flops": 0}


# ---------------------------------------------------------------------------------------------------------------------
# inputs

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, *shape, dtype=torch.float16):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=dtype)


def prepare(case, seed):
    return {"case": case, **globals()["_prepare_" + case["kind"]](case, _generator(seed))}


def _prepare_rope(case, gen):
    B, n, nh, H, D, P = (case[x] for x in ("batch", "new", "heads", "kv_heads", "head_dim", "page"))
    # the sequences' fp16 pages before this call hold between 0 and P - 1 tokens of the page that is being written; packed pages
    # of thousands of tokens lie before them
    lens, far = [n + (7 * b + 5) % P for b in range(B)], [P * (61 * b % 113) for b in range(B)]
    per = max(-(-m // P) for m in lens)
    pages = torch.randperm(B * per + 3, generator=gen, device=DEV).cpu()[:B * per].reshape(B, per)
    qkv = _normal(gen, B * n, nh + 2 * H, D)
    qkv[:, nh:nh + H] *= 1.0 + 9.0 * (torch.rand(H, D, generator=gen, device=DEV).argsort(-1) < 4).half()
    at = torch.tensor([[m - n + i for i in range(n)] for m in lens])
    pos = (at + torch.tensor(far)[:, None]).reshape(-1).to(DEV)
    angle = pos.double()[:, None] / 10000.0 ** (torch.arange(0, D, 2, device=DEV, dtype=torch.float64) / D)
    angle = torch.cat([angle, angle], -1)
    kind = getattr(torch, case["tables"])
    s = {"qkv": qkv, "cos": angle.cos().to(kind), "sin": angle.sin().to(kind), "rows": _normal(gen, B * per + 3, H, 2, P, D),
         "slot": (pages.gather(1, at // P) * P + at % P).reshape(-1).to(DEV)}
    if own:
        from kvmix_amd import ops

        # (the packed pages do not matter here: the plan is of the pages that are written)
        s["plan"] = ops.paged_plan(pages.to(torch.int32), lens, [0] * B, [n] * B, nh, H, D, P, DEV)
    return s


def _prepare_adapt(case, gen):
    seqs, kind = _sequences(case), getattr(torch, case["dtype"])
    tokens, k, n, r, count = sum(m for m, _ in seqs), case["k"], case["n"], case["rank"], case["adapters"]
    x = _normal(gen, tokens, k, dtype=torch.float32)
    x *= 1.0 + 19.0 * (torch.rand(k, generator=gen, device=DEV) < 0.005)
    s = {"base": _normal(gen, tokens, n, dtype=torch.float32).to(kind), "x": x.to(kind),
         "a": torch.stack([(_normal(gen, r, k, dtype=torch.float32) * k ** -0.5).to(kind) for _ in range(count)]),
         "b": torch.stack([(_normal(gen, n, r, dtype=torch.float32) * r ** -0.5).to(kind) for _ in range(count)]),
         "scales": 0.25 + torch.rand(count, generator=gen, device=DEV), "seqs": seqs}
    if own:
        from kvmix_amd import ops

        s["plan"] = ops.adapter_plan([a for _, a in seqs], [m for m, _ in seqs], count, DEV)
    else:
        s["singles"] = torch.tensor([a for _, a in seqs[case["chunks"]:]], device=DEV)
    return s


def _prepare_beam(case, gen):
    R, W, V = case["requests"], case["beams"], case["vocab"]
    x = _normal(gen, R, W, V, dtype=torch.float32) * 2.5
    # the model has some idea of what comes next
    likely = torch.randint(0, V, (R, W, 8), generator=gen, device=DEV)
    x.scatter_add_(2, likely, 8.0 * torch.rand(R, W, 8, generator=gen, device=DEV))
    kind = getattr(torch, case["dtype"])
    if kind == torch.float32:
        x = x.half()  # what a head in 16 bits gives, as 32
    scores = -(torch.rand(R, W, generator=gen, device=DEV) * 6.0).sort(-1).values - 3.0
    s = {"logits": x.to(kind), "scores": scores, "done": None, "end": None}
    if case["ended"]:
        s["done"], s["end"] = torch.rand(R, W, generator=gen, device=DEV) < 0.25, 2
    return s


def _prepare_reorder(case, gen):
    R, W = case["requests"], case["beams"]
    B, H, D, T = R * W, case["kv_heads"], case["head_dim"], case["tokens"] // 32 * 32
    cap = -(-max(T, 1) // 352) * 352

    def random(*shape):
        return torch.randint(-2 ** 31, 2 ** 31 - 1, shape, generator=gen, device=DEV, dtype=torch.int32)

    tensors = []
    for _ in range(case["layers"]):
        kw, vw = case["k_bits"], D * case["v_bits"] // 32
        tensors.append(random(B, H, D, cap // 32 * kw)[..., :T // 32 * kw])
        tensors += [_normal(gen, B, H, D, cap // 32)[..., :T // 32] for _ in range(2)]
        tensors.append(random(B, H, cap, vw)[:, :, :T])
        tensors += [_normal(gen, B, H, cap, D // 32)[:, :, :T] for _ in range(2)]
        tensors += [_normal(gen, B, H, 2 * TAIL, D)[:, :, 3:3 + TAIL] for _ in range(2)]
    # half of a request's beams go on where they are, the others become copies of some of them
    keep = (W + 1) // 2
    index = torch.empty(R, W, dtype=torch.int64)
    for r in range(R):
        beams = torch.randperm(W, generator=gen, device=DEV).cpu()
        index[r, beams[:keep]], index[r, beams[keep:]] = beams[:keep], beams[:W - keep]
    return {"tensors": tensors, "index": (index + W * torch.arange(R)[:, None]).reshape(-1).to(DEV)}


# ---------------------------------------------------------------------------------------------------------------------
# the calls

def run(s):
    return globals()[("_own_" if own else "_plain_") + s["case"]["kind"]](s, s["case"])


def _own_rope(s, c):
    from kvmix_amd import ops

    q = ops.paged_rope_append(s["qkv"], s["cos"], s["sin"], s["rows"], s["plan"])
    return {"q": q, "rows": s["rows"]}


def _own_adapt(s, c):
    from kvmix_amd import ops

    return ops.add_adapters(s["base"], s["x"], s["a"], s["b"], s["plan"], s["scales"])


def _own_beam(s, c):
    from kvmix_amd import ops

    scores, parents, tokens = ops.beam_select(s["logits"], s["scores"], c["count"], s["done"], s["end"], c["stay"])
    return {"scores": scores, "parents": parents, "tokens": tokens}


def _own_reorder(s, c):
    from kvmix_amd import ops

    ops.reorder_rows(s["tensors"], s["index"])
    return s["tensors"]


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms

def _place(rows, slot, k, v, P):
    """Keys and values [tokens, heads, D] into their places of the fp16 pages."""
    page, at = slot // P, slot % P
    rows[page, :, 0, at] = k
    rows.view(rows.shape[0], rows.shape[1], 2, P // 32, rows.shape[4], 32)[page, :, 1, at // 32, :, at % 32] = v


def _plain_rope(s, c):
    nh, H, half = c["heads"], c["kv_heads"], c["head_dim"] // 2
    x = s["qkv"][:, :nh + H].float()
    turned = torch.cat([-x[..., half:], x[..., :half]], -1)
    x = (x * s["cos"].float()[:, None] + turned * s["sin"].float()[:, None]).half()
    _place(s["rows"], s["slot"], x[:, nh:], s["qkv"][:, nh + H:], c["page"])
    return {"q": x[:, :nh], "rows": s["rows"]}


def _plain_adapt(s, c):
    out, x, a, b, at = s["base"].float(), s["x"], s["a"], s["b"], 0
    for m, i in s["seqs"][:c["chunks"]]:
        if i >= 0:
            u = torch.matmul(x[at:at + m].float(), a[i].float().t())
            out[at:at + m] += s["scales"][i] * torch.matmul(u, b[i].float().t())
        at += m
    ids = s["singles"]
    if ids.numel():
        some = ids.clamp(min=0)
        u = torch.matmul(a[some].float(), x[at:].float()[:, :, None])
        more = torch.matmul(b[some].float(), u)[:, :, 0] * s["scales"][some][:, None]
        out[at:] += torch.where(ids[:, None] >= 0, more, torch.zeros_like(more))
    return out.to(s["base"].dtype)


def _plain_beam(s, c):
    R, W, V, C = c["requests"], c["beams"], c["vocab"], c["count"]
    x = s["logits"].float()
    top = x.amax(-1, keepdim=True)
    lse = (x - top).double().exp_().sum(-1, keepdim=True).log() + top.double()
    # of equal logits the one of the lowest index first: both in one 64-bit key
    bits = (x + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32 | (V - 1 - torch.arange(V, device=DEV))
    token = order.topk(C, dim=-1).indices
    score = s["scores"].double()[:, :, None] + (x.gather(2, token).double() - lse)
    if s["done"] is not None:  # a beam that has ended goes on as it is
        score = torch.where(s["done"][:, :, None], torch.full_like(score, -math.inf), score)
        score[:, :, 0] = torch.where(s["done"], s["scores"].double(), score[:, :, 0])
        token = token.masked_fill(s["done"][:, :, None], s["end"])
    score, at = score.reshape(R, W * C).sort(dim=-1, descending=True, stable=True)
    score, at = score[:, :C], at[:, :C]
    parent, token = at // C, token.reshape(R, W * C).gather(1, at)
    if c["stay"]:
        slot = _slots(parent)
        score, parent, token = (torch.empty_like(t).scatter_(1, slot, t) for t in (score, parent, token))
    return {"scores": score.float(), "parents": parent, "tokens": token}


def _slots(parent):
    """Where each child goes: the first of a beam takes its place, the others take those left free, in order."""
    C = parent.shape[1]
    first = ~((parent[:, :, None] == parent[:, None, :]) & torch.ones(C, C, dtype=torch.bool, device=DEV).tril(-1)).any(-1)
    taken = torch.zeros_like(first).scatter_(1, parent, True)
    free = taken.long().sort(dim=-1, stable=True).indices
    nth = (~first).long().cumsum(-1) - 1
    return torch.where(first, parent, free.gather(1, nth.clamp(min=0)))


def _plain_reorder(s, c):
    for t in s["tensors"]:
        t.copy_(t[s["index"]])
    return s["tensors"]


# ---------------------------------------------------------------------------------------------------------------------
# in 64 bits, from the definitions

def exact(case, seed):
    global own
    was, own = own, False
    try:
        s = prepare(case, seed)
    finally:
        own = was
    return globals()["_exact_" + case["kind"]](s, case)


def _exact_rope(s, c):
    nh, H, D, P = c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    z = torch.complex(s["qkv"][:, :nh + H, :D // 2].double(), s["qkv"][:, :nh + H, D // 2:].double())
    z = z * torch.complex(s["cos"][:, None, :D // 2].double(), s["sin"][:, None, :D // 2].double())
    x = torch.cat([z.real, z.imag], -1)
    rows = s["rows"].double()
    for h in range(H):
        flat = rows[:, h].reshape(-1, 2, P * D)
        place = s["slot"] % P
        page = (s["slot"] // P)[:, None]
        d = torch.arange(D, device=DEV)
        flat[page, 0, place[:, None] * D + d] = x[:, nh + h]
        flat[page, 1, (place // 32 * 32 * D)[:, None] + d * 32 + (place % 32)[:, None]] = s["qkv"][:, nh + H + h].double()
        rows[:, h] = flat.reshape(-1, 2, P, D)
    return {"q": x[:, :nh], "rows": rows}


def _exact_adapt(s, c):
    out, at = [], 0
    for m, i in s["seqs"]:
        y = s["base"][at:at + m].double()
        if i >= 0:
            y = y + s["scales"][i].double() * ((s["x"][at:at + m].double() @ s["a"][i].double().t()) @ s["b"][i].double().t())
        out.append(y)
        at += m
    return torch.cat(out)


def _exact_beam(s, c):
    R, W, V, C = c["requests"], c["beams"], c["vocab"], c["count"]
    scores = []
    for r in range(R):
        lp = torch.log_softmax(s["logits"][r].double(), -1) + s["scores"][r].double()[:, None]
        if s["done"] is not None:
            for w in range(W):
                if s["done"][r, w]:
                    lp[w] = -math.inf
                    lp[w, s["end"]] = s["scores"][r, w].double()
        best, at = lp.reshape(-1).sort(dim=0, descending=True, stable=True)
        best, parent = best[:C].tolist(), (at[:C] // V).tolist()
        if c["stay"]:
            row, free = [None] * C, [w for w in range(C) if w not in parent]
            for score, w in zip(best, parent):
                row[w if row[w] is None else free.pop(0)] = score
            best = row
        scores.append(best)
    return {"scores": torch.tensor(scores, dtype=torch.float64, device=DEV), "parents": None, "tokens": None}


def _exact_reorder(s, c):
    return None
