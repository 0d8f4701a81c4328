"""The operators of paged serving and scoring, as cases with sizes, for measuring them.

Four kinds of calls, through the public entry points only:

* ``store``   new tokens of many sequences go into their fp16 pages (``ops.paged_append``); pages that are full are quantized to
              packed pages (``ops.paged_quantize``) and read back as the values that they stand for (``ops.paged_read``);
* ``attend``  the newest tokens of every sequence, one or a chunk of them, attend over the sequence's pages, packed and fp16
              (``ops.paged_attention``);
* ``copy``    pages copied in the pools of all layers, as a fork or a compaction of sequences needs it (``ops.paged_copy``);
* ``score``   log probabilities of given tokens with the entropy and the most likely tokens, or with the gradient
              (``ops.token_logprobs``).

Pages hold P tokens of one layer, a multiple of 32.  A pool of fp16 pages is [pages, kv heads, 2, P, D]: the keys [P][D], and the
values as one [D][32] matrix for every 32 tokens.  A pool of packed pages is int32 [pages, kv heads, P / 32 blocks of words]; a
block holds 32 tokens: the codes of the keys and of the values, the keys' scales and minima (one per channel), the values'
(one per token and 32 channels, channels' groups outside).  Codes lie in the order of the lanes that use them: lane
g * 16 + m (g = 0..3) has, of the keys, channels 32 s + 8 g + j of token 8 (m / 4) + 4 u + m % 4 as piece u * D / 32 + s, and of
the values, token 8 g + j of channel 16 t + m as piece t, eight codes j to a piece.  A lane's codes fill D * bits / 64 words, two
at a time, the first of a pair in the low half of the word, and 32 / (2 bits) pairs to a word; with 3 bits five pairs, and the
pairs left over take the halves' top bits, one bit from each of three words.  Words lie in runs of 4, 2 or 1 per lane.

Keys have four channels per head ten times larger than the others, as real key caches do.  Without `own` the operators are
computed with elementary torch operations in 32 bits.
"""
from __future__ import annotations

import math

import numpy as np
import torch

own = False

DEV = "cuda"
WINDOW = 128  # tokens at least that a sequence keeps in fp16


# ---------------------------------------------------------------------------------------------------------------------
# the cases

def listed():
    return [
        # a step of a running batch: one new token for each of 64 sequences, and the four pages that it fills are quantized
        {"name": "store_b64_n1_h8_k4v4", "kind": "store", "batch": 64, "new": 1, "kv_heads": 8, "head_dim": 128, "page": 64,
         "full": 4, "k_bits": 4, "v_bits": 4},
        # chunks of prompts of odd length arrive, and the pages that they push out of the fp16 window are quantized
        {"name": "store_b8_n1021_h32_k3v2", "kind": "store", "batch": 8, "new": 1021, "kv_heads": 32, "head_dim": 128, "page": 64,
         "full": 120, "k_bits": 3, "v_bits": 2},
        # one user at 4k context: the smallest useful step, bound by latency
        {"name": "attend_b1_q1_t4096_k4v4", "kind": "attend", "batch": 1, "new": 1, "tokens": 4096, "heads": 32, "kv_heads": 32,
         "head_dim": 128, "page": 64, "k_bits": 4, "v_bits": 4},
        # a serving batch of sequences up to 8k, the lowest of the ordinary widths
        {"name": "attend_b16_q1_t8192_k2v2", "kind": "attend", "batch": 16, "new": 1, "tokens": 8192, "heads": 32, "kv_heads": 32,
         "head_dim": 128, "page": 64, "k_bits": 2, "v_bits": 2},
        # grouped-query heads at long context, 3-bit keys and 2-bit values
        {"name": "attend_gqa_b16_q1_t32768_k3v2", "kind": "attend", "batch": 16, "new": 1, "tokens": 32768, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 64, "k_bits": 3, "v_bits": 2},
        # short chunks of odd length over odd contexts: too few rows to fill the chip without splitting the keys
        {"name": "attend_gqa_b6_q101_t3001_k4v2", "kind": "attend", "batch": 6, "new": 101, "tokens": 3001, "heads": 32,
         "kv_heads": 8, "head_dim": 128, "page": 32, "k_bits": 4, "v_bits": 2},
        # long prompts in chunks, the fourth chunk of each: bound by the matrix cores
        {"name": "attend_b4_q2048_t8192_k4v4", "kind": "attend", "batch": 4, "new": 2048, "tokens": 8192, "heads": 32,
         "kv_heads": 32, "head_dim": 128, "page": 64, "k_bits": 4, "v_bits": 4},
        # eight sequences are forked: the page that each is writing, in all layers
        {"name": "copy_fork_l32_n8", "kind": "copy", "layers": 32, "pages": 8, "pool": 64, "kv_heads": 8, "head_dim": 128,
         "page": 64, "packed": False},
        # the packed pages of finished sequences' neighbours move down to the front of the pools of mixed widths
        {"name": "copy_compact_l32_n701", "kind": "copy", "layers": 32, "pages": 701, "pool": 1536, "kv_heads": 8, "head_dim": 128,
         "page": 64, "packed": True},
        # the sampled token of one sequence and its five best alternatives
        {"name": "score_n1_v32000_top5", "kind": "score", "rows": 1, "vocab": 32000, "top": 5, "dtype": "float16", "grad": False},
        # the texts of an evaluation: every token's likelihood, entropy and twenty best alternatives
        {"name": "score_n8192_v32000_top20", "kind": "score", "rows": 8192, "vocab": 32000, "top": 20, "dtype": "float16",
         "grad": False},
        # the likelihood as a loss over a batch of odd size, with its gradient
        {"name": "score_n4099_v32000_grad", "kind": "score", "rows": 4099, "vocab": 32000, "top": 0, "dtype": "bfloat16",
         "grad": True},
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["store", "attend", "attend", "attend", "copy", "score", "score"])
    heads, kv_heads = rng.choice([(32, 32), (32, 8), (32, 8), (16, 4), (12, 12), (8, 1)])
    dim = 128 if rng.random() < 0.8 else 64
    page = rng.choice([32, 64, 64, 128])
    kb, vb = rng.choice([1, 2, 3, 4]), rng.choice([1, 2, 3, 4])
    if kind == "store":
        new = _log_int(rng, 1, 1021)
        batch = max(1, min(_log_int(rng, 1, 128), 8168 * 32 // (new * kv_heads)))
        return {"kind": kind, "batch": batch, "new": new, "kv_heads": kv_heads, "head_dim": dim, "page": page,
                "full": max(1, min(batch * max(1, new // page), 120 * 32 * 64 // (kv_heads * page))), "k_bits": kb, "v_bits": vb}
    if kind == "attend":
        new = 1 if rng.random() < 0.5 else _log_int(rng, 2, 2048)
        tokens = max(_log_int(rng, 40, 32768), new)
        batch = max(1, min(_log_int(rng, 1, 32), 4194304 // (kv_heads * tokens), 2147483648 // (new * tokens * heads)))
        return {"kind": kind, "batch": batch, "new": new, "tokens": tokens, "heads": heads, "kv_heads": kv_heads,
                "head_dim": dim, "page": page, "k_bits": kb, "v_bits": vb}
    if kind == "copy":
        pages = max(1, _log_int(rng, 1, 700) * 64 * 8 // (page * max(kv_heads, 8)))
        return {"kind": kind, "layers": rng.randint(1, 32), "pages": pages, "pool": 2 * pages + rng.randint(1, 30),
                "kv_heads": kv_heads, "head_dim": dim, "page": page, "packed": pages > 200 or rng.random() < 0.5}
    vocab = 32000 if rng.random() < 0.5 else _log_int(rng, 300, 130000)
    rows = max(1, min(_log_int(rng, 1, 8192), 8192 * 32000 // vocab // 2))
    grad = rng.random() < 0.4
    return {"kind": kind, "rows": rows, "vocab": vocab, "top": 0 if grad else rng.choice([0, 1, 5, 20]),
            "dtype": rng.choice(["float16", "float16", "bfloat16", "float32"]), "grad": grad}


def _lengths(case):
    """Tokens of each sequence, newest included: the first has all, the others down to a third of them."""
    n, most, new = case["batch"], case["tokens"], case["new"]
    return [max(new, most - (most * 2 * i) // (3 * n)) for i in range(n)]


def _packed_lengths(case):
    """What of it is packed: whole pages, as long as the window and the new tokens stay in fp16."""
    return [max(0, n - case["new"] - WINDOW) // case["page"] * case["page"] for n in _lengths(case)]


def _pages(n, page):
    return -(-n // page)


def work(case):
    D = case.get("head_dim", 128)
    if case["kind"] == "store":
        new = case["batch"] * case["new"] * case["kv_heads"] * D * 2 * 2          # keys and values, fp16
        full = case["full"] * case["page"] * case["kv_heads"] * D * 2 * 2         # the pages read, and their values written
        packed = full // 32 * (case["k_bits"] + case["v_bits"] + 2)               # of 32 bits for a key and a value
        return {"bytes": 2 * new + 2 * full + 2 * packed, "flops": 8 * (full // 2)}
    if case["kind"] == "attend":
        token = case["kv_heads"] * D * 4                                          # bytes of a token in fp16
        lens, packed, new = _lengths(case), _packed_lengths(case), case["new"]
        cache = sum(p * token // 32 * (case["k_bits"] + case["v_bits"] + 2) + (n - p) * token for n, p in zip(lens, packed))
        pairs = sum(new * (n - new) + new * (new + 1) // 2 for n in lens)
        return {"bytes": cache + 2 * len(lens) * new * case["heads"] * D * 2, "flops": 4 * D * case["heads"] * pairs}
    if case["kind"] == "copy":
        row = case["page"] * case["kv_heads"] * D * 4
        per = [row // 32 * (a + b + 2) if case["packed"] else row for a, b in _layer_bits(case["layers"])]
        return {"bytes": 2 * case["pages"] * sum(per), "flops": 0}
    size = torch.empty((), dtype=getattr(torch, case["dtype"])).element_size()
    one = case["rows"] * case["vocab"] * size
    return {"bytes": (3 * one if case["grad"] else one) + case["rows"] * (16 + 12 * case["top"]),
            "flops": (9 if case["grad"] else 5) * case["rows"] * case["vocab"]}


# ---------------------------------------------------------------------------------------------------------------------
# inputs

def _generator(seed):
    return torch.Generator(device=DEV).manual_seed(seed)


def _normal(gen, *shape):
    return torch.randn(*shape, generator=gen, device=DEV, dtype=torch.float16)


def _outliers(gen, heads, dim):
    return 1.0 + 9.0 * (torch.rand(heads, dim, generator=gen, device=DEV).argsort(-1) < 4).half()


def _layer_bits(layers):
    """A quarter of the layers 4-bit, half 3-bit, a quarter 2-bit, keys and values in different orders."""
    cycle = [4, 3, 2, 3]
    return [(cycle[i % 4], cycle[(i + 2 * (i // 4) + 1) % 4]) for i in range(layers)]


def _quantize(x, dim, bits):
    """Codes (int64), scale and minimum (fp16) of groups of 32 along dim of x, which is 32 long there."""
    x = x.float()
    lo, hi = x.amin(dim, keepdim=True), x.amax(dim, keepdim=True)
    top = float(2 ** bits - 1)
    t = (x - lo) / ((hi - lo) / torch.full_like(lo, top))
    whole = t.floor()
    code = (whole + (t - whole >= 0.5)).nan_to_num(0.0).clamp(0.0, top)
    scale = (hi - lo) * torch.full_like(lo, 1.0 / top)
    return code.long(), scale.half().squeeze(dim), lo.half().squeeze(dim)


def _run_length(words):
    return 4 if words % 4 == 0 else 2 if words % 2 == 0 else 1


def _to_words(codes, bits):
    """[..., 64 lanes, pieces, 8] -> [..., words]"""
    lead, pairs = codes.shape[:-3], codes.shape[-2] * 4
    n = codes.shape[-2] * bits // 4
    c = codes.reshape(*lead, 64, pairs, 2)
    per = 5 if bits == 3 else 16 // bits
    at = bits * torch.arange(per, device=c.device)[:, None] + torch.tensor([0, 16], device=c.device)
    words = (c[..., :n * per, :].reshape(*lead, 64, n, per, 2) << at).sum((-2, -1))
    if bits == 3:
        left = c[..., n * per:, :].reshape(*lead, 64, n // 3, 1, 2) >> torch.arange(3, device=c.device)[:, None] & 1
        words = words + (left << torch.tensor([15, 31], device=c.device)).sum(-1).reshape(*lead, 64, n)
    w = _run_length(n)
    return words.reshape(*lead, 64, n // w, w).transpose(-3, -2).reshape(*lead, 64 * n).to(torch.int32)


def _pack_block(k, v, kb, vb):
    """k, v [..., 32, D] fp16 -> words [..., D * (kb + vb + 2)]"""
    lead, D = k.shape[:-2], k.shape[-1]
    kc, ks, kz = _quantize(k, -2, kb)
    vc, vs, vz = _quantize(v.reshape(*lead, 32, D // 32, 32), -1, vb)
    n = len(lead)
    kc = kc.reshape(*lead, 4, 2, 4, D // 32, 4, 8)  # token 8 a + 4 u + e, channel 32 s + 8 g + j
    kc = kc.permute(*range(n), n + 4, n + 0, n + 2, n + 1, n + 3, n + 5).reshape(*lead, 64, D // 16, 8)
    vc = vc.reshape(*lead, 4, 8, D // 16, 16)       # token 8 g + j, channel 16 t + m
    vc = vc.permute(*range(n), n + 0, n + 3, n + 2, n + 1).reshape(*lead, 64, D // 16, 8)
    sides = torch.cat([ks, kz, vs.transpose(-1, -2).flatten(-2), vz.transpose(-1, -2).flatten(-2)], -1)
    return torch.cat([_to_words(kc, kb), _to_words(vc, vb), sides.contiguous().view(torch.int32)], -1)


def _packed_pool(gen, pages, heads, page, dim, kb, vb):
    """A pool of packed pages of random tokens, some pages at a time."""
    blocks = page // 32
    pool = torch.empty(pages, heads, blocks, dim * (kb + vb + 2), device=DEV, dtype=torch.int32)
    scale = _outliers(gen, heads, dim)[:, None, None, :]
    some = max(1, (1 << 25) // (heads * page * dim))
    for i in range(0, pages, some):
        n = min(some, pages - i)
        pool[i:i + n] = _pack_block(_normal(gen, n, heads, blocks, 32, dim) * scale, _normal(gen, n, heads, blocks, 32, dim), kb, vb)
    return pool.reshape(pages, heads, blocks * dim * (kb + vb + 2))


def _rows_pool(gen, pages, heads, page, dim):
    pool = _normal(gen, pages, heads, 2, page, dim)
    pool[:, :, 0] *= _outliers(gen, heads, dim)[:, None, :]
    return pool


def _tables(gen, lens, packed, page):
    """Each sequence's pages, packed ones first, scattered over the pools: (table, packed pages, fp16 pages)."""
    np_, nr = [p // page for p in packed], [_pages(n, page) - p // page for n, p in zip(lens, packed)]
    one, two = torch.randperm(sum(np_), generator=gen, device=DEV).cpu(), torch.randperm(sum(nr), generator=gen, device=DEV).cpu()
    table = torch.full((len(lens), max(a + b for a, b in zip(np_, nr))), -1, dtype=torch.int32)
    i = j = 0
    for b, (p, r) in enumerate(zip(np_, nr)):
        table[b, :p], table[b, p:p + r] = one[i:i + p], two[j:j + r]
        i, j = i + p, j + r
    return table, sum(np_), sum(nr)


def prepare(case, seed):
    return {"case": case, **globals()["_prepare_" + case["kind"]](case, _generator(seed))}


def _plan(case, table, lens, packed, heads):
    """What a program makes once per step, for all layers."""
    from kvmix_amd import ops

    return ops.paged_plan(table, lens, packed, [case["new"]] * len(lens), heads, case["kv_heads"], case["head_dim"], case["page"], DEV)


def _prepare_store(case, gen):
    B, n, H, D, P = case["batch"], case["new"], case["kv_heads"], case["head_dim"], case["page"]
    # the sequences' fp16 pages before this call hold between 0 and P - 1 tokens of the page that is being written
    lens = [n + (7 * b + 5) % P for b in range(B)]
    table, _, pages = _tables(gen, lens, [0] * B, P)
    rows = _rows_pool(gen, pages + case["full"], H, P, D)  # behind them the pages that are full
    s = {"k": _normal(gen, B * n, H, D) * _outliers(gen, H, D), "v": _normal(gen, B * n, H, D), "rows": rows,
         "packed": torch.zeros(case["full"] + 3, H, P // 32 * D * (case["k_bits"] + case["v_bits"] + 2), dtype=torch.int32, device=DEV)}
    to = torch.randperm(case["full"] + 3, generator=gen, device=DEV).cpu()[:case["full"]]
    s["pairs"] = torch.stack([torch.arange(pages, pages + case["full"]), to], 1).to(torch.int32)
    if own:
        s["plan"] = _plan(case, table, lens, [0] * B, H)
    pos = torch.tensor([[m - n + i for i in range(n)] for m in lens])
    s["slot"] = (table.long().gather(1, pos // P) * P + pos % P).reshape(-1).to(DEV)
    s["src"] = s["pairs"][:, 0].long().to(DEV)
    return s


def _prepare_attend(case, gen):
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    lens, packed = _lengths(case), _packed_lengths(case)
    table, n_packed, n_rows = _tables(gen, lens, packed, P)
    s = {"q": _normal(gen, len(lens) * case["new"], case["heads"], D), "rows": _rows_pool(gen, n_rows, H, P, D),
         "packed": _packed_pool(gen, n_packed, H, P, D, case["k_bits"], case["v_bits"]),
         "table": table.to(DEV), "lens": torch.tensor(lens, device=DEV), "packed_lens": torch.tensor(packed, device=DEV)}
    if own:
        s["plan"] = _plan(case, table, lens, packed, case["heads"])
    return s


def _prepare_copy(case, gen):
    H, D, P = case["kv_heads"], case["head_dim"], case["page"]
    pools = []
    for kb, vb in _layer_bits(case["layers"]):
        if case["packed"]:
            words = P // 32 * D * (kb + vb + 2)
            pools.append(torch.randint(-2 ** 31, 2 ** 31 - 1, (case["pool"], H, words), generator=gen, device=DEV, dtype=torch.int32))
        else:
            pools.append(_rows_pool(gen, case["pool"], H, P, D))
    ids = torch.randperm(case["pool"], generator=gen, device=DEV).cpu()[:2 * case["pages"]]
    # compaction: from the back to the front
    src, dst = (ids.sort(descending=True).values if case["packed"] else ids).chunk(2)
    pairs = torch.stack([src, dst], 1).to(torch.int32).contiguous()
    return {"pools": pools, "pairs": pairs, "src": src.to(DEV), "dst": dst.to(DEV)}


def _prepare_score(case, gen):
    n, V = case["rows"], case["vocab"]
    x = torch.randn(n, V, generator=gen, device=DEV, dtype=torch.float32) * 2.5
    t = torch.randint(0, V, (n,), generator=gen, device=DEV)
    # the model has some idea of most tokens
    x.scatter_add_(1, t[:, None], 8.0 * torch.rand(n, 1, generator=gen, device=DEV))
    s = {"logits": x.to(getattr(torch, case["dtype"])), "targets": t}
    if case["grad"]:
        s["logits"].requires_grad_()
        s["weights"] = [torch.randn(n, generator=gen, device=DEV) for _ in range(2)]
    return s


# ---------------------------------------------------------------------------------------------------------------------
# the calls

def run(s):
    return globals()[("_own_" if own else "_plain_") + s["case"]["kind"]](s, s["case"])


def _own_store(s, c):
    from kvmix_amd import ops

    ops.paged_append(s["k"], s["v"], s["rows"], s["plan"])
    ops.paged_quantize(s["rows"], s["packed"], s["pairs"], c["k_bits"], c["v_bits"])
    k, v = ops.paged_read(s["packed"], s["pairs"][:, 1], c["k_bits"], c["v_bits"], c["head_dim"])
    return {"rows": s["rows"], "k": k, "v": v}


def _own_attend(s, c):
    from kvmix_amd import ops

    return ops.paged_attention(s["q"], s["rows"], s["packed"], s["plan"], c["k_bits"], c["v_bits"])


def _own_copy(s, c):
    from kvmix_amd import ops

    ops.paged_copy(s["pools"], s["pairs"])
    return s["pools"]


def _own_score(s, c):
    from kvmix_amd import ops

    out = ops.token_logprobs(s["logits"], s["targets"], top=c["top"])
    if not c["grad"]:
        return list(out)
    (grad,) = torch.autograd.grad(out[:2], s["logits"], s["weights"])
    return [out[0].detach(), out[1].detach(), grad]


# ---------------------------------------------------------------------------------------------------------------------
# the plain forms

def _from_words(words, pieces, bits):
    """[..., words] -> codes [..., 64 lanes, pieces, 8]"""
    lead, n = words.shape[:-1], pieces * bits // 4
    w = _run_length(n)
    words = words.reshape(*lead, n // w, 64, w).transpose(-3, -2).reshape(*lead, 64, n, 1, 1)
    per = 5 if bits == 3 else 16 // bits
    at = bits * torch.arange(per, device=words.device, dtype=torch.int32)[:, None] + torch.tensor([0, 16], device=words.device, dtype=torch.int32)
    codes = (words >> at & (1 << bits) - 1).reshape(*lead, 64, n * per, 2)
    if bits == 3:
        top = words.reshape(*lead, 64, n // 3, 3, 1) >> torch.tensor([15, 31], device=words.device, dtype=torch.int32) & 1
        codes = torch.cat([codes, top[..., 0, :] | top[..., 1, :] << 1 | top[..., 2, :] << 2], -2)
    return codes.reshape(*lead, 64, pieces, 8)


def _values(pages, D, kb, vb):
    """packed pages [n, heads, words] -> keys, values [n, P, heads, D] in 32 bits"""
    n, H, words = pages.shape
    blocks = words // (D * (kb + vb + 2))
    block = pages.reshape(n, H, blocks, D * (kb + vb + 2))
    codes_k, codes_v, sides = block.split([D * kb, D * vb, 2 * D], -1)
    ks, kz, vs, vz = sides.contiguous().view(torch.float16).float().split(D, -1)
    k = _from_words(codes_k, D // 16, kb).reshape(n, H, blocks, 4, 4, 4, 2, D // 32, 8)  # g a e u s j
    k = k.permute(0, 2, 4, 6, 5, 1, 7, 3, 8).reshape(n, blocks, 32, H, D).float()
    k = k * ks.transpose(1, 2)[:, :, None] + kz.transpose(1, 2)[:, :, None]
    v = _from_words(codes_v, D // 16, vb).reshape(n, H, blocks, 4, 16, D // 16, 8)       # g m t j
    v = v.permute(0, 2, 3, 6, 1, 5, 4).reshape(n, blocks, 32, H, D // 32, 32).float()
    vs, vz = (t.reshape(n, H, blocks, D // 32, 32).permute(0, 2, 4, 1, 3)[..., None] for t in (vs, vz))
    return k.reshape(n, 32 * blocks, H, D), (v * vs + vz).reshape(n, 32 * blocks, H, D)


def _of_rows(rows):
    """fp16 pages [n, heads, 2, P, D] -> keys, values [n, P, heads, D]"""
    n, H, _, P, D = rows.shape
    return rows[:, :, 0].transpose(1, 2), rows[:, :, 1].reshape(n, H, P // 32, D, 32).permute(0, 2, 4, 1, 3).reshape(n, P, H, D)


def _plain_store(s, c):
    rows, slot, P, D = s["rows"], s["slot"], c["page"], c["head_dim"]
    page, at = slot // P, slot % P
    rows[page, :, 0, at] = s["k"]
    rows.view(rows.shape[0], c["kv_heads"], 2, P // 32, D, 32)[page, :, 1, at // 32, :, at % 32] = s["v"]
    k, v = _of_rows(rows[s["src"]])
    n, H = k.shape[0], c["kv_heads"]
    kc, ks, kz = _quantize(k.reshape(n, P // 32, 32, H, D), 2, c["k_bits"])
    vc, vs, vz = _quantize(v.reshape(n, P, H, D // 32, 32), 4, c["v_bits"])
    k = (kc.float() * ks.float()[:, :, None] + kz.float()[:, :, None]).reshape(n, P, H, D)
    v = (vc.float() * vs.float()[..., None] + vz.float()[..., None]).reshape(n, P, H, D)
    return {"rows": rows, "k": k.half(), "v": v.half()}


def _plain_attend(s, c):
    B, n, nh, H, D, P = c["batch"], c["new"], c["heads"], c["kv_heads"], c["head_dim"], c["page"]
    table, lens = s["table"].long(), s["lens"]
    width = table.shape[1]
    nth = torch.arange(width, device=DEV)
    is_packed = nth < (s["packed_lens"] // P)[:, None]
    is_row = (nth * P < lens[:, None]) & ~is_packed
    k, v = (torch.zeros(B, width, P, H, D, device=DEV) for _ in range(2))
    k[is_packed], v[is_packed] = _values(s["packed"][table[is_packed]], D, c["k_bits"], c["v_bits"])
    kr, vr = _of_rows(s["rows"][table[is_row]])
    k[is_row], v[is_row] = kr.float(), vr.float()
    T = width * P
    at = torch.arange(T, device=DEV)
    v = v.reshape(B, T, H, D).masked_fill_((at >= lens[:, None])[..., None, None], 0.0)
    q = s["q"].float().reshape(B, n, H, nh // H, D).permute(0, 2, 3, 1, 4).reshape(B, H, nh // H * n, D)
    x = torch.matmul(q, k.reshape(B, T, H, D).permute(0, 2, 3, 1).contiguous()).mul_(D ** -0.5).view(B, H, nh // H, n, T)
    last = lens[:, None] - n + torch.arange(n, device=DEV)
    x.masked_fill_((at > last[..., None])[:, None, None], -math.inf)
    x.sub_(x.amax(-1, keepdim=True)).exp_()
    total = x.sum(-1, keepdim=True)
    o = torch.matmul(x.view(B, H, nh // H * n, T), v.permute(0, 2, 1, 3).contiguous()).view(B, H, nh // H, n, D) / total
    return o.permute(0, 3, 1, 2, 4).reshape(B * n, nh, D).half()


def _plain_copy(s, c):
    for pool in s["pools"]:
        pool[s["dst"]] = pool[s["src"]]
    return s["pools"]


def _plain_score(s, c):
    logits, t = s["logits"].detach(), s["targets"]
    x = logits.float()
    x = x - x.amax(-1, keepdim=True)
    e = x.exp()
    total = e.sum(-1, keepdim=True)
    lse = total.log()
    logprob = (x.gather(1, t[:, None]) - lse)[:, 0]
    entropy = (lse - (e * x).sum(-1, keepdim=True) / total)[:, 0]
    if c["grad"]:
        a, b = (w[:, None] for w in s["weights"])
        p = e / total
        grad = -p * (a + b * (x - lse + entropy[:, None]))
        grad.scatter_add_(1, t[:, None], a)
        return [logprob, entropy, grad.to(logits.dtype)]
    if not c["top"]:
        return [logprob, entropy]
    # of equal logits the one of the lowest index first: both in one 64-bit key
    bits = (logits.float() + 0.0).view(torch.int32).long()
    order = torch.where(bits < 0, bits ^ 0x7FFFFFFF, bits) << 32 | (c["vocab"] - 1 - torch.arange(c["vocab"], device=DEV))
    best = order.topk(c["top"], dim=-1).indices
    return [logprob, entropy, x.gather(1, best) - lse, best]


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


def _exact_store(s, c):
    P, D, H = c["page"], c["head_dim"], c["kv_heads"]
    if s["src"].numel() * P * H * D > 1 << 27:
        return None
    rows = s["rows"][s["src"]].cpu().numpy()

    def quantized(x, bits):  # groups along the last axis; the codes are defined by arithmetic in 32 bits
        x = x.astype(np.float32)
        lo, hi = x.min(-1, keepdims=True), x.max(-1, keepdims=True)
        top = np.float32(2 ** bits - 1)
        with np.errstate(invalid="ignore", divide="ignore"):
            t = np.nan_to_num((x - lo) / ((hi - lo) / top))
        code = np.clip(np.trunc(t.astype(np.float64) + 0.5), 0, 2 ** bits - 1)
        scale = ((hi - lo) * np.float32(np.float32(1) / top)).astype(np.float16)
        return torch.from_numpy(code * scale.astype(np.float64) + lo.astype(np.float16).astype(np.float64))

    n = rows.shape[0]
    k = quantized(np.ascontiguousarray(rows[:, :, 0].reshape(n, H, P // 32, 32, D).transpose(0, 2, 1, 4, 3)), c["k_bits"])
    v = quantized(np.ascontiguousarray(rows[:, :, 1].reshape(n, H, P // 32, D // 32, 32, 32).transpose(0, 2, 5, 1, 3, 4)), c["v_bits"])
    return {"rows": None, "k": k.permute(0, 1, 4, 2, 3).reshape(n, P, H, D), "v": v.reshape(n, P, H, D)}


def _places(D, bits, keys):
    """Where the code of (token, channel) lies in a block: its words [bits, 32, D] and the bit in each."""
    t, d = torch.meshgrid(torch.arange(32), torch.arange(D), indexing="ij")
    if keys:
        lane, piece, j = d % 32 // 8 * 16 + t // 8 * 4 + t % 4, t // 4 % 2 * (D // 32) + d // 32, d % 8
    else:
        lane, piece, j = t // 8 * 16 + d % 16, d // 16, t % 8
    n = D * bits // 64
    w = _run_length(n)
    pair, half, per = piece * 4 + j // 2, j % 2 * 16, 5 if bits == 3 else 16 // bits
    word, bit = [], []
    for i in range(bits):
        late = pair >= n * per
        nth = torch.where(late, 3 * (pair - n * per) + i, pair // per)
        word.append(nth // w * 64 * w + lane * w + nth % w)
        bit.append(torch.where(late, torch.tensor(15), pair % per * bits + i) + half)
    return torch.stack(word).to(DEV), torch.stack(bit).to(DEV)


def _exact_attend(s, c):
    n, nh, H, D, P, kb, vb = c["new"], c["heads"], c["kv_heads"], c["head_dim"], c["page"], c["k_bits"], c["v_bits"]
    places = [_places(D, kb, True), _places(D, vb, False)]
    group = torch.arange(D, device=DEV) // 32
    out = []
    for b, (length, packed) in enumerate(zip(_lengths(c), _packed_lengths(c))):
        ids = s["table"][b].long()
        block = s["packed"][ids[:packed // P]].transpose(0, 1).reshape(H, packed // 32, D * (kb + vb + 2))
        row = s["rows"][ids[packed // P:_pages(length, P)]].transpose(0, 1)
        o = []
        for h in range(H):
            sides = block[h, :, D * (kb + vb):].contiguous().view(torch.float16).double().reshape(-1, 4, D)
            codes = []
            for (word, bit), skip in zip(places, (0, D * kb)):
                codes.append(sum((block[h][:, skip + w] >> a & 1).double() * 2 ** i for i, (w, a) in enumerate(zip(word, bit))))
            vs, vz = (sides[:, i].reshape(-1, D // 32, 32).transpose(1, 2)[:, :, group] for i in (2, 3))
            k = torch.cat([(codes[0] * sides[:, 0, None] + sides[:, 1, None]).reshape(-1, D), row[h][:, 0].reshape(-1, D).double()])[:length]
            v = torch.cat([(codes[1] * vs + vz).reshape(-1, D),
                           row[h][:, 1].reshape(-1, D, 32).transpose(1, 2).reshape(-1, D).double()])[:length]
            for g in range(nh // H):
                x = s["q"][b * n:(b + 1) * n, h * (nh // H) + g].double() @ k.t() / math.sqrt(D)
                x.masked_fill_(torch.arange(length, device=DEV) > (length - n + torch.arange(n, device=DEV))[:, None], -math.inf)
                o.append(torch.softmax(x, -1) @ v)
        out.append(torch.stack(o, 1))
    return torch.cat(out)


def _exact_copy(s, c):
    return None


def _exact_score(s, c):
    x, t = s["logits"].detach().double(), s["targets"]
    lse = torch.logsumexp(x, -1, keepdim=True)
    lp = x - lse
    p = lp.exp()
    H = -(p * lp).sum(-1, keepdim=True)
    out = [lp[torch.arange(t.numel(), device=DEV), t], H[:, 0]]
    if c["grad"]:
        a, b = (w.double()[:, None] for w in s["weights"])
        hit = torch.arange(c["vocab"], device=DEV) == t[:, None]
        out.append(a * (hit.double() - p) - b * p * (lp + H))
    elif c["top"]:
        out += [lp.sort(-1, descending=True).values[:, :c["top"]], None]
    return out
