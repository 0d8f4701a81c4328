"""A plain implementation in 64 bits of what the paged operators compute, from the page layout as the header describes it."""
import math

import torch


def places(D, bits, keys):
    """Where the code of (token, channel) of a block lies among the words of its matrix: (word [bits, 32, D], bit [bits, 32, D])."""
    word, bit = torch.empty(bits, 32, D, dtype=torch.long), torch.empty(bits, 32, D, dtype=torch.long)
    n = D * bits // 64
    run = 4 if n % 4 == 0 else 2 if n % 2 == 0 else 1
    for t in range(32):
        for d in range(D):
            if keys:
                lane, piece, j = d % 32 // 8 * 16 + t // 8 * 4 + t % 4, t // 4 % 2 * (D // 32) + d // 32, d % 8
            else:
                lane, piece, j = t // 8 * 16 + d % 16, d // 16, t % 8
            pair, half = 4 * piece + j // 2, 16 * (j % 2)
            for i in range(bits):
                if bits == 3 and pair >= 5 * n:
                    w, b = 3 * (pair - 5 * n) + i, 15 + half
                else:
                    per = 5 if bits == 3 else 16 // bits
                    w, b = pair // per, pair % per * bits + i + half
                word[i, t, d], bit[i, t, d] = w // run * 64 * run + lane * run + w % run, b
    return word, bit


_places = {}


def unpack_pages(packed, D, kb, vb):
    """int32 packed pages [n, heads, words] -> keys, values [n, heads, P, D] in float64, on the CPU."""
    packed = packed.cpu()
    n, H, words = packed.shape
    blocks = words // (D * (kb + vb + 2))
    b = packed.reshape(n, H, blocks, D * (kb + vb + 2))
    halves = b[..., D * (kb + vb):].contiguous().view(torch.float16).double()  # [n, H, blocks, 4 D]
    codes = []
    for bits, keys, skip in ((kb, True, 0), (vb, False, D * kb)):
        if (D, bits, keys) not in _places:
            _places[D, bits, keys] = places(D, bits, keys)
        word, bit = _places[D, bits, keys]
        codes.append(sum(((b[..., skip + word[i]] >> bit[i]) & 1).double() * 2 ** i for i in range(bits)))
    ks, kz = halves[..., :D], halves[..., D:2 * D]
    vs, vz = (halves[..., i * D:(i + 1) * D].reshape(n, H, blocks, D // 32, 32).transpose(3, 4).repeat_interleave(32, -1) for i in (2, 3))
    k = codes[0] * ks[..., None, :] + kz[..., None, :]
    v = codes[1] * vs + vz
    return k.reshape(n, H, 32 * blocks, D), v.reshape(n, H, 32 * blocks, D)


def unpack_rows(rows):
    """fp16 pages [n, heads, 2, P, D] -> keys, values [n, heads, P, D] in float64, on the CPU."""
    rows = rows.cpu().double()
    n, H, _, P, D = rows.shape
    return rows[:, :, 0], rows[:, :, 1].reshape(n, H, P // 32, D, 32).transpose(3, 4).reshape(n, H, P, D)


class Batch:
    """Random pages for sequences of given lengths, with everything else in the pools poisoned."""

    def __init__(self, dev, lens, packed, new, heads, kv_heads, D, page, kb, vb, seed=0, poison=True, scale=1.0):
        from kvmix_amd import ops

        g = torch.Generator().manual_seed(seed)
        self.lens, self.packed_lens, self.new, self.heads, self.kv_heads, self.D, self.page, self.kb, self.vb = lens, packed, new, heads, kv_heads, D, page, kb, vb
        n_packed = [p // page for p in packed]
        n_rows = [-(-n // page) - p // page for n, p in zip(lens, packed)]
        spare = 3
        total_p, total_r = sum(n_packed) + spare, sum(n_rows) + spare
        ids_p, ids_r = torch.randperm(total_p, generator=g), torch.randperm(total_r, generator=g)
        width = max([a + b for a, b in zip(n_packed, n_rows)] + [1])
        self.table = torch.full((len(lens), width), -1, dtype=torch.int32)
        i = j = 0
        used = []
        for b, (p, r) in enumerate(zip(n_packed, n_rows)):
            self.table[b, :p], self.table[b, p:p + r] = ids_p[i:i + p], ids_r[j:j + r]
            used += [(int(ids_r[j + t]), min(page, lens[b] - packed[b] - t * page)) for t in range(r)]
            i, j = i + p, j + r
        bad = float("nan") if poison else 0.0
        self.rows = torch.full((total_r, kv_heads, 2, page, D), bad, dtype=torch.float16)
        out = 1.0 + 9.0 * (torch.rand(kv_heads, D, generator=g).argsort(-1) < 4)
        full = torch.randn(total_p, kv_heads, 2, page, D, generator=g) * scale
        full[:, :, 0] *= out[:, None, :]
        rows_of_packed = full.half()
        self.packed = torch.full((total_p, kv_heads, page // 32 * D * (kb + vb + 2)), -1, dtype=torch.int32, device=dev)
        if i:
            src = rows_of_packed.to(dev)
            pairs = torch.stack([ids_p[:i], ids_p[:i]], 1).to(torch.int32)
            ops.paged_quantize(src, self.packed, pairs, kb, vb)
        for r, n in used:
            k, v = torch.randn(kv_heads, n, D, generator=g) * out[:, None, :] * scale, torch.randn(kv_heads, n, D, generator=g) * scale
            self.rows[r, :, 0, :n] = k.half()
            view = self.rows[r, :, 1].view(kv_heads, page // 32, D, 32)
            for t in range(n):
                view[:, t // 32, :, t % 32] = v[:, t].half()
        self.rows = self.rows.to(dev)
        self.q = torch.randn(sum(new), heads, D, generator=g).half().to(dev)
        self.plan = ops.paged_plan(self.table, lens, packed, new, heads, kv_heads, D, page, dev)

    def dense(self, b):
        """keys, values [heads, tokens, D] of sequence b in float64"""
        P, n, p = self.page, self.lens[b], self.packed_lens[b] // self.page
        ids = self.table[b].long()
        pk, pv = unpack_pages(self.packed[ids[:p]], self.D, self.kb, self.vb) if p else (torch.zeros(0, self.kv_heads, P, self.D, dtype=torch.float64),) * 2
        rk, rv = unpack_rows(self.rows[ids[p:-(-n // P)]])
        return [torch.cat([a, c]).transpose(0, 1).reshape(self.kv_heads, -1, self.D)[:, :n] for a, c in ((pk, rk), (pv, rv))]

    def want(self, scale=None):
        """(outputs [tokens, heads, D] in float64, what they may be off by).

        The packed values are taken as fp16: a value is off by 2^-11 of itself (or half a smallest half, 2^-25), a logit of it
        by e = scale sum |q| |k| 2^-11 at most, of any key by the roundings of the sum in fp32 (D products, 2^-23 each of the
        absolute sum).  A probability is off by a factor exp(2 e) at most, rounds to fp16 (2^-11 of itself; 2^-25 of the
        largest where it is smaller than a normal half), the same for its part of the sum; exponentials and sums in fp32 are
        good to 2^-18 together; the result rounds to fp16."""
        scale = self.D ** -0.5 if scale is None else scale
        G, at, outs, tols = self.heads // self.kv_heads, 0, [], []
        q_all = self.q.cpu().double()
        for b, n in enumerate(self.new):
            if n == 0:
                continue
            k, v = self.dense(b)
            T = self.lens[b]
            q = q_all[at:at + n].reshape(n, self.kv_heads, G, self.D).permute(1, 2, 0, 3)  # [H, G, n, D]
            x = q @ k[:, None].transpose(-1, -2) * scale
            dead = torch.arange(T) > (T - n + torch.arange(n))[:, None]
            x = x.masked_fill(dead, -math.inf)
            p = torch.softmax(x, -1)
            o = p @ v[:, None]
            absx = q.abs() @ k[:, None].abs().transpose(-1, -2) * scale
            rounded = (torch.arange(T) < self.packed_lens[b]).double()
            e = absx * (2.0 ** -11 * rounded + self.D * 2.0 ** -23) + (q.abs().sum(-1, keepdim=True) * scale * 2.0 ** -25) * rounded
            e = e.masked_fill(dead, 0.0).amax(-1, keepdim=True)
            absv = p @ v[:, None].abs()
            vmax = v.abs().amax(1)[:, None, None]
            tol = (torch.exp(2 * e) - 1 + 2.0 ** -10 + 2.0 ** -11 + 2.0 ** -17) * absv + T * 2.0 ** -24 * vmax + 2.0 ** -11 * o.abs() + 2.0 ** -24
            outs.append(o.permute(2, 0, 1, 3).reshape(n, self.heads, self.D))
            tols.append(tol.permute(2, 0, 1, 3).reshape(n, self.heads, self.D))
            at += n
        return torch.cat(outs), torch.cat(tols)
