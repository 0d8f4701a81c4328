"""The decoder stack of kvmix_amd.decoder over a paged cache: sequences of different lengths in one batch, prompts in chunks
beside single tokens, forks of a sequence, and the likelihoods of texts.

    model = PagedDecoder(cfg, weights, k_bits, v_bits)
    a = model.add()
    logits = model.forward({a: prompt_ids})[a]               # of the last new token (every=True: of every one)
    answers = [a] + model.fork(a, 3)
    tokens = model.generate(answers, first_tokens, 64)        # greedy, all in one batch
    logprobs, entropy = model.score(text_ids, chunk=512)      # of every token of a text given those before it

It stands where the reference's evaluation scripts drive its models (pred_long_benchprofile.py:95-133, Inference-comparision.py:126-153).
"""
from __future__ import annotations

from typing import Dict, List, Sequence

import torch
import torch.nn.functional as F

from . import ops
from .decoder import DecoderConfig, add_mlp, add_projection, apply_rope, head_logits, rms_norm, rope_tables
from .paged import PagedKVCache


class PagedDecoder:
    """weights: the dict of decoder.init_weights.  k_bits, v_bits: widths per layer.  row_pages, packed_pages: see PagedKVCache."""

    def __init__(self, cfg: DecoderConfig, weights: dict, k_bits: Sequence[int], v_bits: Sequence[int], row_pages: int = 256,
                 packed_pages: int = 1024, page_size: int = 64, window: int = 128):
        self.cfg, self.w = cfg, weights
        self.cache = PagedKVCache(k_bits, v_bits, cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, row_pages, packed_pages, page_size, window,
                                  weights["embed"].device)

    def add(self) -> int:
        return self.cache.new()

    def fork(self, s: int, count: int = 1):
        return self.cache.fork(s, count)

    def free(self, s: int) -> None:
        self.cache.free(s)

    @torch.no_grad()
    def forward(self, new_ids: Dict[int, torch.Tensor], every: bool = False) -> Dict[int, torch.Tensor]:
        """New token ids [n] of some sequences -> their logits in fp32: [vocab] of the last new token, or with every=True
        [n, vocab]."""
        cfg, cache = self.cfg, self.cache
        new_ids = {s: ids.reshape(-1) for s, ids in new_ids.items() if ids.numel()}
        if not new_ids:
            return {}
        before = {s: cache.length(s) for s in new_ids}
        step = cache.step({s: ids.numel() for s, ids in new_ids.items()})
        device = self.w["embed"].device
        ids = torch.cat([ids.to(device) for ids in new_ids.values()])
        pos = torch.cat([torch.arange(before[s], before[s] + i.numel(), device=device) for s, i in new_ids.items()])
        x = self.w["embed"][ids][:, None]                       # [tokens, 1, hidden]: rows, as the projections' kernels take them
        cos, sin = (t[0, 0][:, None] for t in rope_tables(cfg, pos, x.dtype))
        nh, nkv = cfg.num_heads, cfg.num_kv_heads
        for layer, lw in enumerate(self.w["layers"]):
            qkv = F.linear(rms_norm(x, lw["input_norm"], cfg.rms_norm_eps), lw["wqkv"]).view(-1, nh + 2 * nkv, cfg.head_dim)
            qk = apply_rope(qkv[:, :nh + nkv], cos, sin)
            cache.append(layer, step, qk[:, nh:], qkv[:, nh + nkv:])
            out = cache.attend(layer, step, qk[:, :nh])
            x = add_projection(x, out.reshape(-1, 1, cfg.hidden_size), lw["wo"])
            x = add_mlp(x, lw, cfg.rms_norm_eps)
        spans = step.tokens()
        if not every:
            x = x[[spans[s].stop - 1 for s in new_ids]]
            logits = head_logits(x, self.w, cfg.rms_norm_eps)
            return {s: logits[i] for i, s in enumerate(new_ids)}
        logits = head_logits(x, self.w, cfg.rms_norm_eps)
        return {s: logits[spans[s]] for s in new_ids}

    def generate(self, sequences: Sequence[int], first: torch.Tensor, new_tokens: int, alternatives: int = 0):
        """Greedy decoding of several sequences at once, from their next tokens `first` [n]: the ids [n, new_tokens], `first`
        among them; with alternatives > 0 also the log probabilities and the ids of the most likely tokens at each step after it,
        [n, new_tokens - 1, alternatives] (none where there is no step after it)."""
        out: List[torch.Tensor] = [first.reshape(-1)]
        if new_tokens < 0 or len(set(sequences)) != len(sequences) or out[0].numel() != len(sequences):
            raise RuntimeError("generate: a number of tokens that is not negative, sequences that are different, and one first token for each")
        best = []
        for _ in range(new_tokens - 1 if len(sequences) else 0):
            logits = self.forward({s: out[-1][i:i + 1] for i, s in enumerate(sequences)})
            stacked = torch.stack([logits[s] for s in sequences])
            _, _, top_logprob, top_id = ops.token_logprobs(stacked, out[-1], top=max(alternatives, 1))
            out.append(top_id[:, 0])
            best.append((top_logprob, top_id))
        ids = torch.stack(out, 1)[:, :new_tokens] if len(sequences) else out[0].new_empty(0, new_tokens)
        if not alternatives:
            return ids
        if not best:
            empty = ids.new_empty(len(sequences), max(new_tokens - 1, 0), alternatives)
            return ids, empty.float(), empty
        return ids, *(torch.stack([b[i] for b in best], 1) for i in range(2))

    def score(self, ids: torch.Tensor, chunk: int = 512):
        """(log probabilities, entropies) [len(ids) - 1] of the tokens of a text after its first, each given those before it, read
        through the quantized cache in chunks."""
        if chunk <= 0:
            raise RuntimeError("score: a chunk has at least one token")
        ids = ids.reshape(-1).to(self.w["embed"].device)
        s = self.add()
        lp, entropy = [], []
        try:
            for at in range(0, ids.numel() - 1, chunk):
                part = ids[at:min(at + chunk, ids.numel() - 1)]
                logits = self.forward({s: part}, every=True)[s]
                a, b = ops.token_logprobs(logits, ids[at + 1:at + 1 + part.numel()])
                lp.append(a)
                entropy.append(b)
        finally:
            self.free(s)
        if not lp:
            return tuple(torch.empty(0, device=ids.device) for _ in range(2))
        return torch.cat(lp), torch.cat(entropy)


def main() -> None:
    """A server in small, on random weights: prompts that arrive in chunks beside sequences that are being answered, several
    answers from one prompt, and what the quantized cache makes of a text's likelihoods."""
    import argparse
    import time

    from .decoder import init_weights

    ap = argparse.ArgumentParser(description=main.__doc__)
    ap.add_argument("--layers", type=int, default=8)
    ap.add_argument("--kv-heads", type=int, default=8)
    ap.add_argument("--prompts", type=int, default=8)
    ap.add_argument("--prompt", type=int, default=2000, help="tokens of the longest prompt")
    ap.add_argument("--chunk", type=int, default=512)
    ap.add_argument("--answers", type=int, default=4, help="sequences forked from each prompt")
    ap.add_argument("--new", type=int, default=32, help="tokens of each answer")
    ap.add_argument("--bits", type=int, default=4)
    args = ap.parse_args()
    cfg = DecoderConfig(num_layers=args.layers, num_kv_heads=args.kv_heads)
    weights = init_weights(cfg, "cuda")
    bits = [args.bits] * args.layers
    pages = args.prompts * args.answers * 8
    model = PagedDecoder(cfg, weights, bits, bits, row_pages=pages + args.prompts * (args.prompt // 64 + 2),
                         packed_pages=args.prompts * (args.prompt // 64 + args.answers * (args.new // 64 + 4)))
    lens = [max(1, args.prompt - i * args.prompt // (2 * args.prompts)) for i in range(args.prompts)]
    texts = {model.add(): torch.randint(0, cfg.vocab_size, (n,), device="cuda") for n in lens}

    def timed(what, count, f):
        torch.cuda.synchronize()
        t = time.perf_counter()
        r = f()
        torch.cuda.synchronize()
        print(f"{what}: {count} tokens, {count / (time.perf_counter() - t):.0f} tokens/s", flush=True)
        return r

    def read_prompts():
        last, at = {}, 0
        while any(at < t.numel() for t in texts.values()):
            last.update(model.forward({s: t[at:at + args.chunk] for s, t in texts.items()}))
            at += args.chunk
        return last

    last = timed("prompts in chunks", sum(lens), read_prompts)
    answers, first = [], []
    for s in texts:
        twins = [s] + [model.fork(s) for _ in range(args.answers - 1)]
        answers += twins
        _, _, _, top = ops.token_logprobs(last[s], last[s].argmax(), top=args.answers)  # each answer begins with another token
        first += list(top)
    ids = timed("answers", len(answers) * (args.new - 1), lambda: model.generate(answers, torch.stack(first), args.new))
    print("pages free (fp16, packed):", model.cache.free_pages())
    for s in answers:
        model.free(s)
    text = torch.cat([next(iter(texts.values())), ids[0]])
    lp, entropy = timed("likelihoods", text.numel() - 1, lambda: model.score(text, args.chunk))
    print(f"mean log probability {lp.mean():.4f}, mean entropy {entropy.mean():.4f}")


__all__ = ["PagedDecoder"]

if __name__ == "__main__":
    main()
