"""The decoder stack of kvmix_amd.decoder over a paged cache: sequences of different lengths in one batch, prompts in chunks
beside single tokens, forks of a sequence, and the likelihoods of texts.

    model = PagedDecoder(cfg, weights, k_bits, v_bits)
    a = model.add()
    logits = model.forward({a: prompt_ids})[a]               # of the last new token (every=True: of every one)
    answers = [a] + model.fork(a, 3)
    tokens = model.generate(answers, first_tokens, 64)        # greedy, all in one batch
    best, scores = model.beam_search([a], logits[None], 4, 64)  # four beams, the best first
    logprobs, entropy = model.score(text_ids, chunk=512)      # of every token of a text given those before it

With a pool of low-rank adapters (kvmix_amd.adapters.AdapterPool) every sequence may have one of its own, model.add(adapter=2).

It stands where the reference's evaluation scripts drive its models (pred_long_benchprofile.py:95-133, Inference-comparision.py:126-153).
"""
from __future__ import annotations

from typing import Dict, List, Optional, Sequence

import torch
import torch.nn.functional as F

from . import ops
from .adapters import AdapterPool
from .decoder import DecoderConfig, add_mlp, add_projection, check_beams, head_logits, rms_norm, rope_tables
from .paged import PagedKVCache


class PagedDecoder:
    """weights: the dict of decoder.init_weights.  k_bits, v_bits: widths per layer.  row_pages, packed_pages: see PagedKVCache.
    adapters: a pool of which every sequence may have one."""

    def __init__(self, cfg: DecoderConfig, weights: dict, k_bits: Sequence[int], v_bits: Sequence[int], row_pages: int = 256,
                 packed_pages: int = 1024, page_size: int = 64, window: int = 128, adapters: Optional[AdapterPool] = None):
        if adapters is not None:
            adapters.check(weights)
        self.cfg, self.w, self.adapters = cfg, weights, adapters
        self._adapter_of: Dict[int, int] = {}  # of the sequences that have one
        self.cache = PagedKVCache(k_bits, v_bits, cfg.num_heads, cfg.num_kv_heads, cfg.head_dim, row_pages, packed_pages, page_size, window,
                                  weights["embed"].device)

    def add(self, adapter: Optional[int] = None) -> int:
        if adapter is not None and (self.adapters is None or not 0 <= adapter < self.adapters.count):
            raise RuntimeError(f"no adapter {adapter} in this model's pool")
        s = self.cache.new()
        if adapter is not None:
            self._adapter_of[s] = adapter
        return s

    def fork(self, s: int, count: int = 1):
        made = self.cache.fork(s, count)
        if s in self._adapter_of:
            self._adapter_of.update((t, self._adapter_of[s]) for t in ([made] if count == 1 else made))
        return made

    def free(self, s: int) -> None:
        self.cache.free(s)
        self._adapter_of.pop(s, None)

    def _adapted_layer(self, layer: int, x: torch.Tensor, plan, attend):
        """A layer of a step in which sequences have adapters: the projections, each with what the adapters add to it."""
        lw, cfg, pool = self.w["layers"][layer], self.cfg, self.adapters
        h = rms_norm(x, lw["input_norm"], cfg.rms_norm_eps)
        out = attend(pool.add(F.linear(h, lw["wqkv"]), h, layer, "wqkv", plan))
        x = pool.add(add_projection(x, out, lw["wo"]), out, layer, "wo", plan)
        h = rms_norm(x, lw["post_norm"], cfg.rms_norm_eps)
        gate, up = pool.add(F.linear(h, lw["w_gate_up"]), h, layer, "w_gate_up", plan).chunk(2, -1)
        h = F.silu(gate) * up
        return pool.add(add_projection(x, h, lw["w_down"]), h, layer, "w_down", plan)

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
        cos, sin = (t[0, 0] for t in rope_tables(cfg, pos, x.dtype))
        nh, nkv = cfg.num_heads, cfg.num_kv_heads
        of = [self._adapter_of.get(s, -1) for s in new_ids]
        plan = ops.adapter_plan(of, [i.numel() for i in new_ids.values()], self.adapters.count, device) if max(of) >= 0 else None
        for layer, lw in enumerate(self.w["layers"]):
            def attend(qkv):
                q = cache.append_rotated(layer, step, qkv.view(-1, nh + 2 * nkv, cfg.head_dim), cos, sin, as_tensors=True)
                return cache.attend(layer, step, q).reshape(-1, 1, cfg.hidden_size)

            if plan is not None:
                x = self._adapted_layer(layer, x, plan, attend)
                continue
            out = attend(F.linear(rms_norm(x, lw["input_norm"], cfg.rms_norm_eps), lw["wqkv"]))
            x = add_projection(x, out, lw["wo"])
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

    def beam_search(self, sequences: Sequence[int], logits: torch.Tensor, beams: int, new_tokens: int, end: Optional[int] = None):
        """Beam search from sequences and the logits [n, vocab] of their last tokens: (token ids [n, beams, new_tokens], sums of
        their log probabilities [n, beams]), the best first.  A beam ends with the token `end`, which then fills it up.  The
        sequences stay as they are; the beams are forks of them, which share pages for as long as they agree, and end with the call."""
        if new_tokens < 1 or len(set(sequences)) != len(sequences) or logits.dim() != 2 or logits.shape[0] != len(sequences):
            raise RuntimeError("beam_search: a new token at least, sequences that are different, and a row of logits for each")
        check_beams(len(sequences), beams, end, logits.shape[1])
        for s in sequences:
            self.cache.length(s)  # (refuses what is no sequence)
        n, groups = len(sequences), []
        if not n:
            return logits.new_empty(0, beams, new_tokens, dtype=torch.int64), logits.new_empty(0, beams, dtype=torch.float32)
        logits = logits[:, None].expand(n, beams, logits.shape[-1])
        scores = torch.full((n, beams), float("-inf"), device=logits.device)
        scores[:, 0] = 0.0  # (the beams of a sequence are alike still)
        ids = torch.zeros(n * beams, new_tokens, dtype=torch.int64, device=logits.device)
        first, done = beams * torch.arange(n, device=logits.device)[:, None], None
        try:
            for step in range(new_tokens):
                scores, parents, tokens = ops.beam_select(logits, scores, beams, done, end, stay=True)
                ops.reorder_rows([ids], (first + parents).reshape(-1))
                ids[:, step] = tokens.reshape(-1)
                done = None if end is None else tokens == end
                if step + 1 == new_tokens:
                    break
                if not groups:
                    for s in sequences:
                        groups.append([])
                        for _ in range(beams):  # (one by one: what there are is known if the pages do not suffice)
                            groups[-1].append(self.fork(s))
                else:
                    for group, of in zip(groups, parents.tolist()):
                        self._replace(group, of)
                new = [s for group in groups for s in group]
                out = self.forward({s: tokens.view(-1)[i:i + 1] for i, s in enumerate(new)})
                logits = torch.stack([out[s] for s in new]).view(n, beams, -1)
        finally:
            for group in groups:
                for s in group:
                    if s is not None:
                        self.free(s)
        scores, order = scores.sort(dim=-1, descending=True, stable=True)
        return ids.view(n, beams, -1).gather(1, order[:, :, None].expand(-1, -1, new_tokens)), scores

    def _replace(self, group: List[int], parents: List[int]) -> None:
        """The beams of a sequence become those of their parents: where a beam is not its own, it has no children."""
        moved = [i for i, p in enumerate(parents) if i != p]
        for i in moved:
            self.free(group[i])
            group[i] = None
        for i in moved:
            group[i] = self.fork(group[parents[i]])

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
    answers from one prompt, beams, adapters, and what the quantized cache makes of a text's likelihoods."""
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
    some = list(texts)[:2]
    best, scores = timed("beams", len(some) * args.answers * args.new, lambda: model.beam_search(
        some, torch.stack([model.forward({s: texts[s][-1:]})[s] for s in some]), args.answers, args.new))
    print("best beams' log probabilities:", [round(float(x), 3) for x in scores[:, 0]])
    print("pages free (fp16, packed):", model.cache.free_pages())
    for s in answers:
        model.free(s)
    text = torch.cat([next(iter(texts.values())), ids[0]])
    lp, entropy = timed("likelihoods", text.numel() - 1, lambda: model.score(text, args.chunk))
    print(f"mean log probability {lp.mean():.4f}, mean entropy {entropy.mean():.4f}")
    pool = AdapterPool(cfg, 2, 16)
    for i in range(2):
        pool.load(i, {(layer, "wo"): (torch.randn(16, cfg.hidden_size, device="cuda") / 64, torch.randn(cfg.hidden_size, 16, device="cuda") / 4)
                      for layer in range(cfg.num_layers)}, scale=0.1)
    tuned = PagedDecoder(cfg, weights, bits, bits, adapters=pool)
    users = [tuned.add(), tuned.add(adapter=0), tuned.add(adapter=1)]
    prompt = next(iter(texts.values()))[:args.chunk]
    last = tuned.forward({s: prompt for s in users})
    ids = timed("answers with adapters", len(users) * (args.new - 1), lambda: tuned.generate(users, torch.stack([last[s].argmax() for s in users]), args.new))
    print("adapters' answers that differ from the plain one:", int((ids[1:] != ids[:1]).any(-1).sum()))


__all__ = ["PagedDecoder"]

if __name__ == "__main__":
    main()
