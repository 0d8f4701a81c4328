"""A quantized KV cache in pages: many sequences of different lengths that come and go, grow by single tokens or by chunks, and
share what they have in common.

The reference's cache (models/modeling_llama_KVmix.py:107-167) is one batch whose sequences have the same length; it grows by
concatenation.  Here the tokens of all sequences lie in pages of pools that are allocated once: a sequence's oldest pages packed
(codes of 1 to 4 bits per layer, fp16 scales and minima, the reference's quantizer in groups of 32), its newest in fp16, at
least `window` tokens of them.  A page is packed as a whole once it has left the window.  All layers use the same page numbers, so
that one table per sequence serves all of them; a packed page never changes and is shared by the sequences forked from one
another, as is every full fp16 page: the first of them that packs such a page does it for all.

    cache = PagedKVCache(k_bits, v_bits, heads=32, kv_heads=8, head_dim=128, row_pages=256, packed_pages=4096)
    a = cache.new()
    step = cache.step({a: 700})                       # room for 700 new tokens of `a`; pages that left the window are packed
    for layer in range(layers):
        cache.append(layer, step, k, v)               # k, v [700, kv_heads, head_dim]
        out = cache.attend(layer, step, q)            # q [700, heads, head_dim]
    b = cache.fork(a)                                 # shares a's pages, but for the one that is being written
    cache.free(a)
    cache.compact()                                   # what is left moves to the front of the pools

The numbers of pages are kept on the host; nothing here waits for the GPU.
"""
from __future__ import annotations

import weakref
from dataclasses import dataclass, field
from typing import Dict, List, Sequence

import torch

from . import ops


class OutOfPages(RuntimeError):
    """The pools do not hold what a call asks for; the cache is as it was before the call."""


class _Pages:
    """Numbers of a pool's pages: which are in use, and by how many sequences."""

    def __init__(self, count: int):
        self.users = [0] * count
        self.free = list(range(count - 1, -1, -1))

    def take(self) -> int:
        page = self.free.pop()
        self.users[page] = 1
        return page

    def share(self, page: int) -> None:
        self.users[page] += 1

    def drop(self, page: int) -> None:
        self.users[page] -= 1
        if self.users[page] == 0:
            self.free.append(page)

    def compacted(self) -> dict:
        """Moves {page: new page} that bring the pages in use to the front; the numbers are as after the moves."""
        used = len(self.users) - len(self.free)
        holes = [p for p in range(used) if self.users[p] == 0]
        moves = dict(zip((p for p in range(used, len(self.users)) if self.users[p]), holes))
        for old, new in moves.items():
            self.users[new], self.users[old] = self.users[old], 0
        self.free = list(range(len(self.users) - 1, used - 1, -1))
        return moves


@dataclass
class _Sequence:
    length: int = 0
    packed: List[int] = field(default_factory=list)  # packed pages, oldest first
    rows: List[int] = field(default_factory=list)    # the fp16 pages after them


@dataclass(eq=False)
class Step:
    """What PagedKVCache.step returns: the plan that append and attend of every layer use, and where each sequence's new tokens
    lie among those of the step.  It serves until one of its sequences takes another step or ends, or pages move."""
    plan: object
    sequences: List[int]
    counts: List[int]
    cache: object = field(default=None, repr=False)
    over: bool = False

    def tokens(self) -> Dict[int, slice]:
        out, at = {}, 0
        for s, n in zip(self.sequences, self.counts):
            out[s] = slice(at, at + n)
            at += n
        return out


class PagedKVCache:
    def __init__(self, k_bits: Sequence[int], v_bits: Sequence[int], heads: int, kv_heads: int, head_dim: int, row_pages: int,
                 packed_pages: int, page_size: int = 64, window: int = 128, device="cuda"):
        """k_bits, v_bits: widths per layer.  row_pages, packed_pages: pages of the pools, for all sequences together."""
        if len(k_bits) != len(v_bits) or not k_bits:
            raise RuntimeError("k_bits and v_bits: one width per layer each")
        for bits in (*k_bits, *v_bits):
            ops._check_bits(bits)
        if page_size < 32 or page_size > 1024 or page_size & (page_size - 1):
            raise RuntimeError("page_size must be 32, 64, 128, 256, 512 or 1024")
        if head_dim not in (64, 128):
            raise RuntimeError("head_dim must be 64 or 128")
        if kv_heads <= 0 or heads <= 0 or heads % kv_heads:
            raise RuntimeError("Total heads must be divisible by KV heads")
        if window < 0 or row_pages <= 0 or packed_pages < 0:
            raise RuntimeError("window and the numbers of pages must not be negative")
        self.k_bits, self.v_bits = list(k_bits), list(v_bits)
        self.heads, self.kv_heads, self.head_dim, self.page_size, self.window = heads, kv_heads, head_dim, page_size, window
        self.device = ops._cuda(device)
        self.rows = [torch.zeros(row_pages, kv_heads, 2, page_size, head_dim, dtype=torch.float16, device=self.device) for _ in k_bits]
        self.packed = [torch.zeros(packed_pages, kv_heads, page_size // 32 * head_dim * (kb + vb + 2), dtype=torch.int32, device=self.device)
                       for kb, vb in zip(k_bits, v_bits)]
        self._row_pages, self._packed_pages = _Pages(row_pages), _Pages(packed_pages)
        self._packed_as: Dict[int, int] = {}  # fp16 pages still in use -> the packed page made of them, in use too
        self._made_of: Dict[int, int] = {}    # the other way round
        self._sequences: Dict[int, _Sequence] = {}
        self._next = 0
        self._steps: Dict[int, weakref.ref] = {}  # the latest step of each sequence

    # -- sequences ---------------------------------------------------------------------------
    def new(self) -> int:
        self._sequences[self._next] = _Sequence()
        self._next += 1
        return self._next - 1

    def _sequence(self, s: int) -> _Sequence:
        if s not in self._sequences:
            raise RuntimeError(f"no sequence {s} in this cache")
        return self._sequences[s]

    def length(self, s: int) -> int:
        return self._sequence(s).length

    def free_pages(self):
        """(fp16 pages, packed pages) that no sequence uses"""
        return len(self._row_pages.free), len(self._packed_pages.free)

    def fork(self, s: int, count: int = 1):
        """`count` new sequences with the tokens of `s` (the one sequence's number for a count of 1, else a list).  Pages are
        shared; the one that is not full yet is copied, in all layers with one call (so the tokens of the latest step are appended
        before)."""
        old, P = self._sequence(s), self.page_size
        partial = old.length % P != 0
        if count < 1:
            raise RuntimeError("fork: at least one new sequence")
        if partial and len(self._row_pages.free) < count:
            raise OutOfPages(f"fork needs {count} fp16 pages, {len(self._row_pages.free)} are free")
        made, pairs = [], []
        for _ in range(count):
            n = self.new()
            twin = self._sequences[n]
            twin.length, twin.packed, twin.rows = old.length, list(old.packed), list(old.rows)
            for p in twin.packed:
                self._packed_pages.share(p)
            if partial:
                page = self._row_pages.take()
                pairs.append((twin.rows[-1], page))
                twin.rows[-1] = page
            for p in twin.rows[:-1] if partial else twin.rows:
                self._row_pages.share(p)
            made.append(n)
        if pairs:
            ops.paged_copy(self.rows, torch.tensor(pairs, dtype=torch.int32))
        return made[0] if count == 1 else made

    def free(self, s: int) -> None:
        """Ends a sequence: pages that no other one uses can be taken again."""
        old = self._sequence(s)
        self._end_steps([s])
        del self._sequences[s]
        for p in old.packed:
            self._drop_packed(p)
        for p in old.rows:
            self._drop_row(p)

    def _end_steps(self, sequences) -> None:
        """The plans of these sequences' steps name pages that are written, given away or moved from now on."""
        for s in sequences:
            step = self._steps.pop(s, lambda: None)()
            if step is not None:
                step.over = True

    def _drop_row(self, page: int) -> None:
        self._row_pages.drop(page)
        if not self._row_pages.users[page] and page in self._packed_as:
            del self._made_of[self._packed_as.pop(page)]

    def _drop_packed(self, page: int) -> None:
        self._packed_pages.drop(page)
        if not self._packed_pages.users[page] and page in self._made_of:
            del self._packed_as[self._made_of.pop(page)]

    def compact(self) -> int:
        """Moves the pages in use to the front of the pools, all layers with one call per kind of page (what lies behind them
        can then be given to something else); returns the number of pages moved."""
        moved = 0
        for pages, pools, of in ((self._row_pages, self.rows, "rows"), (self._packed_pages, self.packed, "packed")):
            moves = pages.compacted()
            if not moves:
                continue
            ops.paged_copy(pools, torch.tensor(list(moves.items()), dtype=torch.int32))
            for seq in self._sequences.values():
                setattr(seq, of, [moves.get(p, p) for p in getattr(seq, of)])
            if of == "rows":
                self._packed_as = {moves.get(r, r): p for r, p in self._packed_as.items()}
            else:
                self._packed_as = {r: moves.get(p, p) for r, p in self._packed_as.items()}
            self._made_of = {p: r for r, p in self._packed_as.items()}
            moved += len(moves)
        if moved:
            self._end_steps(list(self._steps))
        return moved

    # -- steps -------------------------------------------------------------------------------
    def _leaves_window(self, seq: _Sequence) -> int:
        """fp16 pages at the front of a sequence that hold none of its newest `window` tokens"""
        return max(0, min((seq.length - self.window) // self.page_size - len(seq.packed), len(seq.rows)))

    def step(self, new_tokens: Dict[int, int]) -> Step:
        """Room for new tokens {sequence: how many}, and the plan of the step.  Pages whose tokens have all left the window
        are packed first, in all layers."""
        P = self.page_size
        seqs = [(s, self._sequence(s), int(n)) for s, n in new_tokens.items()]
        if any(n < 0 for _, _, n in seqs):
            raise RuntimeError("step: a negative number of new tokens")
        if self.device.type == "cuda" and torch.cuda.is_current_stream_capturing():
            raise RuntimeError("step: pages are not taken while a graph is captured")
        flush = [(seq, self._leaves_window(seq)) for _, seq, _ in seqs]
        need_packed = len({page for seq, n in flush for page in seq.rows[:n]} - self._packed_as.keys())
        need_rows = sum(-(-(seq.length + n) // P) - len(seq.packed) - len(seq.rows) for _, seq, n in seqs)
        gained = self._freed(flush)
        if need_packed > len(self._packed_pages.free) or need_rows > len(self._row_pages.free) + gained:
            raise OutOfPages(f"step needs {need_packed} packed and {need_rows} fp16 pages; {len(self._packed_pages.free)} and "
                             f"{len(self._row_pages.free) + gained} can be had")
        self._end_steps([s for s, _, _ in seqs])
        pairs = []
        for seq, n in flush:
            for page in seq.rows[:n]:
                to = self._packed_as.get(page)
                if to is None:
                    to = self._packed_pages.take()
                    pairs.append((page, to))
                    self._packed_as[page], self._made_of[to] = to, page
                else:  # (by a fork before, or in this step)
                    self._packed_pages.share(to)
                seq.packed.append(to)
        if pairs:
            listed = torch.tensor(pairs, dtype=torch.int32)
            for layer, (kb, vb) in enumerate(zip(self.k_bits, self.v_bits)):
                ops.paged_quantize(self.rows[layer], self.packed[layer], listed, kb, vb)
        for seq, n in flush:
            for page in seq.rows[:n]:
                self._drop_row(page)
            del seq.rows[:n]
        for _, seq, n in seqs:
            seq.length += n
            while (len(seq.packed) + len(seq.rows)) * P < seq.length:
                seq.rows.append(self._row_pages.take())
        return self._planned(seqs)

    def _freed(self, flush) -> int:
        """fp16 pages that packing these frees: those that no other sequence uses as well"""
        drops: Dict[int, int] = {}
        for seq, n in flush:
            for page in seq.rows[:n]:
                drops[page] = drops.get(page, 0) + 1
        return sum(self._row_pages.users[p] == n for p, n in drops.items())

    def _planned(self, seqs) -> Step:
        P = self.page_size
        width = max([len(seq.packed) + len(seq.rows) for _, seq, _ in seqs] + [1])
        table = torch.full((len(seqs), width), -1, dtype=torch.int32)
        for i, (_, seq, _) in enumerate(seqs):
            pages = seq.packed + seq.rows
            table[i, :len(pages)] = torch.tensor(pages, dtype=torch.int32)
        plan = ops.paged_plan(table, [seq.length for _, seq, _ in seqs], [len(seq.packed) * P for _, seq, _ in seqs], [n for _, _, n in seqs],
                              self.heads, self.kv_heads, self.head_dim, P, self.device)
        step = Step(plan, [s for s, _, _ in seqs], [n for _, _, n in seqs], self)
        self._steps.update((s, weakref.ref(step)) for s, _, _ in seqs)
        return step

    # -- what a layer does in a step ---------------------------------------------------------
    def _plan(self, step: Step):
        if step.cache is not self:
            raise RuntimeError("this step is of another cache")
        if step.over:
            raise RuntimeError("this step is over: a sequence of it has taken another one or ended, or its pages have moved")
        return step.plan

    def append(self, layer: int, step: Step, k: torch.Tensor, v: torch.Tensor) -> None:
        """The new tokens' keys and values [tokens, kv_heads, head_dim], sequence after sequence."""
        ops.paged_append(k, v, self.rows[layer], self._plan(step))

    def attend(self, layer: int, step: Step, q: torch.Tensor, scale: float = None) -> torch.Tensor:
        """Attention of the new tokens' queries [tokens, heads, head_dim] over their sequences, themselves included."""
        return ops.paged_attention(q, self.rows[layer], self.packed[layer], self._plan(step), self.k_bits[layer], self.v_bits[layer], scale)

    def read(self, layer: int, s: int):
        """Keys and values [length, kv_heads, head_dim] of a sequence as the cache holds them, in fp16."""
        seq = self._sequence(s)
        parts = []
        if seq.packed:
            parts.append(ops.paged_read(self.packed[layer], torch.tensor(seq.packed, dtype=torch.int32), self.k_bits[layer], self.v_bits[layer], self.head_dim))
        if seq.rows:
            parts.append(ops.paged_read(self.rows[layer], torch.tensor(seq.rows, dtype=torch.int32)))
        if not parts:
            return tuple(torch.empty(0, self.kv_heads, self.head_dim, dtype=torch.float16, device=self.device) for _ in range(2))
        return tuple(torch.cat([p[i] for p in parts]).flatten(0, 1)[:seq.length] for i in range(2))


__all__ = ["OutOfPages", "PagedKVCache", "Step"]
