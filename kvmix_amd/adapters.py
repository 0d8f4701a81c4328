"""Low-rank adapters of the decoder's projections, many of them at once: every sequence of a batch may have its own.

    pool = AdapterPool(cfg, count=8, rank=16, device="cuda")
    pool.load(2, {(layer, "wo"): (a, b) for ...}, scale=alpha / rank)   # a [rank, k], b [n, rank] of the projection [n, k]
    model = PagedDecoder(cfg, weights, k_bits, v_bits, adapters=pool)
    s = model.add(adapter=2)

The adapters of one projection lie in one tensor for all of them, smaller ranks filled up with zeros, so that the tokens of a step
take one call per projection whichever adapters they have (ops.add_adapters).
"""
from __future__ import annotations

from typing import Dict, Sequence, Tuple

import torch

from . import ops
from .decoder import DecoderConfig

TARGETS = ("wqkv", "wo", "w_gate_up", "w_down")


class AdapterPool:
    """`count` adapters of rank `rank` at most (a multiple of 8 up to 128) for the projections `targets` of every layer, all
    zero until they are loaded.  Projections are the fused ones of decoder.init_weights: queries, keys and values; gate and up."""

    def __init__(self, cfg: DecoderConfig, count: int, rank: int, targets: Sequence[str] = TARGETS, dtype=torch.float16, device="cuda"):
        if count < 1 or rank < 8 or rank > 128 or rank % 8:
            raise RuntimeError("an adapter at least, and a rank that is a multiple of 8 up to 128")
        if not targets or any(t not in TARGETS for t in targets):
            raise RuntimeError(f"targets are some of {TARGETS}")
        h, i = cfg.hidden_size, cfg.intermediate_size
        shapes = {"wqkv": ((cfg.num_heads + 2 * cfg.num_kv_heads) * cfg.head_dim, h), "wo": (h, h), "w_gate_up": (2 * i, h), "w_down": (h, i)}
        if any(size % 8 for t in targets for size in shapes[t]):
            raise RuntimeError("the projections' sizes must be multiples of 8")
        self.count, self.rank, self.targets = count, rank, tuple(targets)
        self.scales = torch.ones(count, dtype=torch.float32, device=device)
        self._pool: Dict[Tuple[int, str], Tuple[torch.Tensor, torch.Tensor]] = {}
        for layer in range(cfg.num_layers):
            for t in self.targets:
                n, k = shapes[t]
                self._pool[layer, t] = (torch.zeros(count, rank, k, dtype=dtype, device=device), torch.zeros(count, n, rank, dtype=dtype, device=device))

    def check(self, weights: dict) -> None:
        """Refuses a decoder's weights (decoder.init_weights) that these adapters are not for: other layers, sizes, types or devices."""
        layers = {layer for layer, _ in self._pool}
        if len(layers) != len(weights["layers"]):
            raise RuntimeError(f"the adapters are for {len(layers)} layers, the weights have {len(weights['layers'])}")
        for (layer, t), (a, b) in self._pool.items():
            w = weights["layers"][layer][t]
            if tuple(w.shape) != (b.shape[1], a.shape[2]) or w.dtype != a.dtype or w.device != a.device:
                raise RuntimeError(f"the adapters' projection {(layer, t)} is [{b.shape[1]}, {a.shape[2]}], {a.dtype}, on {a.device}; the weights' "
                                   f"is {list(w.shape)}, {w.dtype}, on {w.device}")

    def load(self, i: int, weights: Dict[Tuple[int, str], Tuple[torch.Tensor, torch.Tensor]], scale: float = 1.0) -> None:
        """Adapter i becomes {(layer, projection): (a [r, k], b [n, r])}, r up to the pool's rank, times scale; zero elsewhere."""
        if not 0 <= i < self.count:
            raise RuntimeError(f"no adapter {i} in this pool")
        for at, (a, b) in weights.items():
            if at not in self._pool:
                raise RuntimeError(f"no projection {at} in this pool")
            k, n = self._pool[at][0].shape[2], self._pool[at][1].shape[1]
            if a.dim() != 2 or b.dim() != 2 or a.shape[1] != k or b.shape[0] != n or a.shape[0] != b.shape[1] or a.shape[0] > self.rank:
                raise RuntimeError(f"projection {at} takes a [r, {k}] and b [{n}, r], r up to {self.rank}")
        with torch.no_grad():
            for at, (a, b) in self._pool.items():
                a[i].zero_()
                b[i].zero_()
                if at in weights:
                    new_a, new_b = weights[at]
                    a[i, :new_a.shape[0]].copy_(new_a)
                    b[i, :, :new_b.shape[1]].copy_(new_b)
            self.scales[i] = scale

    def add(self, base: torch.Tensor, x: torch.Tensor, layer: int, target: str, plan) -> torch.Tensor:
        """What the tokens' adapters add to a projection's result `base` of the input x, into `base`, which is returned."""
        if (layer, target) not in self._pool:
            return base
        return ops.add_adapters(base, x, *self._pool[layer, target], plan, self.scales, out=base)


__all__ = ["AdapterPool", "TARGETS"]
