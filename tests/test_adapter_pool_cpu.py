"""Pools of adapters and the weights that they are for.  No GPU."""
import pytest
import torch

from kvmix_amd.adapters import AdapterPool
from kvmix_amd.decoder import DecoderConfig, init_weights


def config(**kw):
    return DecoderConfig(**{**dict(hidden_size=64, num_layers=3, num_heads=2, num_kv_heads=1, intermediate_size=96, vocab_size=50), **kw})


def test_pools_of_other_weights():
    """Fewer layers would leave the others without their adapters, other types or devices would be refused in the midst of a step."""
    w = init_weights(config(), "cpu")
    for targets in (("wo",), ("wqkv", "w_down"), ("wqkv", "wo", "w_gate_up", "w_down")):
        AdapterPool(config(), 2, 8, targets, device="cpu").check(w)
    for pool, match in [
        (AdapterPool(config(num_layers=2), 2, 8, device="cpu"), "2 layers"), (AdapterPool(config(num_layers=4), 2, 8, device="cpu"), "4 layers"),
        (AdapterPool(config(hidden_size=128), 2, 8, device="cpu"), "projection"), (AdapterPool(config(num_kv_heads=2), 2, 8, device="cpu"), "wqkv"),
        (AdapterPool(config(intermediate_size=104), 2, 8, ("w_down",), device="cpu"), "w_down"),
        (AdapterPool(config(), 2, 8, dtype=torch.bfloat16, device="cpu"), "bfloat16"), (AdapterPool(config(), 2, 8, device="meta"), "meta"),
    ]:
        with pytest.raises(RuntimeError, match=match):
            pool.check(w)


def test_a_decoder_asks():
    """(before it makes its cache, which needs a GPU)"""
    from kvmix_amd.paged_decoder import PagedDecoder

    w = init_weights(config(hidden_size=128), "cpu")
    with pytest.raises(RuntimeError, match="2 layers"):
        PagedDecoder(config(hidden_size=128), w, [4] * 3, [4] * 3, adapters=AdapterPool(config(hidden_size=128, num_layers=2), 2, 8, device="cpu"))
