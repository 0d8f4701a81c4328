"""Sizes that a launch over pages cannot have: refused when the plan is made.  No GPU."""
import ctypes

import pytest

from kvmix_amd import _lib


def plan_of(sequences, new, heads, page=64):
    """kvmix_paged_plan of equal sequences of `new` tokens in the same page: (code, plan)"""
    n = (ctypes.c_int64 * sequences)
    batch, plan = _lib.PagedBatch(), _lib.PagedPlan()
    pages, lens, packed = (ctypes.c_int32 * sequences)(), n(*[new] * sequences), n()
    batch.table, batch.table_stride = ctypes.addressof(pages), 1
    batch.kv_lens = batch.q_lens = ctypes.addressof(lens)
    batch.packed_lens = ctypes.addressof(packed)
    batch.sequences, batch.heads, batch.kv_heads, batch.head_dim, batch.page_size = sequences, heads, heads, 64, page
    return _lib.load().kvmix_paged_plan(ctypes.byref(batch), None, 0, ctypes.byref(plan)), plan


@pytest.mark.parametrize("sequences,ok", [(4095, True), (4096, False), (5000, False)])
def test_blocks_of_the_attention(sequences, ok):
    """33 tokens of 4096 heads are 4096 blocks of 256 threads: 2^32 threads or more are more than a launch counts."""
    code, plan = plan_of(sequences, 33, 4096)
    assert code == (0 if ok else -9)
    assert not ok or plan.tiles * plan.kv_heads * 256 < 1 << 32


@pytest.mark.parametrize("sequences,ok", [(16380, True), (16384, False), (20000, False)])
def test_blocks_of_the_store(sequences, ok):
    """One token of 4096 heads each: four heads to a block of 256 threads."""
    code, _ = plan_of(sequences, 1, 4096)
    assert code == (0 if ok else -9)


@pytest.mark.parametrize("head_dim", [1 << 61, 1 << 62, -(1 << 61), 0, -64, 96, (1 << 63) - 1])
def test_head_dimensions_of_packed_pages(head_dim):
    """Refused, whatever their product with the widths is (2^61 times 8 is 0 in 64 bits, and was divided by).  In a process of its own,
    as a division by zero ends it."""
    import subprocess
    import sys

    code = f"""
import torch
from kvmix_amd import ops
try:
    ops.paged_read(torch.zeros(1, 1, 1024, dtype=torch.int32), torch.tensor([0]), 4, 2, {head_dim})
except RuntimeError as e:
    print("refused:", e)
"""
    done = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True, timeout=300)
    assert done.returncode == 0 and "head dimension" in done.stdout, (done.returncode, done.stdout, done.stderr[-500:])


def test_the_most_new_tokens_of_few_rows():
    """What the attention's kernel of few rows is chosen by: sequences of many rows and idle ones do not count."""
    table = [[i] for i in range(4)]
    for new, most in (([1, 1, 0, 1], 1), ([1, 3, 0, 1], 3), ([1, 60, 0, 1], 1), ([0, 60, 0, 0], 0), ([4, 60, 5, 0], 5)):
        plan, _ = _lib.paged_plan(table, [64] * 4, [0] * 4, new, 8, 2, 128, 64)
        assert plan["few_tokens"] == most
