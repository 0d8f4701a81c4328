"""Parts of rows that a request's selection is joined from: never more than the join has places for.  No GPU."""
import ctypes

import pytest

from kvmix_amd import _lib
from test_beams_cpu import select


@pytest.mark.parametrize("dtype,per", [(1, 4), (0, 8), (2, 8)])
def test_no_more_parts_than_places(dtype, per):
    """All numbers of beams, at their largest vocabularies and where a part begins: the 2^25 / 8192 full parts of a request's values in
    32 bits and one part that is not full to each of its beams are what there are places for, 4096 of them alone are too few."""
    L, block, most = _lib.load(), 256 * 8 * per, 0
    for beams in range(1, 65):
        largest = min(1 << 20, (1 << 25) // beams)
        for vocab in {largest, largest // block * block, largest // block * block + 1, largest // block * block - block + 1, largest // 2 + 1, 32000}:
            if not 1 <= vocab <= largest:
                continue
            c = select(requests=1, beams=beams, vocab=vocab, row_stride=vocab, dtype=dtype, count=1)
            lists, left = divmod(L.kvmix_beam_select_workspace_bytes(ctypes.byref(c)), 16)
            assert left == 0 and beams <= lists <= (1 << 25) // 8192 + 64
            most = max(most, lists)
    assert (most > 4096) == (dtype == 1)
