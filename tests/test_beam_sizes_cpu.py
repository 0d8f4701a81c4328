"""What a beam search refuses before its first step: all that a selection of its later steps would.  No GPU."""
import ctypes

import pytest

from kvmix_amd import _lib
from kvmix_amd.decoder import check_beams
from test_beams_cpu import select


@pytest.mark.parametrize("requests,beams,vocab", [
    (1, 1, 1), (1, 1, 1 << 20), (1, 1, (1 << 20) + 1), (1, 32, 1 << 20), (1, 33, 1 << 20), (1, 33, 1016800), (1, 33, 1016801), (16, 64, 1 << 19), (1, 64, (1 << 19) + 1),
    (16, 64, 32000), (17, 64, 32000), (1, 5, 4), (1, 0, 4), (1, 65, 100), (1024, 1, 1 << 20), (1025, 1, 100), (0, 4, 100),
])
def test_sizes(requests, beams, vocab):
    taken = _lib.load().kvmix_beam_select(ctypes.byref(select(requests=requests, beams=beams, count=beams, vocab=vocab, row_stride=vocab)), None, 0, None) in (0, -11)
    if taken and requests * beams <= 1024:
        check_beams(requests, beams, None, vocab)
        check_beams(requests, beams, vocab - 1, vocab)
    else:
        with pytest.raises(RuntimeError, match="beam_search"):
            check_beams(requests, beams, None, vocab)
