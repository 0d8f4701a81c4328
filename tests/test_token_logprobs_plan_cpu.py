"""How the likelihoods' kernels share out a row (csrc/score_plan.h): a block's threads hold every value of its chunk, whatever
the vocabulary, the type and the alignment of the row.  No GPU."""
import os
import shutil
import subprocess

import pytest

CSRC = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "kvmix_amd", "csrc")

# pieces of sixteen bytes that `length` values from an address `skew` values behind a multiple of sixteen bytes lie in
PROGRAM = r"""
#include <algorithm>
#include <cstdio>
#include "score_plan.h"
using namespace kvmix;
int main()
{
    long bad = 0;
    for (int dtype : {KVMIX_F16, KVMIX_F32, KVMIX_BF16}) {
        const int64_t per = dtype == KVMIX_F32 ? 4 : 8;
        for (int64_t rows : {int64_t(1), kManyRows}) {
            for (int64_t vocab = 1; vocab <= 1 << 20; vocab++) {
                const ScorePlan p = score_plan(rows, vocab, dtype);
                int64_t most = 0;
                for (int64_t skew = 0; skew < per; skew++) {  // (chunks begin at multiples of a piece: the row's skew is theirs)
                    most = std::max(most, (std::min(p.chunk, vocab) + skew + per - 1) / per);
                }
                const bool ok = most <= int64_t(p.threads) * kPieces && p.chunks * p.chunk >= vocab && (p.chunks == 1 || p.chunk % per == 0) &&
                                p.chunks <= 17;
                if (!ok && bad++ < 5) std::printf("type %d, %ld rows of %ld: %ld pieces in %d x %d\n", dtype, (long)rows, (long)vocab, (long)most, p.threads, kPieces);
            }
        }
    }
    std::printf("%ld wrong\n", bad);
    return bad != 0;
}
"""


@pytest.mark.skipif(shutil.which("g++") is None, reason="needs a C++ compiler")
def test_a_block_holds_its_chunk(tmp_path):
    source, program = tmp_path / "plan.cpp", tmp_path / "plan"
    source.write_text(PROGRAM)
    subprocess.check_call(["g++", "-O2", "-std=c++17", "-I", CSRC, str(source), "-o", str(program)])
    done = subprocess.run([str(program)], capture_output=True, text=True)
    assert done.returncode == 0, done.stdout
