// How the likelihoods' kernels (token_logprobs.hip) share out rows: plain C++, so that it can be checked without a GPU.
#pragma once

#include <cstdint>

#include "../../include/kvmix_hip.h"

namespace kvmix {

constexpr int kPieces = 16;  // of sixteen bytes that a thread holds
constexpr int64_t kGradChunk = 8192;
constexpr int64_t kManyRows = 512;

// Threads to a row, and chunks of it.  Blocks of 256 threads, of which several share a CU, where there are rows enough for all CUs
// and they fit; else of 1024: a row's latency is what counts, or its length.
struct ScorePlan {
    int threads;
    int64_t chunks, chunk;
};

inline int64_t chunk_of(int64_t vocab, int64_t chunks) { return ((vocab + chunks - 1) / chunks + 7) / 8 * 8; }

inline ScorePlan score_plan(int64_t rows, int64_t vocab, int dtype)
{
    const int64_t per = dtype == KVMIX_F32 ? 4 : 8;
    const int threads = rows >= kManyRows && vocab <= (256 * kPieces - 1) * per ? 256 : 1024;
    // what a block holds, with a piece for a row that is not aligned, in whole eights, as chunks are (of 32-bit values it is four short)
    const int64_t most = (threads * kPieces - 1) * per / 8 * 8;
    const int64_t chunks = (vocab + most - 1) / most;
    return {threads, chunks, chunks > 1 ? chunk_of(vocab, chunks) : vocab};
}

}  // namespace kvmix
