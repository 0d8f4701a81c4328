// The best continuations of beams:  of each request the `count` largest of  scores[w] + x[w, v] - lse_w  over its beams w and the
// vocabulary, equal ones in the order of (w, v).  A beam that has ended has one continuation, `end`, at its score.
//
// Bound by the reads of the logits.  A row is read once, by several blocks where there are few rows: a block keeps its part of the row in
// registers, finds the part's largest value m and the sum s of exp(x - m), and its `count` first values.  A lower bound of the
// count-th largest that few others reach is found by bisection over the largest values of 64 groups of threads (as in
// kvmix_token_logprobs); what reaches it is put in order by counting.  A block per request then joins the parts: the parts are sorted
// lists, of which only those that begin with one of the `count` best beginnings can hold a winner, and of these only what is no
// worse than the count-th best beginning.
//
// Order is decided by 64-bit scores made of sums in 32 bits over parts that begin at multiples of eight values whatever the rows'
// alignment is, so that equal rows have equal scores to the last bit.
#include <algorithm>
#include <type_traits>

#include "score_common.h"

namespace kvmix {

constexpr int kBeamThreads = 256, kBeamPieces = 8;  // of sixteen bytes, of a thread
constexpr int kBeamsMost = 64, kListsMost = 4096;   // (of 2^25 values in 32 bits)

typedef uint32_t uint4u __attribute__((ext_vector_type(4), aligned(2)));  // (rows are aligned as their values are)

struct BeamPart {
    float m, s;
};

struct BeamArgs {
    const void *x;
    int64_t row_stride;
    const float *scores;
    const uint8_t *done;
    int beams, vocab, count, chunk, chunks, end, stay;
    BeamPart *part;   // [rows][chunks]
    uint64_t *keys;   // [rows][chunks][count], 0 where there are fewer
    float *out_scores;
    int64_t *parents, *tokens;
};

__device__ __forceinline__ bool finite(float v) { return fabsf(v) < __builtin_inff(); }

template <typename T>
__global__ void __launch_bounds__(kBeamThreads) beam_rows(BeamArgs a)
{
    constexpr int PER = 16 / sizeof(T), NT = kBeamThreads, W = NT / kWave;
    constexpr uint32_t none = std::is_same<T, _Float16>::value ? 0xfc00fc00u : std::is_same<T, float>::value ? 0xff800000u : 0xff80ff80u;
    __shared__ uint32_t most[NT];
    __shared__ uint64_t key[kCandidates], best[W];
    __shared__ float wave_sum[W], wave_most[W];
    __shared__ int found;
    const int row = blockIdx.x / a.chunks, nth = blockIdx.x % a.chunks, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if ((a.done && a.done[row]) || !finite(a.scores[row])) return;  // (nothing of its logits is asked for)
    const int begin = nth * a.chunk, length = min(a.vocab - begin, a.chunk);
    const T *at = (const T *)a.x + row * a.row_stride + begin;
    Piece<T> x[kBeamPieces];
#pragma unroll
    for (int r = 0; r < kBeamPieces; r++) {
        const int i = (r * NT + (int)threadIdx.x) * PER;
        if (r * NT * PER < length) {
            if (i + PER <= length) {
                x[r].raw = *(const uint4u *)(at + i);
            } else {
                x[r].raw = uint4v{none, none, none, none};
#pragma unroll
                for (int j = 0; j < PER; j++)
                    if (i + j < length) x[r].t[j] = at[i + j];
            }
        }
    }
    float largest = -__builtin_inff();
#pragma unroll
    for (int r = 0; r < kBeamPieces; r++)
        if (r * NT * PER < length) largest = fmaxf(largest, piece_max(x[r]));
    most[threadIdx.x] = value_key(largest);
    const float wave_m = wave_reduce<true>(largest);
    if (lane == 0) wave_most[wave] = wave_m;
    if (threadIdx.x == 0) found = 0;
    __syncthreads();
    float m = wave_most[0];
#pragma unroll
    for (int w = 1; w < W; w++) m = fmaxf(m, wave_most[w]);
    float s = 0.0f;
    const float reference = m > -__builtin_inff() ? m : 0.0f;  // (of nothing but -inf: the sum is zero)
#pragma unroll
    for (int r = 0; r < kBeamPieces; r++)
        if (r * NT * PER < length) {
#pragma unroll
            for (int j = 0; j < PER; j++) s += __builtin_amdgcn_exp2f((to_float(x[r].t[j]) - reference) * kLog2e);  // (NaN of NaN, and of +inf)
        }
    s = wave_reduce<false>(s);
    if (lane == 0) wave_sum[wave] = s;

    // the lower bound: largest prefix of sixteen bits that `count` groups reach, found by every wave for itself
    uint32_t group = most[lane];
#pragma unroll
    for (int w = 1; w < W; w++) group = max(group, most[w * kWave + lane]);
    uint32_t bound = 0;
#pragma unroll
    for (int bit = 31; bit >= 16; bit--) {
        const uint32_t to = bound | 1u << bit;
        if (__popcll(__ballot(group >= to)) >= a.count) bound = to;
    }
    const float least = bound <= value_key(-__builtin_inff()) ? -__builtin_inff() : key_value(bound);
#pragma unroll
    for (int r = 0; r < kBeamPieces; r++) {
        if (r * NT * PER < length && !(piece_max(x[r]) < least)) {
            const int i = (r * NT + (int)threadIdx.x) * PER;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const float v = to_float(x[r].t[j]);
                if (v >= least && i + j < length) {
                    const int to = atomicAdd(&found, 1);
                    if (to < kCandidates) key[to] = full_key(v, begin + i + j);
                }
            }
        }
    }
    __syncthreads();
    if (threadIdx.x == 0) {
        float sum = wave_sum[0];
        for (int w = 1; w < W; w++) sum += wave_sum[w];
        a.part[(int64_t)row * a.chunks + nth] = {m, sum};
    }
    const int n = found;
    uint64_t *out = a.keys + ((int64_t)row * a.chunks + nth) * a.count;
    if (n <= kCandidates) {
        rank_keys<NT>(key, n, a.count, [&](int rank, uint64_t k) { out[rank] = k; });
        for (int i = n + (int)threadIdx.x; i < a.count; i += NT) out[i] = 0;  // (a part shorter than that)
        return;
    }
    // too many are alike: one by one
    uint64_t last = ~(uint64_t)0;
    for (int k = 0; k < a.count; k++) {
        uint64_t mine = 0;
        for (int i = threadIdx.x; i < length; i += NT) {
            const uint64_t one = full_key(to_float(at[i]), begin + i);
            if (one < last && one > mine) mine = one;
        }
        for (int o = 32; o; o /= 2) {
            const uint64_t other = __shfl_xor((unsigned long long)mine, o);
            mine = other > mine ? other : mine;
        }
        __syncthreads();
        if (lane == 0) best[wave] = mine;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < W; w++) mine = best[w] > mine ? best[w] : mine;
        if (threadIdx.x == 0) out[k] = mine;
        last = mine;
    }
}

// Larger score first, then lower beam, then lower token: no two are alike.
struct Candidate {
    double score;
    uint32_t order;  // beam, and what orders its continuations: the token, or their number where it has ended

    __device__ __forceinline__ bool before(const Candidate &o) const { return score > o.score || (score == o.score && order < o.order); }
};

constexpr int kTokenBits = 20;

__global__ void __launch_bounds__(kBeamThreads) beam_join(BeamArgs a)
{
    __shared__ double base[kBeamsMost], lse[kBeamsMost];
    __shared__ bool alive[kBeamsMost];
    __shared__ double list_score[kListsMost];
    __shared__ uint32_t list_order[kListsMost];
    __shared__ int chosen[kTopMost], count;
    __shared__ Candidate last_head, winner[kTopMost];
    const int request = blockIdx.x, t = threadIdx.x;
    const int64_t first = (int64_t)request * a.beams;
    if (t == 0) count = 0;
    if (t < a.beams) {
        const int64_t row = first + t;
        const float score = a.scores[row];
        bool on = finite(score) && !(a.done && a.done[row]);
        base[t] = finite(score) ? (double)score : -__builtin_inf();
        if (on) {
            const BeamPart *p = a.part + row * a.chunks;
            float m = p[0].m;
            for (int i = 1; i < a.chunks; i++) m = fmaxf(m, p[i].m);
            double s = 0.0;
            for (int i = 0; i < a.chunks; i++) s += p[i].m == m ? (double)p[i].s : p[i].m > -__builtin_inff() || p[i].s != p[i].s ? (double)p[i].s * exp((double)p[i].m - (double)m) : 0.0;
            on = finite(m) && s > 0.0 && s < __builtin_inf();
            lse[t] = on ? log(s) + (double)m : 0.0;
        }
        alive[t] = on;
    }
    __syncthreads();
    // Entry i of list l: list l is part l % chunks of beam l / chunks.  A beam that has ended, or of which nothing can be computed, has
    // its first list only.
    auto entry = [&](int l, int i, Candidate &c) {
        const int w = l / a.chunks, nth = l % a.chunks;
        const uint32_t beam = (uint32_t)w << kTokenBits;
        if (!alive[w]) {
            const bool ended = a.done && a.done[first + w];
            c = {ended && i == 0 ? base[w] : -__builtin_inf(), beam | (uint32_t)i};
            return nth == 0;
        }
        const uint64_t key = a.keys[((first + w) * a.chunks + nth) * a.count + i];
        c = {base[w] + ((double)key_value((uint32_t)(key >> 32)) - lse[w]), beam | ~(uint32_t)key};
        return key != 0;
    };
    const int lists = a.beams * a.chunks;
    const bool all = lists <= a.count;
    if (!all) {
        for (int l = t; l < lists; l += kBeamThreads) {
            Candidate c;
            const bool some = entry(l, 0, c);
            list_score[l] = some ? c.score : -__builtin_inf(), list_order[l] = some ? c.order : ~0u - l;  // (none: after all others)
        }
        __syncthreads();
        for (int l = t; l < lists; l += kBeamThreads) {
            const Candidate mine = {list_score[l], list_order[l]};
            int rank = 0;
            for (int j = 0; j < lists; j++) rank += Candidate{list_score[j], list_order[j]}.before(mine);
            if (rank < a.count) chosen[rank] = l;
            if (rank == a.count - 1) last_head = mine;
        }
        __syncthreads();
    }
    const int used = all ? lists : a.count;
    for (int e = t; e < used * a.count; e += kBeamThreads) {
        Candidate c;
        if (entry(all ? e / a.count : chosen[e / a.count], e % a.count, c) && (all || !last_head.before(c))) {
            const int to = atomicAdd(&count, 1);
            list_score[to] = c.score, list_order[to] = c.order;
        }
    }
    __syncthreads();
    for (int i = t; i < count; i += kBeamThreads) {
        const Candidate mine = {list_score[i], list_order[i]};
        int rank = 0;
#pragma unroll 4
        for (int j = 0; j < count; j++) rank += Candidate{list_score[j], list_order[j]}.before(mine);
        if (rank < a.count) winner[rank] = mine;
    }
    __syncthreads();
    if (t >= a.count) return;
    const Candidate c = winner[t];
    const int w = (int)(c.order >> kTokenBits);
    int place = t;
    if (a.stay) {
        // the first child of a beam takes its place, the others the places of beams that have none, in order
        bool has[2] = {false, false};  // an earlier one of the same parent
        int earlier = 0;               // ones before this that are not their parents' first
        for (int i = 0; i <= t; i++) {
            bool again = false;
            for (int j = 0; j < i; j++) again |= winner[j].order >> kTokenBits == winner[i].order >> kTokenBits;
            if (i == t) has[0] = again;
            else earlier += again;
        }
        if (!has[0]) {
            place = w;
        } else {
            for (place = 0; place < a.beams; place++) {
                bool taken = false;
                for (int j = 0; j < a.count; j++) taken |= (int)(winner[j].order >> kTokenBits) == place;
                if (!taken && earlier-- == 0) break;
            }
        }
    }
    const int64_t to = (int64_t)request * a.count + place;
    a.out_scores[to] = (float)c.score;
    a.parents[to] = w;
    a.tokens[to] = a.done && a.done[first + w] ? a.end : (int64_t)(c.order & ((1u << kTokenBits) - 1));
}

namespace {

struct BeamPlan {
    int64_t chunks, chunk;
};

// Parts of a row: as many as a block can hold at most, and shorter ones, down to two pieces to a thread, as long as the chip is not full of
// blocks (or a request has more lists than the join takes).
BeamPlan beam_plan(const kvmix_beam_select_t *p)
{
    const int64_t rows = std::max<int64_t>(p->requests * p->beams, 1), per = p->dtype == KVMIX_F32 ? 4 : 8, piece = kBeamThreads * per;
    const int64_t least = (p->vocab + kBeamPieces * piece - 1) / (kBeamPieces * piece), most = (p->vocab + 2 * piece - 1) / (2 * piece);
    int64_t chunks = std::max(least, std::min(most, 1024 / rows));
    const int64_t chunk = ((p->vocab + chunks - 1) / chunks + 7) / 8 * 8;
    return {(p->vocab + chunk - 1) / chunk, chunk};
}

int beam_check(const kvmix_beam_select_t *p)
{
    if (!p) return KVMIX_ERR_NULL;
    if (p->dtype != KVMIX_F16 && p->dtype != KVMIX_F32 && p->dtype != KVMIX_BF16) return KVMIX_ERR_DTYPE;
    if (p->requests < 0 || p->beams <= 0 || p->vocab <= 0 || p->count <= 0 || p->row_stride < 0 || (p->done && (p->end < 0 || p->end >= p->vocab)) ||
        (p->stay && p->count != p->beams))
        return KVMIX_ERR_SHAPE;
    if (p->beams > kBeamsMost || p->count > kTopMost || p->count > p->vocab || p->vocab > (1 << kTokenBits) || p->beams * p->vocab > (1 << 25))
        return KVMIX_ERR_UNSUPPORTED;
    if ((__int128)p->requests * p->beams * ((p->vocab + 2047) / 2048 + 1) >= 1 << 24) return KVMIX_ERR_UNSUPPORTED;  // (blocks of 256 threads)
    return KVMIX_OK;
}

}  // namespace
}  // namespace kvmix

using namespace kvmix;

extern "C" int64_t kvmix_beam_select_workspace_bytes(const kvmix_beam_select_t *p)
{
    if (beam_check(p) != KVMIX_OK) return 0;
    return p->requests * p->beams * beam_plan(p).chunks * (int64_t)(sizeof(BeamPart) + p->count * sizeof(uint64_t));
}

extern "C" int kvmix_beam_select(const kvmix_beam_select_t *p, void *workspace, int64_t workspace_bytes, kvmix_stream_t stream)
{
    const int rc = beam_check(p);
    if (rc != KVMIX_OK) return rc;
    if (p->requests == 0) return KVMIX_OK;
    if (!p->logits || !p->scores || !p->out_scores || !p->parents || !p->tokens) return KVMIX_ERR_NULL;
    const int64_t need = kvmix_beam_select_workspace_bytes(p);
    if (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < need) return KVMIX_ERR_WORKSPACE;
    const BeamPlan plan = beam_plan(p);
    const int64_t parts = p->requests * p->beams * plan.chunks;
    BeamArgs a{};
    a.x = p->logits, a.row_stride = p->row_stride, a.scores = p->scores, a.done = p->done;
    a.beams = (int)p->beams, a.vocab = (int)p->vocab, a.count = (int)p->count, a.chunk = (int)plan.chunk, a.chunks = (int)plan.chunks;
    a.end = (int)p->end, a.stay = p->stay;
    a.part = (BeamPart *)workspace, a.keys = (uint64_t *)((BeamPart *)workspace + parts);
    a.out_scores = p->out_scores, a.parents = p->parents, a.tokens = p->tokens;
    hipStream_t st = (hipStream_t)stream;
    with_type(p->dtype, [&](auto zero) { beam_rows<decltype(zero)><<<(unsigned)parts, kBeamThreads, 0, st>>>(a); });
    beam_join<<<(unsigned)p->requests, kBeamThreads, 0, st>>>(a);
    return launch_status();
}
