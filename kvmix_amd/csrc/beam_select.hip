// The best continuations of beams:  of each request the `count` largest of  scores[w] + x[w, v] - lse_w  over its beams w and the
// vocabulary, equal ones in the order of (w, v).  A beam that has ended has one continuation, `end`, at its score.
//
// Bound by the reads of the logits.  A row is read once, by several blocks where there are few rows: a block keeps its part of the row in
// registers, finds the part's largest value m and the sum s of exp(x - m), and its `count` first values.  A lower bound of the
// count-th largest that few others reach is found by bisection over the largest values of 64 groups of threads (as in
// kvmix_token_logprobs); what reaches it is put in order by counting.  A block per request then joins the parts: the parts are sorted
// lists, of which only those that begin with one of the `count` best beginnings can hold a winner, and of these only what is no
// worse than the count-th best beginning.  That block has little to do and waits for everything it does, so it reads all there is at its
// start (where that is up to eight keys to a thread), sums a beam's parts with a lane to a part, and shares the comparisons of few
// lists or candidates among all threads: 6 us, where a thread to a beam and to a list took 12 to 17.
// 64 x 8 beams of 32000 in fp32, a quarter of them ended: 19.1 us, of which 12 to 14 for the 50 MB of rows; 16 x 5 in fp16, 10 of each: 12.4 to 14 us;
// 4 beams: 10.6 us.
//
// Order is decided by 64-bit scores made of sums in 32 bits over parts that begin at multiples of eight values whatever the rows'
// alignment is, so that equal rows have equal scores to the last bit.
#include <algorithm>
#include <type_traits>

#include "score_common.h"

namespace kvmix {

constexpr int kBeamThreads = 256, kBeamPieces = 8;  // of sixteen bytes, of a thread
constexpr int64_t kBeamValues = int64_t(1) << 25;   // of all beams of a request
constexpr int kBeamsMost = 64;
// Parts of a request at most: what a block holds in 32 bits to each, and one that is not full to a beam.
constexpr int kListsMost = kBeamValues / (kBeamThreads * kBeamPieces * 4) + kBeamsMost;
static_assert(kListsMost >= kTopMost * kTopMost && kListsMost >= 1024, "the join keeps as many candidates; beam_plan makes as many parts of few values");

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

// STREAM: the logits are more than the caches of the dies keep, and are read as what nobody wants again soon.
template <typename T, bool STREAM>
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
                x[r].raw = STREAM ? __builtin_nontemporal_load((const uint4u *)(at + i)) : *(const uint4u *)(at + i);
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

constexpr int kTokenBits = 20, kKeysAhead = 8;  // keys that a thread reads at once, before anything is known of the sums

__global__ void __launch_bounds__(kBeamThreads) beam_join(BeamArgs a)
{
    constexpr int NT = kBeamThreads;
    __shared__ double base[kBeamsMost], lse[kBeamsMost];
    __shared__ bool alive[kBeamsMost], ended[kBeamsMost];
    __shared__ double list_score[kListsMost];
    __shared__ uint32_t list_order[kListsMost];
    __shared__ int chosen[kTopMost], before[NT], count;
    __shared__ Candidate last_head, winner[kTopMost];
    const int request = blockIdx.x, t = threadIdx.x, lane = t % kWave, wave = t / kWave;
    const int64_t first = (int64_t)request * a.beams;
    const int lists = a.beams * a.chunks, entries = lists * a.count;
    const bool few = entries <= NT * kKeysAhead, all = lists <= a.count;
    const uint64_t *keys = a.keys + first * a.chunks * a.count;
    uint64_t key[kKeysAhead];
    if (few) {
#pragma unroll
        for (int i = 0; i < kKeysAhead; i++) key[i] = keys[min(t + NT * i, entries - 1)];
    }
    if (t == 0) count = 0;
    before[t] = 0;

    // the sum of a beam's parts, by as many lanes as there are parts
    const int group = a.chunks > 32 ? kWave : a.chunks > 1 ? 1 << (32 - __clz(a.chunks - 1)) : 1, at = t % group;
    for (int w = t / group; w < a.beams; w += NT / group) {
        const int64_t row = first + w;
        const BeamPart *p = a.part + row * a.chunks;
        const float score = a.scores[row];
        const bool over = a.done && a.done[row];
        bool on = finite(score) && !over;
        BeamPart one = {-__builtin_inff(), 0.0f};
        if (at < a.chunks) one = p[at];  // (of a beam of which nothing is asked: anything)
        float m = one.m;
        for (int i = at + group; i < a.chunks; i += group) m = fmaxf(m, p[i].m);
        for (int o = group / 2; o; o /= 2) m = fmaxf(m, __shfl_xor(m, o));
        double s = 0.0;
        for (int i = at; i < a.chunks; i += group) {
            const BeamPart q = i == at ? one : p[i];
            // (nothing but -inf: nothing, unless there is NaN)
            if (q.m == m) s += q.s;
            else if (q.m > -__builtin_inff() || q.s != q.s) s += q.s * __builtin_amdgcn_exp2f((q.m - m) * kLog2e);
        }
        for (int o = group / 2; o; o /= 2) s += __shfl_xor(s, o);
        on = on && finite(m) && s > 0.0 && s < __builtin_inf();
        if (at == 0) {
            base[w] = finite(score) ? (double)score : -__builtin_inf();
            lse[w] = on ? log(s) + (double)m : 0.0;
            alive[w] = on, ended[w] = over;
        }
    }
    __syncthreads();
    // Entry i of list l: list l is part l % chunks of beam l / chunks.  A beam that has ended, or of which nothing can be computed, has
    // its first list only.
    auto entry = [&](int l, int i, uint64_t key, Candidate &c) {
        const int w = l / a.chunks, nth = l % a.chunks;
        const uint32_t beam = (uint32_t)w << kTokenBits;
        if (!alive[w]) {
            c = {ended[w] && i == 0 ? base[w] : -__builtin_inf(), beam | (uint32_t)i};
            return nth == 0;
        }
        c = {base[w] + ((double)key_value((uint32_t)(key >> 32)) - lse[w]), beam | ~(uint32_t)key};
        return key != 0;
    };
    auto head = [&](int l, bool some, const Candidate &c) {
        list_score[l] = some ? c.score : -__builtin_inf(), list_order[l] = some ? c.order : ~0u - l;  // (none: after all others)
    };
    // how many of [from, to) come before `mine`
    auto rank_of = [&](const Candidate &mine, int from, int to) {
        int rank = 0;
        for (int j = from; j < to; j += 8) {
            double score[8];
            uint32_t order[8];
#pragma unroll
            for (int i = 0; i < 8; i++) score[i] = list_score[min(j + i, to - 1)], order[i] = list_order[min(j + i, to - 1)];
#pragma unroll
            for (int i = 0; i < 8; i++) rank += j + i < to && Candidate{score[i], order[i]}.before(mine);
        }
        return rank;
    };
    // Calls f(rank, i) for each of the n in the lists; few of them are compared by all threads, who add to `counts`.
    auto rank_all = [&](int n, int *counts, auto f) {
        if (n <= NT / 2) {
            const int wide = n > 1 ? 1 << (32 - __clz(n - 1)) : 1, parts = NT / wide, i = t % wide, each = (n + parts - 1) / parts, from = t / wide * each;
            if (i < n) atomicAdd(&counts[i], rank_of({list_score[i], list_order[i]}, from, min(n, from + each)));
            __syncthreads();
            if (t < n) f(counts[t], t);
        } else {
            for (int i = t; i < n; i += NT) f(rank_of({list_score[i], list_order[i]}, 0, n), i);
        }
    };
    Candidate mine[kKeysAhead];
    uint32_t some = 0;
    if (few) {
#pragma unroll
        for (int i = 0; i < kKeysAhead; i++) {
            const int e = t + NT * i, l = e / a.count;
            if (e < entries) {
                const bool is = entry(l, e - l * a.count, key[i], mine[i]);
                some |= (uint32_t)is << i;
                if (!all && e == l * a.count) head(l, is, mine[i]);
            }
        }
    } else if (!all) {
        for (int l = t; l < lists; l += NT) {
            Candidate c;
            const bool is = entry(l, 0, keys[(int64_t)l * a.count], c);
            head(l, is, c);
        }
    }
    if (!all) {
        __syncthreads();
        rank_all(lists, before, [&](int rank, int l) {
            if (rank < a.count) chosen[rank] = l;
            if (rank == a.count - 1) last_head = {list_score[l], list_order[l]};
        });
        __syncthreads();
    }
    // what is no worse than the last of the `count` best beginnings
    auto keep = [&](const Candidate &c) {
        if (!all && last_head.before(c)) return;
        const int to = atomicAdd(&count, 1);
        list_score[to] = c.score, list_order[to] = c.order;
    };
    if (few) {
#pragma unroll
        for (int i = 0; i < kKeysAhead; i++)
            if (some >> i & 1) keep(mine[i]);
    } else {
        const int used = all ? lists : a.count;
        for (int e = t; e < used * a.count; e += NT) {
            const int l = all ? e / a.count : chosen[e / a.count], i = e % a.count;
            Candidate c;
            if (entry(l, i, keys[(int64_t)l * a.count + i], c)) keep(c);
        }
    }
    __syncthreads();
    rank_all(count, before + NT / 2, [&](int rank, int i) {
        if (rank < a.count) winner[rank] = {list_score[i], list_order[i]};
    });
    __syncthreads();
    if (wave != 0) return;
    const Candidate c = winner[min(t, a.count - 1)];
    const int w = (int)(c.order >> kTokenBits);
    int place = t;
    if (a.stay) {
        // the first child of a beam takes its place, the others the places of beams that have none, in order
        uint64_t taken = 0, others = 0;
        for (int i = 0; i < a.count; i++) {
            const uint64_t parent = 1ull << __builtin_amdgcn_readlane(w, i);
            if (taken & parent) others |= 1ull << i;
            taken |= parent;
        }
        place = w;
        if (others >> t & 1) {
            uint64_t left = ~taken;
            for (int i = __popcll(others & ((1ull << t) - 1)); i; i--) left &= left - 1;
            place = __builtin_ctzll(left);
        }
    }
    if (t >= a.count) return;
    const int64_t to = (int64_t)request * a.count + place;
    a.out_scores[to] = (float)c.score;
    a.parents[to] = w;
    a.tokens[to] = ended[w] ? a.end : (int64_t)(c.order & ((1u << kTokenBits) - 1));
}

namespace {

struct BeamPlan {
    int64_t chunks, chunk;
};

// Parts of a row: as many as a block can hold at most, and shorter ones, down to two pieces to a thread, as long as the chip is not full of
// blocks: 512 or 2048 blocks take the same time as 1024.
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
    if (p->beams > kBeamsMost || p->count > kTopMost || p->count > p->vocab || p->vocab > (1 << kTokenBits) || p->beams * p->vocab > kBeamValues)
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
    // Logits of more than the eight dies' caches hold (32 MB): 16.3 instead of 18.1 us behind a kernel that writes 64 x 8 rows of 32000 in fp32, 84
    // instead of 143 of 64 x 16 of 128000; 5 MB in fp16 11.4 instead of 10.4.
    const bool stream_by = p->requests * p->beams * p->vocab > (1 << 25) / (p->dtype == KVMIX_F32 ? 4 : 2);
    with_type(p->dtype, [&](auto zero) {
        using T = decltype(zero);
        if (stream_by) beam_rows<T, true><<<(unsigned)parts, kBeamThreads, 0, st>>>(a);
        else beam_rows<T, false><<<(unsigned)parts, kBeamThreads, 0, st>>>(a);
    });
    beam_join<<<(unsigned)p->requests, kBeamThreads, 0, st>>>(a);
    return launch_status();
}
