// Log probabilities of given tokens under rows of logits, with the entropy and the most likely tokens, and their gradient.
//
//   lse = log sum_i exp(x_i),  logprob = x_t - lse,  entropy = lse - sum_i p_i x_i,  p_i = exp(x_i - lse)
//   dx_i = a (1[i = t] - p_i) - b p_i (log p_i + entropy)   for the gradients a of logprob and b of entropy
//
// Bound by the reads: a row (up to 128k values of 16 bits) is read once into registers by one block, and everything is made of it
// there: the largest value, the sums s = sum 2^d and u = sum 2^d d with d = (x - m) log2(e), from which lse - m = ln 2 log2 s and
// entropy = ln 2 (log2 s - u / s), and the most likely tokens.  The sums run while the row arrives, relative to the wave's largest
// value so far (with the largest value first and the sums after it the blocks of a CU all read and then all computed: 122
// against 106 us for 8192 rows of 32000 halves and the top 20).
//
// Most likely tokens: lanes of one number in all waves make a group, 64 of them; the k-th largest of the groups' largest values is
// a lower bound of the row's k-th largest value that few others reach (25 values for k = 20).  It is found by bisection over
// the lanes, by its upper sixteen bits; what reaches it is collected and put in order by counting.  Equal logits come in the
// order of their indexes.  Rows in which too many reach it (constant ones), or with NaN, are searched value by value.
//
// 8192 rows of 32000 halves with the top 20: 100 us, 5.2 TB/s (a pure read 6.2); one row with the top 5: 6.8 us, a launch of one
// chain of latencies; 4099 rows with both gradients 161 us (787 MB, 4.9 TB/s; a large copy 4.75); 4096 rows with the top 20 in bf16
// 74 us, in fp32 140 (3.5 and 3.7 TB/s).
#include <algorithm>
#include <type_traits>

#include "kvmix_common.h"
#include "score_plan.h"

namespace kvmix {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr float kStale = 20.0f;    // how far a value may exceed what sums are relative to: 2^d stays below 2^29
constexpr float kFar = 16777216.0f;  // up to there the rounding of m log2(e) is 1 at most (at 1e10 it is 512 and more, and 2^512 no number)
constexpr float kNothing = -1024.0f;  // 2^d is zero from here on, and its products with sums and gradients of any size are finite
constexpr int kTopMost = 64, kCandidates = 1024;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

struct ScoreStats {
    float m, s, u;  // reference (as a logit), sum of 2^d, sum of 2^d d
};

struct ScoreArgs {
    const void *x;
    int64_t row_stride;
    const int64_t *targets;
    float *logprob, *entropy, *top_logprob;
    int64_t *top_id;
    float *stats;             // [rows][4]: m, log2 of the sum of exp(x - m), entropy; NULL where no gradient is wanted
    int rows, vocab, top, chunk, chunks;
    ScoreStats *part;         // [rows][chunks]
    uint64_t *part_keys;      // [rows][chunks][top]
    // the gradient
    const float *grad_logprob, *grad_entropy;
    void *dx;
    int64_t dx_stride;
};

template <typename T>
__device__ __forceinline__ float to_float(T v)
{
    return (float)v;
}

// A row's values from `begin` on as sixteen-byte pieces of memory: the first and the last may hold others, of no concern, beside
// it (they lie in the same sixteen aligned bytes as values of the row do).
template <typename T>
struct Span {
    static constexpr int PER = 16 / sizeof(T);
    const uint4v *at;
    int first, length, pieces;  // piece p holds values first + p * PER .. of [0, length)

    __device__ __forceinline__ Span(const T *row, int begin, int end)
    {
        const int skew = (int)((uintptr_t)(row + begin) / sizeof(T) % PER);
        at = (const uint4v *)(row + begin - skew);
        first = -skew, length = max(end - begin, 0), pieces = length ? (length + skew + PER - 1) / PER : 0;
    }
};

template <typename T>
union Piece {
    uint4v raw;
    T t[16 / sizeof(T)];
};

// The largest of a piece's values (not NaN), two at a time where the type allows it.
__device__ __forceinline__ float piece_max(const Piece<_Float16> &w)
{
    typedef _Float16 half2v __attribute__((ext_vector_type(2)));
    uint32_t word = w.raw[0];
#pragma unroll
    for (int j = 1; j < 4; j++) asm("v_pk_max_f16 %0, %0, %1" : "+v"(word) : "v"(w.raw[j]));  // (without the builtin's quieting of both)
    const half2v most = __builtin_bit_cast(half2v, word);
    return fmaxf((float)most[0], (float)most[1]);
}

template <typename T>
__device__ __forceinline__ float piece_max(const Piece<T> &w)
{
    float most = to_float(w.t[0]);
#pragma unroll
    for (int j = 1; j < Span<T>::PER; j++) most = fmaxf(most, to_float(w.t[j]));
    return most;
}

// A piece of a span, with -inf for what is none of it.
template <typename T>
__device__ __forceinline__ Piece<T> span_piece(const Span<T> &span, int p)
{
    constexpr int PER = Span<T>::PER;
    constexpr uint32_t none = std::is_same<T, _Float16>::value ? 0xfc00fc00u : std::is_same<T, float>::value ? 0xff800000u : 0xff80ff80u;
    Piece<T> w;
    w.raw = uint4v{none, none, none, none};
    if (p < span.pieces) {
        w.raw = span.at[p];
        const int i = span.first + p * PER;
        if (__builtin_expect(i < 0 || i + PER > span.length, 0)) {
#pragma unroll
            for (int k = 0; k < 4; k++) {
                uint32_t keep = 0;
#pragma unroll
                for (int j = k * PER / 4; j < (k + 1) * PER / 4; j++)
                    if (i + j >= 0 && i + j < span.length) keep |= PER == 4 ? 0xffffffffu : 0xffffu << 16 * (j % 2);
                w.raw[k] = (w.raw[k] & keep) | (none & ~keep);
            }
        }
    }
    return w;
}

__device__ __forceinline__ ScoreStats merged(ScoreStats a, ScoreStats b)
{
    // (references of -inf: nothing summed yet; the difference is kept finite, so that nothing times it is nothing)
    const float m = fmaxf(a.m, b.m);
    const float da = fmaxf((a.m - m) * kLog2e, kNothing), db = fmaxf((b.m - m) * kLog2e, kNothing);
    const float fa = __builtin_amdgcn_exp2f(da), fb = __builtin_amdgcn_exp2f(db);
    return {m, a.s * fa + b.s * fb, (a.u + a.s * da) * fa + (b.u + b.s * db) * fb};
}

// order of the most likely: larger value first, then lower index; NaN is larger than anything
__device__ __forceinline__ uint32_t value_key(float v)
{
    const uint32_t b = __float_as_uint(v + 0.0f);  // (-0 is 0)
    return v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ uint64_t full_key(float v, int index) { return (uint64_t)value_key(v) << 32 | (uint32_t)~index; }

template <int NT>
struct TopShared {
    uint32_t most[NT];
    uint64_t key[kCandidates];
    uint64_t best[NT / kWave];
    int count;
};

// Calls f(rank, key) for the `top` first of `count` different keys, by the threads of a block.
template <int NT, typename F>
__device__ __forceinline__ void rank_keys(const uint64_t *key, int count, int top, F f)
{
    for (int i = threadIdx.x; i < count; i += NT) {
        const uint64_t mine = key[i];
        int rank = 0;
#pragma unroll 8
        for (int j = 0; j < count; j++) rank += key[j] > mine;
        if (rank < top) f(rank, mine);
    }
}

// The `top` first keys of a span, one by one: for rows in which too many values are alike.
template <typename T, int NT, typename F>
__device__ void search_keys(const Span<T> &span, int begin, int top, uint64_t *shared, F f)
{
    constexpr int PER = Span<T>::PER;
    uint64_t last = ~(uint64_t)0;
    for (int k = 0; k < top; k++) {
        uint64_t best = 0;
        for (int p = threadIdx.x; p < span.pieces; p += NT) {
            const Piece<T> w = span_piece(span, p);
            const int i = span.first + p * PER;
#pragma unroll
            for (int j = 0; j < PER; j++) {
                const uint64_t key = full_key(to_float(w.t[j]), begin + i + j);
                if (i + j >= 0 && i + j < span.length && (key < last || k == 0) && key > best) best = key;
            }
        }
        for (int o = 32; o; o /= 2) {
            const uint64_t other = __shfl_xor((unsigned long long)best, o);
            best = other > best ? other : best;
        }
        __syncthreads();
        if (threadIdx.x % kWave == 0) shared[threadIdx.x / kWave] = best;
        __syncthreads();
        for (int w = 0; w < NT / kWave; w++) best = shared[w] > best ? shared[w] : best;
        if (threadIdx.x == 0 && best) f(k, best);
        last = best;
    }
}

// The logit of a row's target (NaN if it is past the vocabulary).
template <typename T>
__device__ __forceinline__ float target_logit(const ScoreArgs &a, int row, int64_t target)
{
    return target >= 0 && target < a.vocab ? to_float(((const T *)a.x)[row * a.row_stride + target]) : __builtin_nanf("");
}

// A row's results from its sums: by one thread.
__device__ __forceinline__ float finish_row(const ScoreArgs &a, int row, ScoreStats t, int64_t target, float x)
{
    float sum2 = log2f(t.s), entropy = kLn2 * (log2f(t.s) - t.u / t.s);
    if (t.m == __builtin_inff() || !(t.s > 0.0f)) sum2 = entropy = __builtin_nanf("");
    a.logprob[row] = target < 0 ? 0.0f : (x - t.m) - kLn2 * sum2;
    a.entropy[row] = entropy;
    if (a.stats) {
        float *s = a.stats + 4 * (int64_t)row;
        s[0] = t.m, s[1] = sum2, s[2] = entropy, s[3] = 0.0f;
    }
    return sum2;
}

__device__ __forceinline__ void write_top(const ScoreArgs &a, int row, int rank, uint64_t key, float m, float sum2)
{
    a.top_logprob[(int64_t)row * a.top + rank] = (key_value((uint32_t)(key >> 32)) - m) - kLn2 * sum2;
    a.top_id[(int64_t)row * a.top + rank] = (int64_t)~(uint32_t)key;
}

template <typename T, int NT, bool TOP>
__global__ void __launch_bounds__(NT) score_rows(ScoreArgs a)
{
    constexpr int PER = 16 / sizeof(T), W = NT / kWave;
    __shared__ ScoreStats wave_stats[W];
    __shared__ typename std::conditional<TOP, TopShared<NT>, int>::type sh;
    __shared__ float done[2];
    const int row = blockIdx.x / a.chunks, nth = blockIdx.x % a.chunks, lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    const int begin = nth * a.chunk, end = min(a.vocab, begin + a.chunk);
    const Span<T> span((const T *)a.x + row * a.row_stride, begin, end);
    Piece<T> x[kPieces];
#pragma unroll
    for (int r = 0; r < kPieces; r++)
        if (r * NT < span.pieces) x[r] = span_piece(span, r * NT + (int)threadIdx.x);

    const int64_t target = a.targets[row];
    const float at_target = target_logit<T>(a, row, target);  // (here, so that it has arrived when it is wanted)

    // The sums as the pieces arrive, relative to a value of the wave's that is moved when another exceeds it by kStale.  One
    // operation for x log2(e) - m log2(e); the rounding of the latter, the same in every term, leaves the sums at the end.  Two
    // beyond kFar.
    float largest = -__builtin_inff(), m2 = 0.0f;
    ScoreStats t = {-__builtin_inff(), 0.0f, 0.0f};
    bool far = false;
    auto add = [&](const Piece<T> &w, auto difference) {
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const float d = difference(to_float(w.t[j])), e = __builtin_amdgcn_exp2f(d);
            t.s += e;
            t.u = fmaf(e, fmaxf(d, kNothing), t.u);  // (zero times -inf is to be zero)
        }
    };
#pragma unroll
    for (int r = 0; r < kPieces; r++) {
        if (r * NT < span.pieces) {
            const float most = piece_max(x[r]);
            largest = fmaxf(largest, most);
            if (__any(most > t.m + kStale)) {  // (also what leaves -inf)
                const float m = wave_reduce<true>(largest);
                const bool was = far;
                far = !std::is_same<T, _Float16>::value && __builtin_amdgcn_readfirstlane(!(fabsf(m) < kFar));
                const float d = fmaxf(far || was || t.m == -__builtin_inff() ? (t.m - m) * kLog2e : m2 - m * kLog2e, kNothing);
                const float f = __builtin_amdgcn_exp2f(d);
                t.u = fmaf(t.s, d, t.u) * f, t.s *= f, t.m = m, m2 = m * kLog2e;
            }
            // (until then a wave has seen -inf only: zero as the reference, nothing to the sums.  NaN, and +inf against itself, make
            // the sum NaN.)
            if (!far) add(x[r], [&](float v) { return fmaf(v, kLog2e, -m2); });
            else add(x[r], [&](float v) { return (v - t.m) * kLog2e; });
        }
    }
    // At the end relative to the wave's largest value itself, with one rounding.  (Relative to one up to kStale below it log2 s and
    // u / s are both near 29, and every rounding of a merge is one of that size in their difference: the entropy of 196585 values of
    // which one takes nearly all came out as 1.06e-5 for 2.6e-6.)
    const float m = wave_reduce<true>(largest);
    if (m != -__builtin_inff()) {
        const float d = far ? fmaxf((t.m - m) * kLog2e, kNothing) : fmaf(-m, kLog2e, m2), f = __builtin_amdgcn_exp2f(d);
        t.u = fmaf(t.s, d, t.u) * f, t.s *= f, t.m = m;
    }
    t.s = wave_reduce<false>(t.s), t.u = wave_reduce<false>(t.u);
    if (lane == 0) wave_stats[wave] = t;
    if constexpr (TOP) {
        sh.most[threadIdx.x] = value_key(largest);
        if (threadIdx.x == 0) sh.count = 0;
    }
    __syncthreads();
    if (!TOP || threadIdx.x == 0) {
        if (threadIdx.x == 0) {
            t = wave_stats[0];
            for (int w = 1; w < W; w++) t = merged(t, wave_stats[w]);
            if (a.chunks == 1) done[0] = t.m, done[1] = finish_row(a, row, t, target, at_target);
            else a.part[(int64_t)row * a.chunks + nth] = t;
        }
        if (!TOP) return;
    }
    if constexpr (TOP) {
        // the lower bound: largest prefix of sixteen bits that `top` groups reach, found by every wave for itself
        // (`least`: as a number; there is no NaN where it is used)
        uint32_t group = sh.most[lane];
#pragma unroll
        for (int w = 1; w < W; w++) group = max(group, sh.most[w * kWave + lane]);
        uint32_t bound = 0;
#pragma unroll
        for (int bit = 31; bit >= 16; bit--) {
            const uint32_t to = bound | 1u << bit;
            if (__popcll(__ballot(group >= to)) >= a.top) bound = to;
        }
        const float least = bound <= value_key(-__builtin_inff()) ? -__builtin_inff() : key_value(bound);
        bool nan = false;
        for (int w = 0; w < W; w++) nan |= !(wave_stats[w].s >= 0.0f);
        if (!nan) {
#pragma unroll
            for (int r = 0; r < kPieces; r++) {
                if (r * NT >= span.pieces) break;
                if (piece_max(x[r]) < least) continue;
                const int i = span.first + (r * NT + (int)threadIdx.x) * PER;
#pragma unroll
                for (int j = 0; j < PER; j++) {
                    const float v = to_float(x[r].t[j]);
                    if (v >= least && i + j >= 0 && i + j < span.length) {
                        const int at = atomicAdd(&sh.count, 1);
                        if (at < kCandidates) sh.key[at] = full_key(v, begin + i + j);
                    }
                }
            }
        }
        __syncthreads();
        const int count = sh.count;
        uint64_t *part = a.part_keys + ((int64_t)row * a.chunks + nth) * a.top;
        const float dm = done[0], sum2 = done[1];
        auto found = [&](int rank, uint64_t key) {
            if (a.chunks > 1) part[rank] = key;
            else write_top(a, row, rank, key, dm, sum2);
        };
        if (!nan && count <= kCandidates) {
            rank_keys<NT>(sh.key, count, a.top, found);
            if (a.chunks > 1)  // (a chunk shorter than that)
                for (int i = count + (int)threadIdx.x; i < a.top; i += NT) part[i] = 0;
        } else {
            if (a.chunks > 1)
                for (int i = span.length + (int)threadIdx.x; i < a.top; i += NT) part[i] = 0;
            search_keys<T, NT>(span, begin, a.top, sh.best, found);
        }
    }
}

// The chunks of a row together.
template <typename T, bool TOP>
__global__ void __launch_bounds__(256) score_join(ScoreArgs a)
{
    __shared__ uint64_t key[TOP ? 2 * kCandidates : 1];  // (of 2^20 values in 32 bits there are 17 chunks)
    __shared__ float done[2];
    const int row = blockIdx.x;
    if (threadIdx.x == 0) {
        ScoreStats t = a.part[(int64_t)row * a.chunks];
        for (int i = 1; i < a.chunks; i++) t = merged(t, a.part[(int64_t)row * a.chunks + i]);
        const int64_t target = a.targets[row];
        done[0] = t.m, done[1] = finish_row(a, row, t, target, target_logit<T>(a, row, target));
    }
    if constexpr (TOP) {
        const int count = a.chunks * a.top;
        for (int i = threadIdx.x; i < count; i += 256) key[i] = a.part_keys[(int64_t)row * count + i];
        __syncthreads();
        rank_keys<256>(key, count, a.top, [&](int rank, uint64_t k) { write_top(a, row, rank, k, done[0], done[1]); });
    }
}

// The gradient, a piece per thread: pieces of dx lie as those of x do where their rows are aligned alike, else value by value.
template <typename T>
__global__ void __launch_bounds__(256) score_grad(ScoreArgs a)
{
    constexpr int PER = 16 / sizeof(T);
    const int row = blockIdx.x / a.chunks, nth = blockIdx.x % a.chunks;
    const int begin = nth * a.chunk, end = min(a.vocab, begin + a.chunk);
    const Span<T> span((const T *)a.x + row * a.row_stride, begin, end);
    T *dx = (T *)a.dx + row * a.dx_stride + begin;
    const float *s = a.stats + 4 * (int64_t)row;
    const float m = s[0], sum2 = s[1], entropy = s[2];
    const int64_t target = a.targets[row];
    const float ga = a.grad_logprob && target >= 0 ? a.grad_logprob[row] : 0.0f, gb = a.grad_entropy ? a.grad_entropy[row] : 0.0f;
    const int hit = target >= begin && target < end ? (int)target - begin : -PER;
    const bool alike = (((uintptr_t)span.at ^ (uintptr_t)(dx + span.first)) & 15) == 0;
    for (int p = threadIdx.x; p < span.pieces; p += 256) {
        const int i = span.first + p * PER;
        Piece<T> w = span_piece(span, p);
        float g[PER];
#pragma unroll
        for (int j = 0; j < PER; j++) {
            const float q = fmaxf(fmaf(to_float(w.t[j]) - m, kLog2e, -sum2), kNothing);
            g[j] = -__builtin_amdgcn_exp2f(q) * (ga + gb * (q * kLn2 + entropy));
        }
        if (hit >= i && hit < i + PER) {
#pragma unroll
            for (int j = 0; j < PER; j++) g[j] += i + j == hit ? ga : 0.0f;
        }
#pragma unroll
        for (int j = 0; j < PER; j++) w.t[j] = (T)g[j];
        if (alike && i >= 0 && i + PER <= span.length) {
            *(uint4v *)(dx + i) = w.raw;
        } else {
#pragma unroll
            for (int j = 0; j < PER; j++)
                if (i + j >= 0 && i + j < span.length) dx[i + j] = w.t[j];
        }
    }
}

namespace {

int score_check(const kvmix_token_logprobs_t *p)
{
    if (!p) return KVMIX_ERR_NULL;
    if (p->dtype != KVMIX_F16 && p->dtype != KVMIX_F32 && p->dtype != KVMIX_BF16) return KVMIX_ERR_DTYPE;
    if (p->rows < 0 || p->vocab < 0 || p->top < 0 || (p->rows > 1 && p->row_stride < p->vocab)) return KVMIX_ERR_SHAPE;
    if (p->top > kTopMost || p->top > p->vocab || p->vocab > (1 << 20) || p->vocab == 0) return KVMIX_ERR_UNSUPPORTED;
    if ((__int128)p->rows * ((p->vocab + kGradChunk - 1) / kGradChunk) > 0x7fffffff) return KVMIX_ERR_UNSUPPORTED;
    return KVMIX_OK;
}

// f(first, rows) for launches of fewer than 2^32 threads together
template <typename F>
void launches_of(int64_t rows, int64_t threads_per_row, F f)
{
    const int64_t most = 0xffffffffll / threads_per_row;
    for (int64_t first = 0; first < rows; first += most) f(first, (unsigned)std::min(most, rows - first));
}

// The rows from `first` on.
template <typename T>
ScoreArgs rows_from(ScoreArgs a, int64_t first)
{
    a.x = (const T *)a.x + first * a.row_stride;
    a.targets += first;
    if (a.logprob) a.logprob += first, a.entropy += first;
    if (a.top) a.top_logprob += first * a.top, a.top_id += first * a.top;
    if (a.stats) a.stats += 4 * first;
    if (a.chunks > 1) a.part += first * a.chunks, a.part_keys += first * a.chunks * a.top;
    if (a.grad_logprob) a.grad_logprob += first;
    if (a.grad_entropy) a.grad_entropy += first;
    if (a.dx) a.dx = (T *)a.dx + first * a.dx_stride;
    return a;
}

template <typename F>
void with_type(int dtype, F f)
{
    if (dtype == KVMIX_F16) f((_Float16)0);
    else if (dtype == KVMIX_F32) f(0.0f);
    else f((__bf16)0.0f);
}

}  // namespace
}  // namespace kvmix

using namespace kvmix;

extern "C" int64_t kvmix_token_logprobs_workspace_bytes(const kvmix_token_logprobs_t *p)
{
    if (score_check(p) != KVMIX_OK) return 0;
    const int64_t n = score_plan(p->rows, p->vocab, p->dtype).chunks;
    return n > 1 ? p->rows * n * (p->top * 8 + (int64_t)sizeof(ScoreStats)) : 0;
}

extern "C" int kvmix_token_logprobs(const kvmix_token_logprobs_t *p, void *workspace, int64_t workspace_bytes, kvmix_stream_t stream)
{
    const int rc = score_check(p);
    if (rc != KVMIX_OK) return rc;
    if (p->rows == 0) return KVMIX_OK;
    if (!p->logits || !p->targets || !p->logprob || !p->entropy || (p->top && (!p->top_logprob || !p->top_id))) return KVMIX_ERR_NULL;
    const int64_t need = kvmix_token_logprobs_workspace_bytes(p);
    if (need && (!workspace || (uintptr_t)workspace % 8 || workspace_bytes < need)) return KVMIX_ERR_WORKSPACE;
    ScoreArgs a{};
    a.x = p->logits, a.row_stride = p->row_stride, a.targets = p->targets;
    a.logprob = p->logprob, a.entropy = p->entropy, a.top_logprob = p->top_logprob, a.top_id = p->top_id, a.stats = p->stats;
    a.rows = (int)p->rows, a.vocab = (int)p->vocab, a.top = (int)p->top;
    const ScorePlan plan = score_plan(p->rows, p->vocab, p->dtype);
    a.chunks = (int)plan.chunks, a.chunk = (int)plan.chunk;
    a.part_keys = (uint64_t *)workspace;
    a.part = (ScoreStats *)((uint64_t *)workspace + p->rows * a.chunks * p->top);
    hipStream_t st = (hipStream_t)stream;
    with_type(p->dtype, [&](auto zero) {
        using T = decltype(zero);
        launches_of(p->rows, plan.threads * a.chunks, [&](int64_t first, unsigned rows) {
            const ScoreArgs part = rows_from<T>(a, first);
            const unsigned grid = rows * (unsigned)a.chunks;
            if (plan.threads == 256) {
                if (p->top) score_rows<T, 256, true><<<grid, 256, 0, st>>>(part);
                else score_rows<T, 256, false><<<grid, 256, 0, st>>>(part);
            } else {
                if (p->top) score_rows<T, 1024, true><<<grid, 1024, 0, st>>>(part);
                else score_rows<T, 1024, false><<<grid, 1024, 0, st>>>(part);
            }
            if (a.chunks > 1) {
                if (p->top) score_join<T, true><<<rows, 256, 0, st>>>(part);
                else score_join<T, false><<<rows, 256, 0, st>>>(part);
            }
        });
    });
    return launch_status();
}

extern "C" int kvmix_token_logprobs_grad(const kvmix_token_logprobs_t *p, const float *grad_logprob, const float *grad_entropy, void *grad_logits,
                                         int64_t grad_row_stride, kvmix_stream_t stream)
{
    const int rc = score_check(p);
    if (rc != KVMIX_OK) return rc;
    if (p->rows > 1 && grad_row_stride < p->vocab) return KVMIX_ERR_SHAPE;
    if (p->rows == 0) return KVMIX_OK;
    if (!p->logits || !p->targets || !p->stats || !grad_logits) return KVMIX_ERR_NULL;
    ScoreArgs a{};
    a.x = p->logits, a.row_stride = p->row_stride, a.targets = p->targets, a.stats = p->stats;
    a.rows = (int)p->rows, a.vocab = (int)p->vocab;
    a.chunks = (int)((p->vocab + kGradChunk - 1) / kGradChunk);
    a.chunk = (int)chunk_of(p->vocab, a.chunks);
    a.grad_logprob = grad_logprob, a.grad_entropy = grad_entropy, a.dx = grad_logits, a.dx_stride = grad_row_stride;
    with_type(p->dtype, [&](auto zero) {
        using T = decltype(zero);
        launches_of(p->rows, 256 * a.chunks, [&](int64_t first, unsigned rows) {
            score_grad<T><<<rows * (unsigned)a.chunks, 256, 0, (hipStream_t)stream>>>(rows_from<T>(a, first));
        });
    });
    return launch_status();
}
