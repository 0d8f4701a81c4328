// Log probabilities of given tokens under rows of logits, with the entropy and the most likely tokens, and their gradient.
//
//   lse = log sum_i exp(x_i),  logprob = x_t - lse,  entropy = lse - sum_i p_i x_i,  p_i = exp(x_i - lse)
//   dx_i = a (1[i = t] - p_i) - b p_i (log p_i + entropy)   for the gradients a of logprob and b of entropy
//
// Bound by the reads: the logits are read once, with a running reference m, sum s = sum 2^d and sum u = sum 2^d d, where
// d = (x - m) log2(e), from which lse - m = ln 2 log2 s and entropy = ln 2 (log2 s - u / s).  The reference is any value near the
// largest: it is moved only when a value exceeds it by kStale.  The difference is taken before the product with log2(e): logits
// far from zero lose nothing, and those at the type's lowest value, whose product would overflow, are as good as any.
//
// Most likely tokens: the k-th largest of the threads' own largest values is a lower bound of the row's k-th largest value, so
// that few others reach it; those that do are collected in a second look at the row and put in order by counting.  Equal logits
// come in the order of their indexes.  Rows in which too many reach the bound (constant ones) are searched value by value.
#include <type_traits>

#include "kvmix_common.h"

namespace kvmix {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kScoreThreads = 256, kScoreWaves = kScoreThreads / kWave;
constexpr int kTopMost = 64, kCandidates = 1024;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;
constexpr float kStale = 20.0f;  // how far a value may exceed the reference: 2^d stays below 2^29

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

// Values of a row by sixteen bytes where it is aligned to them, one by one before and after: f(index, values, how many).
template <typename T, typename F>
__device__ __forceinline__ void each_value(const T *row, int begin, int end, F f)
{
    constexpr int PER = 16 / sizeof(T);
    const int skew = (int)((uintptr_t)(row + begin) / sizeof(T) % PER);
    const int body = min(end, begin + (skew ? PER - skew : 0)), tail = body + (end - body) / PER * PER;
    float v[PER];
    if (begin + (int)threadIdx.x < body) {
        v[0] = to_float(row[begin + threadIdx.x]);
        f(begin + (int)threadIdx.x, v, std::integral_constant<int, 1>());
    }
    for (int i = body + threadIdx.x * PER; i < tail; i += kScoreThreads * PER) {
        union {
            uint4v raw;
            T t[PER];
        } w;
        w.raw = *(const uint4v *)(row + i);
#pragma unroll
        for (int j = 0; j < PER; j++) v[j] = to_float(w.t[j]);
        f(i, v, std::integral_constant<int, PER>());
    }
    if (tail + (int)threadIdx.x < end) {
        v[0] = to_float(row[tail + threadIdx.x]);
        f(tail + (int)threadIdx.x, v, std::integral_constant<int, 1>());
    }
}

__device__ __forceinline__ ScoreStats merged(ScoreStats a, ScoreStats b)
{
    // (references of -inf: nothing summed yet; the difference is kept finite, so that nothing times it is nothing)
    const float m = fmaxf(a.m, b.m);
    const float da = fmaxf((a.m - m) * kLog2e, -1e30f), db = fmaxf((b.m - m) * kLog2e, -1e30f);
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

struct TopShared {
    uint32_t most[kScoreThreads];
    uint64_t key[kCandidates];
    uint64_t best[kScoreWaves];
    int count;
    uint32_t bound;
};

// The `top` first keys among `count` in key[], in order, to out[] (padded with zeros).
__device__ __forceinline__ void rank_keys(const uint64_t *key, int count, int top, uint64_t *out)
{
    for (int i = threadIdx.x; i < count; i += kScoreThreads) {
        const uint64_t mine = key[i];
        int rank = 0;
        for (int j = 0; j < count && rank < top; j++) rank += key[j] > mine;
        if (rank < top) out[rank] = mine;
    }
    for (int i = count + threadIdx.x; i < top; i += kScoreThreads) out[i] = 0;
}

// The `top` first keys of row[begin, end): to out[] (shared or global memory).  `largest`: this thread's largest value.
template <typename T>
__device__ void top_of(const T *row, int begin, int end, int top, float largest, TopShared &sh, uint64_t *out)
{
    sh.most[threadIdx.x] = value_key(largest);
    if (threadIdx.x == 0) sh.count = 0;
    __syncthreads();
    // the top-th largest of the threads' largest: the value that fewer than `top` exceed
    {
        const uint32_t mine = sh.most[threadIdx.x];
        int above = 0, equal = 0;
        for (int j = 0; j < kScoreThreads; j++) {
            above += sh.most[j] > mine;
            equal += sh.most[j] == mine;
        }
        if (above < top && above + equal >= top) sh.bound = mine;
    }
    __syncthreads();
    const uint32_t bound = sh.bound;
    each_value(row, begin, end, [&](int i, const float *v, auto n) {
#pragma unroll
        for (int j = 0; j < n.value; j++) {
            if (value_key(v[j]) >= bound) {
                const int at = atomicAdd(&sh.count, 1);
                if (at < kCandidates) sh.key[at] = full_key(v[j], i + j);
            }
        }
    });
    __syncthreads();
    const int count = sh.count;
    if (count <= kCandidates) {
        rank_keys(sh.key, count, top, out);
        return;
    }
    // too many: the next key below the last one, `top` times
    uint64_t last = ~(uint64_t)0;
    for (int k = 0; k < top; k++) {
        uint64_t best = 0;
        each_value(row, begin, end, [&](int i, const float *v, auto n) {
#pragma unroll
            for (int j = 0; j < n.value; j++) {
                const uint64_t key = full_key(v[j], i + j);
                if (key < last && key > best) best = key;
            }
        });
        for (int o = 32; o; o /= 2) {
            const uint64_t other = __shfl_xor((unsigned long long)best, o);
            best = other > best ? other : best;
        }
        __syncthreads();
        if (threadIdx.x % kWave == 0) sh.best[threadIdx.x / kWave] = best;
        __syncthreads();
        for (int w = 0; w < kScoreWaves; w++) best = sh.best[w] > best ? sh.best[w] : best;
        if (threadIdx.x == 0) out[k] = best;
        last = best;
    }
}

// A row's results from its sums: by one thread.  x_t: the target's logit, read again.
template <typename T>
__device__ __forceinline__ float finish_row(const ScoreArgs &a, int row, ScoreStats t)
{
    float sum2 = log2f(t.s), entropy = kLn2 * (log2f(t.s) - t.u / t.s);
    if (t.m == __builtin_inff() || !(t.s > 0.0f)) sum2 = entropy = __builtin_nanf("");
    const int64_t target = a.targets[row];
    const float x = target >= 0 && target < a.vocab ? to_float(((const T *)a.x)[row * a.row_stride + target]) : __builtin_nanf("");
    a.logprob[row] = target < 0 ? 0.0f : (x - t.m) - kLn2 * sum2;
    a.entropy[row] = entropy;
    if (a.stats) {
        float *s = a.stats + 4 * (int64_t)row;
        s[0] = t.m, s[1] = sum2, s[2] = entropy, s[3] = 0.0f;
    }
    return sum2;
}

__device__ __forceinline__ void write_top(const ScoreArgs &a, int row, const uint64_t *keys, float m, float sum2)
{
    for (int i = threadIdx.x; i < a.top; i += kScoreThreads) {
        const uint64_t key = keys[i];
        a.top_logprob[(int64_t)row * a.top + i] = (key_value((uint32_t)(key >> 32)) - m) - kLn2 * sum2;
        a.top_id[(int64_t)row * a.top + i] = (int64_t)~(uint32_t)key;
    }
}

template <typename T, bool TOP>
__global__ void __launch_bounds__(kScoreThreads) score_rows(ScoreArgs a)
{
    __shared__ ScoreStats wave_stats[kScoreWaves];
    __shared__ uint32_t wave_nan[kScoreWaves];
    __shared__ TopShared sh;
    __shared__ uint64_t best[kTopMost];
    __shared__ float done[2];
    const int row = blockIdx.x / a.chunks, nth = blockIdx.x % a.chunks;
    const int begin = nth * a.chunk, end = min(a.vocab, begin + a.chunk);
    const T *x = (const T *)a.x + row * a.row_stride;
    ScoreStats t = {-__builtin_inff(), 0.0f, 0.0f};
    float largest = -__builtin_inff();
    bool nan = false;
    each_value(x, begin, end, [&](int, const float *v, auto n) {
        float most = v[0];
#pragma unroll
        for (int j = 0; j < n.value; j++) most = fmaxf(most, v[j]), nan |= v[j] != v[j];
        if constexpr (TOP) largest = fmaxf(largest, most);
        if (most > t.m + kStale) {  // (also what leaves -inf)
            const float d = fmaxf((t.m - most) * kLog2e, -1e30f), f = __builtin_amdgcn_exp2f(d);
            t.u = (t.u + t.s * d) * f, t.s *= f, t.m = most;
        }
#pragma unroll
        for (int j = 0; j < n.value; j++) {
            const float d = fmaxf((v[j] - t.m) * kLog2e, -1e30f), e = __builtin_amdgcn_exp2f(d);  // (-inf, and -inf against -inf: nothing)
            t.s += e;
            t.u = fmaf(e, d, t.u);
        }
    });
    for (int o = 1; o < kWave; o *= 2) t = merged(t, {__shfl_xor(t.m, o), __shfl_xor(t.s, o), __shfl_xor(t.u, o)});
    if (threadIdx.x % kWave == 0) wave_stats[threadIdx.x / kWave] = t;
    const uint64_t any_nan = __ballot(nan);
    if (threadIdx.x % kWave == 0) wave_nan[threadIdx.x / kWave] = any_nan != 0;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < kScoreWaves; w++) t = merged(t, wave_stats[w]), wave_nan[0] |= wave_nan[w];
        if (wave_nan[0]) t.s = __builtin_nanf("");
        if (a.chunks == 1) done[0] = t.m, done[1] = finish_row<T>(a, row, t);
        else a.part[(int64_t)row * a.chunks + nth] = t;
    }
    if constexpr (TOP) {
        if (a.chunks > 1) {
            top_of(x, begin, end, a.top, largest, sh, a.part_keys + ((int64_t)row * a.chunks + nth) * a.top);
        } else {
            top_of(x, begin, end, a.top, largest, sh, best);
            __syncthreads();
            write_top(a, row, best, done[0], done[1]);
        }
    }
}

// The chunks of a row together.
template <typename T, bool TOP>
__global__ void __launch_bounds__(kScoreThreads) score_join(ScoreArgs a)
{
    __shared__ uint64_t key[TOP ? kCandidates * 2 : 1], best[kTopMost];
    __shared__ float done[2];
    const int row = blockIdx.x;
    if (threadIdx.x < kWave) {
        ScoreStats t = {-__builtin_inff(), 0.0f, 0.0f};
        for (int i = threadIdx.x; i < a.chunks; i += kWave) t = merged(t, a.part[(int64_t)row * a.chunks + i]);
        for (int o = 1; o < kWave; o *= 2) t = merged(t, {__shfl_xor(t.m, o), __shfl_xor(t.s, o), __shfl_xor(t.u, o)});
        if (threadIdx.x == 0) done[0] = t.m, done[1] = finish_row<T>(a, row, t);
    }
    if constexpr (TOP) {
        const int count = a.chunks * a.top;
        for (int i = threadIdx.x; i < count; i += kScoreThreads) key[i] = a.part_keys[(int64_t)row * count + i];
        __syncthreads();
        rank_keys(key, count, a.top, best);
        __syncthreads();
        write_top(a, row, best, done[0], done[1]);
    }
}

template <typename T>
__global__ void __launch_bounds__(kScoreThreads) score_grad(ScoreArgs a)
{
    constexpr int PER = 16 / sizeof(T);
    const int row = blockIdx.x / a.chunks, nth = blockIdx.x % a.chunks;
    const int begin = nth * a.chunk, end = min(a.vocab, begin + a.chunk);
    const T *x = (const T *)a.x + row * a.row_stride;
    T *dx = (T *)a.dx + row * a.dx_stride;
    const float *s = a.stats + 4 * (int64_t)row;
    const float m = s[0], sum2 = s[1], entropy = s[2];
    const int64_t target = a.targets[row];
    const float ga = a.grad_logprob && target >= 0 ? a.grad_logprob[row] : 0.0f, gb = a.grad_entropy ? a.grad_entropy[row] : 0.0f;
    auto one = [&](int i, float v) {
        const float q = fmaxf(fmaf(v - m, kLog2e, -sum2), -1e30f), p = __builtin_amdgcn_exp2f(q);
        const float g = -p * (ga + gb * (q * kLn2 + entropy));
        return i == target ? g + ga : g;
    };
    // (rows of dx and of x may be aligned differently: stores as wide as both allow)
    const bool wide = (((uintptr_t)(x + begin) | (uintptr_t)(dx + begin)) & 15) == 0;
    const int body = wide ? begin + (end - begin) / PER * PER : begin;
    for (int i = begin + threadIdx.x * PER; i < body; i += kScoreThreads * PER) {
        union {
            uint4v raw;
            T t[PER];
        } w;
        w.raw = *(const uint4v *)(x + i);
#pragma unroll
        for (int j = 0; j < PER; j++) w.t[j] = (T)one(i + j, to_float(w.t[j]));
        *(uint4v *)(dx + i) = w.raw;
    }
    for (int i = body + threadIdx.x; i < end; i += kScoreThreads) dx[i] = (T)one(i, to_float(x[i]));
}

namespace {

constexpr int64_t kScoreBlocks = 512;  // blocks that a launch over few rows is cut into ...
constexpr int64_t kScoreChunk = 1024;  // ... of that many values at least
constexpr int64_t kGradChunk = 8192;

// Chunks of a row: one, as long as there are rows enough; as many as their most likely tokens' list holds at most.
int64_t score_chunks(int64_t rows, int64_t vocab, int64_t top)
{
    int64_t n = rows ? kScoreBlocks / rows : 1;
    n = n < 1 ? 1 : n;
    const int64_t most = (vocab + kScoreChunk - 1) / kScoreChunk;
    n = n < most ? n : most;
    if (top > 0 && n > 2 * kCandidates / top) n = 2 * kCandidates / top;
    return n;
}

int64_t chunk_of(int64_t vocab, int64_t chunks) { return ((vocab + chunks - 1) / chunks + 7) / 8 * 8; }

int score_check(const kvmix_token_logprobs_t *p)
{
    if (!p) return KVMIX_ERR_NULL;
    if (p->dtype != KVMIX_F16 && p->dtype != KVMIX_F32 && p->dtype != KVMIX_BF16) return KVMIX_ERR_DTYPE;
    if (p->rows < 0 || p->vocab < 0 || p->top < 0 || (p->rows > 1 && p->row_stride < p->vocab)) return KVMIX_ERR_SHAPE;
    if (p->top > kTopMost || p->top > p->vocab || p->vocab > (1 << 30) || p->vocab == 0) return KVMIX_ERR_UNSUPPORTED;
    if ((__int128)p->rows * ((p->vocab + kScoreChunk - 1) / kScoreChunk) > 0x7fffffff) return KVMIX_ERR_UNSUPPORTED;
    return KVMIX_OK;
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
    const int64_t n = score_chunks(p->rows, p->vocab, p->top);
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
    a.chunks = (int)score_chunks(p->rows, p->vocab, p->top);
    a.chunk = (int)chunk_of(p->vocab, a.chunks);
    a.part_keys = (uint64_t *)workspace;
    a.part = (ScoreStats *)((uint64_t *)workspace + p->rows * a.chunks * p->top);
    hipStream_t st = (hipStream_t)stream;
    with_type(p->dtype, [&](auto zero) {
        using T = decltype(zero);
        const unsigned grid = (unsigned)(p->rows * a.chunks);
        if (p->top) score_rows<T, true><<<grid, kScoreThreads, 0, st>>>(a);
        else score_rows<T, false><<<grid, kScoreThreads, 0, st>>>(a);
        if (a.chunks > 1) {
            if (p->top) score_join<T, true><<<(unsigned)p->rows, kScoreThreads, 0, st>>>(a);
            else score_join<T, false><<<(unsigned)p->rows, kScoreThreads, 0, st>>>(a);
        }
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
    with_type(p->dtype, [&](auto zero) { score_grad<decltype(zero)><<<(unsigned)(p->rows * a.chunks), kScoreThreads, 0, (hipStream_t)stream>>>(a); });
    return launch_status();
}
