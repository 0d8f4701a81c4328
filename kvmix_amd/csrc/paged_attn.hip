// Attention of a batch's newest tokens, one or many of each sequence, over its paged cache: packed pages first, fp16 pages after
// them (paged_common.h).  out_i = sum_j softmax_j(scale q_i . k_j) v_j over the tokens j of i's sequence up to itself; one pass
// over the tokens with a running maximum and sum, values of codes in registers or in the LDS only.
//
// The query heads of a kv head and the new tokens of a sequence are the rows of one problem: row r is token r / G, head r % G of
// the group.  Sequences of few rows go to paged_few (bound by the reads of the cache), the others to paged_tile (bound by the
// matrix cores and the vector ALU beside them); both take spans of a sequence, so that a long one with few rows fills the chip,
// and paged_join puts the spans together.  Who takes what is decided on the host, once for all layers of a step
// (kvmix_paged_plan): lengths that differ within a batch then cost no idle blocks.
#include <algorithm>
#include <functional>
#include <new>
#include <vector>

#include "paged_common.h"

namespace kvmix {

typedef float floatx16 __attribute__((ext_vector_type(16)));

// sequence, first row, rows, first and last block (tile), part (-1: the whole sequence); of the sequence: first new token, new
// tokens, tokens, packed tokens (here, so that what a block needs is one load away); in paged_few, with the first item of a block,
// how many it has and where the others begin
constexpr int kItemWords = 12;
constexpr int kTileRows = 128, kTileKeys = 64;
constexpr float kLog2e = 1.44269504088896340736f;
// Probabilities are halves relative to 2^-kAbove of the largest, so that one of 2^-31 of it still is a number (from 1 on, those
// below 2^-25 were none: 100000 tokens just below that, 2.6e-3 of the mass together, went missing).  The reference may lag behind
// a larger one by kLag in all: 2^15 is well inside fp16's range.
constexpr float kAbove = 7.0f, kLag = 15.0f;

struct PagedArgs {
    const _Float16 *q;
    _Float16 *out;
    int64_t q_ts, q_hs, o_ts, o_hs;
    const _Float16 *rows;
    const uint32_t *packed;
    PlanWords table, items;
    int table_stride, kv_heads, group, blocks_log2;  // blocks_log2: of 32 tokens to a page
    float scale;                                     // with log2(e)
    float *part;                                     // [kv heads][part_rows][D], relative to the reference in part_ml
    float2 *part_ml;                                 // [kv heads][part_rows] reference (of log2) and sum
    int64_t part_rows;
};

struct PagedItem {
    int seq, row0, rows, begin, end, part, q_start, q_len, kv_len, packed, items, next;
};

__device__ __forceinline__ PagedItem item_of(PlanWords items, int nth)
{
    const PlanWords p = items + nth * kItemWords;
    return {p[0], p[1], p[2], p[3], p[4], p[5], p[6], p[7], p[8], p[9], p[10], p[11]};
}

// the larger of a lane's and those of the lanes with its place in the other rows of sixteen
__device__ __forceinline__ float max_of_rows(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}

__device__ __forceinline__ float sum_of_rows(float v)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    const auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// Values that are no numbers.  The products are made for whole blocks of tokens, and zero times an infinite value of a token that
// a row does not see is not zero.  So the values of blocks that not every new token sees wholly are looked through; where one is
// infinite or NaN, a finite one goes into the products instead, and which token first brings such a value to a channel is kept
// here, to be added to the results of the rows that see it.
template <int D>
struct Beyond {
    int first[3][D];  // +inf, -inf, NaN
    int any;

    // by `count` threads
    __device__ __forceinline__ void clear(int thread, int count)
    {
#pragma unroll
        for (int i = thread; i < 3 * D; i += count) first[0][i] = 0x7fffffff;
        if (thread == 0) any = 0;
    }

    // value `bits` of a token and channel
    __device__ __forceinline__ void note(uint32_t bits, int token, int channel)
    {
        if ((bits & 0x7c00u) != 0x7c00u) return;
        atomicMin(&first[bits & 0x3ffu ? 2 : bits >> 15][channel], token);
        any = 1;
    }

    // what to add to channel c of a row that sees the tokens up to `limit`
    __device__ __forceinline__ float of(int c, int limit) const
    {
        const bool up = first[0][c] <= limit, down = first[1][c] <= limit;
        return first[2][c] <= limit || (up && down) ? __builtin_nanf("") : up ? __builtin_inff() : down ? -__builtin_inff() : 0.0f;
    }
};

// NaN from the first infinite value or NaN on
__device__ __forceinline__ float beyond_sum(uint32_t pair, float sum)
{
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2v, pair), half2v{(_Float16)0.0f, (_Float16)0.0f}, sum, false);
}

// A packed block as a lane holds it: its codes, and its share of the scales and minima, which go through the LDS to the lanes
// that need them (each is wanted by sixteen).
template <int D, int KB, int VB>
struct PackedBlock {
    uint32_t k[lane_words(D, KB)], v[lane_words(D, VB)], side[D / 32];
};

template <int D, int KB, int VB>
__device__ __forceinline__ void load_packed(PackedBlock<D, KB, VB> &b, const uint32_t *at, int lane)
{
    load_words<lane_words(D, KB)>(at, lane, b.k);
    load_words<lane_words(D, VB)>(at + D * KB, lane, b.v);
    load_words<D / 32>(at + D * (KB + VB), lane, b.side);
}

// Few rows.  A block works through the items of its column (parts of sequences that add up to the same number of tokens for every
// column).  Every wave takes every fourth block of 32 tokens of an item's span, sixteen (NR times) rows of queries
// at once, with v_mfma_f32_16x16x32: the logits transposed (tokens as rows of the result), so that a lane holds those of one query
// and its probabilities are the operand of out^T = v^T p^T as they are.  Codes go from memory to registers, DEPTH blocks ahead, become
// fp16 there and are used once.
//
// q.k = sum_d (q_d s_d) c_d + q_d z_d with a channel's scale s and minimum z: the scales go to the queries (a product per block,
// row and channel, not per code), in two halves, so that the logits of packed keys are exact but for the sums (with
// one half the error of the whole against 64 bits was 1.2 to 1.5e-3, with keys rounded to fp16 4e-4, with two 2.7 to 3.2e-4; a result's
// own rounding is 2.1e-4.  For sixteen rows it costs 5 us of 70, for 32 rows, 16 x 16384 tokens of 8 heads, 12 of 67).
//
// Bound by vector instructions and memory together: 16 x 8192 tokens of 32 heads, 2/2 bits, 64 us (314 MB, 4.9 TB/s; a byte of
// codes is four values to convert; the vector ALU is at work for 65 % of the time, the matrix cores for 28), 4/4 bits 94 us (490 MB,
// 5.2 TB/s), 3/2 bits of 8 heads over 32768 tokens 73 us (4.6 TB/s; 69 and 27 %).
//
// LATER: whether values may be infinite in tokens that some row does not see, which takes a sequence of several new tokens.  Where
// there is none the kernel is made without looking for them: at 168 registers it costs 0 to 8 % (16 x 8192 tokens, 3/1 bits, 86.4
// instead of 93.3 us; 2/2 bits 79 both).
template <int D, int KB, int VB, int NR, bool LATER>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(NR == 1 ? 3 : 2))) paged_few(PagedArgs a)
{
    constexpr int KS = D / 32, DT = D / 16, NK = lane_words(D, KB), NV = lane_words(D, VB);
    constexpr int DEPTH = KB + VB > 5 ? 2 : KB + VB + NR > 4 ? 3 : 4;  // blocks in flight: what the registers hold (4/4 bits, 16 x 8192 tokens: 96 us, with three 99)
    // whether keys' channels, and values' tokens, are taken in the order in which two- and four-bit codes come cheapest (a lane then
    // has whole pieces of scales and minima, D = 128)
    constexpr bool kTurnK = KB % 2 == 0 && D == 128, kTurnV = VB % 2 == 0 && D == 128;
    constexpr int kPad = D + 4;
    __shared__ union {
        uint32_t side[4][2 * D];
        struct {
            float out[4][16 * NR][kPad];
            float2 ml[4][16 * NR];
        } join;
    } lds;
    __shared__ typename std::conditional<LATER, Beyond<D>, int>::type beyond[4];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), m = lane % 16, g = lane / 16;
    const int head = blockIdx.x % a.kv_heads, column = blockIdx.x / a.kv_heads;
    const int per_page = 1 << a.blocks_log2;
    const Exponents<KB> ke;
    const Exponents<VB> ve;

    PagedItem it = item_of(a.items, column);
    const int items = it.items, next = it.next;
    for (int nth = 0; nth < items; nth++) {
        if (nth) it = item_of(a.items, next + nth - 1);
        const int q_start = it.q_start, q_len = it.q_len, kv_len = it.kv_len, packed = it.packed;
        const PlanWords table = a.table + it.seq * a.table_stride;
        if constexpr (LATER) beyond[wave].clear(lane, kWave);

        half8v q[NR][KS];
        int limit[NR];  // the row's own token
        float scale[NR];
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const int r = it.row0 + min(16 * n + m, it.rows - 1), token = r / a.group;
            limit[n] = kv_len - q_len + token;
            const _Float16 *at = a.q + (int64_t)(q_start + token) * a.q_ts + (int64_t)(head * a.group + r % a.group) * a.q_hs + 8 * g;
#pragma unroll
            for (int s = 0; s < KS; s++) {
                q[n][s] = *(const half8v *)(at + 32 * s);
                if constexpr (kTurnK) q[n][s] = turned(q[n][s]);
            }
        }
        // A row's queries times the power of two that puts the largest into [0.5, 1): their products with the keys' scales are then
        // finite whatever both are, and small queries keep their bits.
#pragma unroll
        for (int n = 0; n < NR; n++) {
            half8v most = q[n][0] < (_Float16)0.0f ? -q[n][0] : q[n][0];
#pragma unroll
            for (int s = 1; s < KS; s++) most = __builtin_elementwise_max(most, q[n][s] < (_Float16)0.0f ? -q[n][s] : q[n][s]);
            float largest = (float)most[0];
#pragma unroll
            for (int j = 1; j < 8; j++) largest = fmaxf(largest, (float)most[j]);
            const int e = min(max((int)(__float_as_uint(max_of_rows(largest)) >> 23) - 126, -24), 16);
            const _Float16 once = (_Float16)__builtin_ldexpf(1.0f, -e / 2), twice = (_Float16)__builtin_ldexpf(1.0f, -e - -e / 2);
#pragma unroll
            for (int s = 0; s < KS; s++) q[n][s] = q[n][s] * once * twice;
            scale[n] = __builtin_ldexpf(a.scale, e);
        }
        const int first_limit = kv_len - q_len + it.row0 / a.group;

        floatx4 acc[NR][DT];
        float top[NR], sum[NR];
#pragma unroll
        for (int n = 0; n < NR; n++) {
            top[n] = -1e30f, sum[n] = 0.0f;
#pragma unroll
            for (int t = 0; t < DT; t++) acc[n][t] = floatx4{};
        }

        // a block's logits to probabilities, relative to a reference that is moved when some row's largest is kLag above it
        auto probabilities = [&](floatx4 (&x)[2][NR], half8v (&p)[NR], int block, auto packed_tokens) {
            if (!packed_tokens.value && block * kBlock + kBlock - 1 > first_limit) {  // (every new token sees all packed ones)
#pragma unroll
                for (int n = 0; n < NR; n++) {
#pragma unroll
                    for (int i = 0; i < 8; i++)
                        if (block * kBlock + 8 * g + i > limit[n]) x[i / 4][n][i % 4] = -__builtin_inff();
                }
            }
#pragma unroll
            for (int n = 0; n < NR; n++) {
                float most = x[0][n][0];
#pragma unroll
                for (int i = 1; i < 8; i++) most = fmaxf(most, x[i / 4][n][i % 4]);
                most *= scale[n];
                if (__any(most > top[n] + kLag)) {
                    const float grown = fmaxf(top[n], max_of_rows(most) - kAbove);
                    const float shrink = __builtin_amdgcn_exp2f(top[n] - grown);
                    top[n] = grown;
                    sum[n] *= shrink;
#pragma unroll
                    for (int t = 0; t < DT; t++) acc[n][t] *= shrink;
                }
#pragma unroll
                for (int i = 0; i < 8; i++) {
                    const int t = kTurnV && packed_tokens.value ? i / 2 + i % 2 * 4 : i;  // (the order of the values' tokens)
                    p[n][i] = (_Float16)__builtin_amdgcn_exp2f(fmaf(x[t / 4][n][t % 4], scale[n], -top[n]));
                    if (i % 2) sum[n] = __builtin_amdgcn_fdot2(half2v{p[n][i - 1], p[n][i]}, half2v{(_Float16)1.0f, (_Float16)1.0f}, sum[n], false);
                }
            }
        };

        auto key_codes = [&](const PackedBlock<D, KB, VB> &b, int piece) {
            if constexpr (kTurnK) return piece_codes_turned<KB>(b.k, piece);
            else return piece_codes<KB, NK>(b.k, piece, ke);
        };
        auto value_codes = [&](const PackedBlock<D, KB, VB> &b, int piece) {
            if constexpr (kTurnV) return piece_codes_turned<VB>(b.v, piece);
            else return piece_codes<VB, NV>(b.v, piece, ve);
        };
        auto take_packed = [&](const PackedBlock<D, KB, VB> &b) {
            uint32_t *side = lds.side[wave];
            if constexpr (kTurnK || kTurnV) {  // (lanes 0 .. 31 have the keys', the others the values')
                const half8v natural = __builtin_bit_cast(half8v, uint4v{b.side[0], b.side[1], b.side[2], b.side[3]}), other = turned(natural);
                const bool turn = kTurnK && kTurnV ? true : kTurnV == (lane >= 32);
                *(uint4v *)(side + 4 * lane) = turn ? __builtin_bit_cast(uint4v, other) : __builtin_bit_cast(uint4v, natural);
            } else {
                store_words<D / 32>(side, lane, b.side);
            }
            __builtin_amdgcn_wave_barrier();  // (a wave's LDS operations are done in order)
            const _Float16 *sides = (const _Float16 *)side + 8 * g;
            floatx4 x[2][NR] = {}, low[2][NR] = {};  // (sums of their own: half as long a chain of products)
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const half8v zeros = *(const half8v *)(sides + D + 32 * s);
#pragma unroll
                for (int n = 0; n < NR; n++) low[0][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(zeros, q[n][s], low[0][n], 0, 0, 0);
            }
#pragma unroll
            for (int n = 0; n < NR; n++) low[1][n] = low[0][n];
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const half8v scales = *(const half8v *)(sides + 32 * s);
                // in two halves, the product and what it rounds off: the logits are then exact but for the sums
                half8v scaled[NR], rest[NR];
#pragma unroll
                for (int n = 0; n < NR; n++) scaled[n] = q[n][s] * scales, rest[n] = __builtin_elementwise_fma(q[n][s], scales, -scaled[n]);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const half8v codes = key_codes(b, u * KS + s);
#pragma unroll
                    for (int n = 0; n < NR; n++) {
                        low[u][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, rest[n], low[u][n], 0, 0, 0);
                        x[u][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes, scaled[n], x[u][n], 0, 0, 0);
                    }
                }
            }
#pragma unroll
            for (int u = 0; u < 2; u++) {
#pragma unroll
                for (int n = 0; n < NR; n++) x[u][n] += low[u][n];
            }
            half8v p[NR];
            probabilities(x, p, 0, std::true_type());
#pragma unroll
            for (int s = 0; s < KS; s++) {
                const half8v scales = *(const half8v *)(sides + 2 * D + 32 * s), zeros = *(const half8v *)(sides + 3 * D + 32 * s);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const half8v v = __builtin_elementwise_fma(value_codes(b, 2 * s + u), scales, zeros);
#pragma unroll
                    for (int n = 0; n < NR; n++) acc[n][2 * s + u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v, p[n], acc[n][2 * s + u], 0, 0, 0);
                }
            }
            __builtin_amdgcn_wave_barrier();
        };

        const int packed_end = min(it.end, packed / kBlock);
        int block = it.begin + wave;
        if (block < packed_end) {
            // The coming blocks are on their way while one is worked on.  Every turn loads one, past the end the last one again:
            // with the loads under a condition each use waited for all of them.
            const int last_block = packed_end - 1;
            auto page_of = [&](int block) { return table[min(block, last_block) >> a.blocks_log2]; };
            auto fetch = [&](PackedBlock<D, KB, VB> &to, int block, int page) {
                const int in_page = min(block, last_block) & (per_page - 1);
                load_packed(to, a.packed + ((((int64_t)page * a.kv_heads + head) << a.blocks_log2) + in_page) * block_words(D, KB, VB), lane);
            };
            PackedBlock<D, KB, VB> held[DEPTH];
#pragma unroll
            for (int i = 0; i < DEPTH; i++) fetch(held[i], block + 4 * i, page_of(block + 4 * i));
            int page = page_of(block + 4 * DEPTH);
            const int count = (packed_end - block + 3) / 4;
            for (int turn = 0; turn < count / DEPTH; turn++) {
#pragma unroll
                for (int i = 0; i < DEPTH; i++) {
                    take_packed(held[i]);
                    fetch(held[i], block + 4 * DEPTH, page);
                    block += 4;
                    page = page_of(block + 4 * DEPTH);
                }
            }
#pragma unroll
            for (int i = 0; i < DEPTH - 1; i++) {
                if (i < count % DEPTH) {
                    take_packed(held[i]);
                    block += 4;
                }
            }
        }
        if constexpr (kTurnK) {
#pragma unroll
            for (int n = 0; n < NR; n++) {
#pragma unroll
                for (int s = 0; s < KS; s++) q[n][s] = turned_back(q[n][s]);
            }
        }
        for (; block < it.end; block += 4) {
            const int64_t page = table[block >> a.blocks_log2];
            const int64_t P = kBlock << a.blocks_log2;
            const _Float16 *keys = a.rows + (page * a.kv_heads + head) * 2 * P * D + (block & (per_page - 1)) * kBlock * D;
            const _Float16 *values = keys + P * D;
            floatx4 x[2][NR] = {};
            half8v v[DT];
#pragma unroll
            for (int s = 0; s < KS; s++) {
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const half8v k = *(const half8v *)(keys + (8 * (m / 4) + 4 * u + m % 4) * D + 32 * s + 8 * g);
                    v[2 * s + u] = *(const half8v *)(values + (16 * (2 * s + u) + m) * kBlock + 8 * g);
#pragma unroll
                    for (int n = 0; n < NR; n++) x[u][n] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k, q[n][s], x[u][n], 0, 0, 0);
                }
            }
            if constexpr (LATER) if (block * kBlock + kBlock - 1 > first_limit) {
                float found = 0.0f;
#pragma unroll
                for (int t = 0; t < DT; t++) {
#pragma unroll
                    for (int j = 0; j < 4; j++) found = beyond_sum(__builtin_bit_cast(uint4v, v[t])[j], found);
                }
                if (__builtin_expect(__any(found != found), 0)) {
                    int from = lane;
                    asm volatile("" : "+v"(from));  // (nothing of this is worked out before)
#pragma unroll 1
                    for (int i = from; i < D * kBlock; i += kWave) {
                        const int token = block * kBlock + i % kBlock;
                        if (token < kv_len) beyond[wave].note(((const uint16_t *)values)[i], token, i / kBlock);
                    }
                    const half8v largest = (half8v)(_Float16)65504.0f;
#pragma unroll
                    for (int t = 0; t < DT; t++) v[t] = __builtin_elementwise_max(__builtin_elementwise_min(v[t], largest), -largest);
                }
            }
            half8v p[NR];
            probabilities(x, p, block, std::false_type());
            if (block * kBlock + kBlock > kv_len) {  // (whatever lies behind the last token: zero times it may not be zero)
#pragma unroll
                for (int t = 0; t < DT; t++) {
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (block * kBlock + 8 * g + j >= kv_len) v[t][j] = (_Float16)0.0f;
                }
            }
#pragma unroll
            for (int t = 0; t < DT; t++) {
#pragma unroll
                for (int n = 0; n < NR; n++) acc[n][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[t], p[n], acc[n][t], 0, 0, 0);
            }
        }

        // the four waves' sums together
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NR; n++) {
            const float total = sum_of_rows(sum[n]);
            if (g == 0) lds.join.ml[wave][16 * n + m] = make_float2(top[n], total);
        }
        __syncthreads();
#pragma unroll
        for (int n = 0; n < NR; n++) {
            float most = top[n];
#pragma unroll
            for (int w = 0; w < 4; w++) most = fmaxf(most, lds.join.ml[w][16 * n + m].x);
            const float shrink = __builtin_amdgcn_exp2f(top[n] - most);
#pragma unroll
            for (int t = 0; t < DT; t++) *(floatx4 *)&lds.join.out[wave][16 * n + m][16 * t + 4 * g] = acc[n][t] * shrink;
        }
        __syncthreads();
        for (int i = threadIdx.x; i < it.rows * (D / 8); i += 256) {
            const int r = i / (D / 8), c = i % (D / 8) * 8;
            float most = lds.join.ml[0][r].x, total = 0.0f;
#pragma unroll
            for (int w = 1; w < 4; w++) most = fmaxf(most, lds.join.ml[w][r].x);
            floatx4 o[2] = {};
#pragma unroll
            for (int w = 0; w < 4; w++) {
                total += lds.join.ml[w][r].y * __builtin_amdgcn_exp2f(lds.join.ml[w][r].x - most);
                o[0] += *(const floatx4 *)&lds.join.out[w][r][c];
                o[1] += *(const floatx4 *)&lds.join.out[w][r][c + 4];
            }
            if constexpr (LATER) if (__builtin_expect(beyond[0].any | beyond[1].any | beyond[2].any | beyond[3].any, 0)) {
                const int sees = kv_len - q_len + (it.row0 + r) / a.group;
#pragma unroll 1
                for (int w = 0; w < 4; w++) {
#pragma unroll
                    for (int j = 0; j < 8; j++) o[j / 4][j % 4] += beyond[w].of(c + j, sees);
                }
            }
            if (it.part >= 0) {
                const int64_t to = head * a.part_rows + it.part + r;
                *(floatx4 *)(a.part + to * D + c) = o[0];
                *(floatx4 *)(a.part + to * D + c + 4) = o[1];
                if (c == 0) a.part_ml[to] = make_float2(most, total);
            } else {
                const float inv = 1.0f / total;
                half8v w;
#pragma unroll
                for (int j = 0; j < 8; j++) w[j] = (_Float16)(o[j / 4][j % 4] * inv);
                const int token = (it.row0 + r) / a.group, h = head * a.group + (it.row0 + r) % a.group;
                *(half8v *)(a.out + (int64_t)(q_start + token) * a.o_ts + (int64_t)h * a.o_hs + c) = w;
            }
        }
        __syncthreads();  // (the next item's scales go where these sums are)
    }
}

// Where the pieces of a tile lie in the LDS, so that neither side has bank conflicts: keys [64][D] and values [D][64], 16-byte
// pieces exchanged by the row's low bits.
template <int D>
__device__ __forceinline__ int tile_key(int key, int c)
{
    return D == 128 ? key * 256 + ((c ^ (key & 15)) << 4) : key * 128 + ((c ^ ((key >> 1) & 7)) << 4);
}

__device__ __forceinline__ int tile_value(int channel, int c) { return channel * 128 + ((c ^ ((channel >> 1) & 7)) << 4); }

// Many rows: 128 of them to a block, 32 to a wave, over tiles of 64 tokens.  A tile is four matrices of 32 tokens, keys and values
// of two blocks; each wave turns one of them from codes to fp16, for all four.  Products with v_mfma_f32_32x32x16: logits
// transposed, keys as rows in an order in which a lane's logits are those of eight tokens that follow one another, as the
// values' pieces are.  Packed keys and values are rounded to fp16 once (code * scale + minimum): the matrix cores take no others at this rate.
//
// Bound by the matrix cores and, in turns with them, the vector ALU (exponentials 9 cycles each, conversions of codes): 4 chunks of 2048 tokens over
// 8192, 32 heads, 4/4 bits: 826 us, 831 TFLOP/s of the 1490 that a fp16 product of 16384 reaches; matrix cores at work for 41 % of the time,
// vector ALU for 52 (with the codes converted between tiles 855 us, on a box on which the others took 786).  Two blocks to a CU is what the LDS (66 KB each) and the registers (256) hold.
template <int D, int KB, int VB>
__global__ void __launch_bounds__(256) __attribute__((amdgpu_waves_per_eu(2, 2))) paged_tile(PagedArgs a)
{
    constexpr int KS = D / 16, DT = D / 32, NP = D / 16;
    constexpr int kBytes = kTileKeys * D * 2;
    __shared__ __attribute__((aligned(16))) uint8_t lds[2][2][kBytes];
    __shared__ uint32_t sides[4][D];
    __shared__ Beyond<D> beyond;
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), col = lane & 31, h2 = lane >> 5;
    const int m = lane % 16, g = lane / 16;
    const int head = blockIdx.x % a.kv_heads;
    const PagedItem it = item_of(a.items, blockIdx.x / a.kv_heads);
    const int q_start = it.q_start, q_len = it.q_len, kv_len = it.kv_len, packed_blocks = it.packed / kBlock, blocks = (kv_len + kBlock - 1) / kBlock;
    const PlanWords table = a.table + it.seq * a.table_stride;
    const int per_page = 1 << a.blocks_log2;
    beyond.clear(threadIdx.x, 256);  // (a barrier follows before fp16 pages are placed)

    const int own = 32 * wave + col, r = it.row0 + min(own, it.rows - 1), token = r / a.group, limit = kv_len - q_len + token;
    const int wave_first = kv_len - q_len + (it.row0 + min(32 * wave, it.rows - 1)) / a.group;
    const int wave_last = 32 * wave < it.rows ? kv_len - q_len + (it.row0 + min(32 * wave + 31, it.rows - 1)) / a.group : -1;
    half8v q[KS];
    {
        const _Float16 *at = a.q + (int64_t)(q_start + token) * a.q_ts + (int64_t)(head * a.group + r % a.group) * a.q_hs + 8 * h2;
#pragma unroll
        for (int s = 0; s < KS; s++) q[s] = *(const half8v *)(at + 16 * s);
    }

    // This wave's matrix of a tile: on its way from memory in `held`, then into the LDS.
    const int matrix = wave & 1, which = wave >> 1;
    uint32_t held[4 * NP], side[D / 64];
    auto fetch = [&](int tile) {
        const int block = 2 * tile + which;
        if (block >= blocks) return;
        const int64_t page = table[block >> a.blocks_log2];
        const int in_page = block & (per_page - 1);
        if (block < packed_blocks) {
            const uint32_t *at = a.packed + (((page * a.kv_heads + head) << a.blocks_log2) + in_page) * block_words(D, KB, VB);
            if (matrix) load_words<lane_words(D, VB)>(at + D * KB, lane, held);
            else load_words<lane_words(D, KB)>(at, lane, held);
            load_words<D / 64>(at + D * (KB + VB) + matrix * D, lane, side);
        } else {
            const int64_t P = kBlock << a.blocks_log2;
            const _Float16 *at = a.rows + (page * a.kv_heads + head) * 2 * P * D + (matrix ? P * D : 0) + (int64_t)in_page * kBlock * D;
#pragma unroll
            for (int p = 0; p < NP; p++) {
                const int off = matrix ? (16 * p + m) * kBlock + 8 * g : (8 * (m / 4) + 4 * (p / (D / 32)) + m % 4) * D + 32 * (p % (D / 32)) + 8 * g;
                *(uint4v *)&held[4 * p] = *(const uint4v *)(at + off);
            }
        }
    };
    auto place = [&](int tile, int buf) {
        const int block = 2 * tile + which;
        uint8_t *to = lds[buf][matrix];
        auto put = [&](int p, half8v x) {
            const int at = matrix ? tile_value(16 * p + m, 4 * which + g)
                                  : tile_key<D>(kBlock * which + 8 * (m / 4) + 4 * (p / (D / 32)) + m % 4, 4 * (p % (D / 32)) + g);
            *(half8v *)(to + at) = x;
        };
        if (block < packed_blocks) {
            store_words<D / 64>(sides[wave], lane, side);
            __builtin_amdgcn_wave_barrier();
            const _Float16 *s = (const _Float16 *)sides[wave] + 8 * g;
            auto turn = [&](auto bits) {
                constexpr int B = decltype(bits)::value;
                const Exponents<B> e;
#pragma unroll
                for (int p = 0; p < NP; p++) {
                    const int set = matrix ? p / 2 : p % (D / 32);
                    put(p, piece_values<B, lane_words(D, B)>(held, p, *(const half8v *)(s + 32 * set), *(const half8v *)(s + D + 32 * set), e));
                }
            };
            if (matrix) turn(std::integral_constant<int, VB>());
            else turn(std::integral_constant<int, KB>());
            __builtin_amdgcn_wave_barrier();
        } else if (block < blocks) {
            float found = 0.0f;
            if (matrix && block * kBlock + kBlock - 1 > kv_len - q_len) {
#pragma unroll
                for (int i = 0; i < 4 * NP; i++) found = beyond_sum(held[i], found);
            }
#pragma unroll
            for (int p = 0; p < NP; p++) {
                half8v x = __builtin_bit_cast(half8v, *(const uint4v *)&held[4 * p]);
                if (matrix && block * kBlock + kBlock > kv_len) {  // (zero times what lies behind the last token may not be zero)
#pragma unroll
                    for (int j = 0; j < 8; j++)
                        if (block * kBlock + 8 * g + j >= kv_len) x[j] = (_Float16)0.0f;
                }
                put(p, x);
            }
            if (__builtin_expect(__any(found != found), 0)) {  // (in the LDS: a wave's operations there are done in order)
                int row = m;
                asm volatile("" : "+v"(row));  // (nothing of this is worked out before)
#pragma unroll 1
                for (int p = 0; p < NP; p++, row += 16) {
                    _Float16 *at = (_Float16 *)(to + tile_value(row, 4 * which + g));
#pragma unroll 1
                    for (int j = 0; j < 8; j++) {
                        const uint32_t bits = __builtin_bit_cast(uint16_t, at[j]);
                        beyond.note(bits, block * kBlock + 8 * g + j, row);
                        if ((bits & 0x7c00u) == 0x7c00u) at[j] = (_Float16)0.0f;
                    }
                }
            }
        } else {
#pragma unroll
            for (int p = 0; p < NP; p++) put(p, half8v{});
        }
    };

    // where a lane reads: keys row R of 32 as token R with its bits 2 and 3 exchanged
    const int k_row = (col & 19) | (col & 4) << 1 | (col & 8) >> 1;
    floatx16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; t++) o[t] = floatx16{};
    float top = -1e30f, sum = 0.0f;

    auto key_piece = [&](int buf, int t, int s) { return *(const half8v *)(lds[buf][0] + tile_key<D>(32 * t + k_row, 2 * s + h2)); };
    auto value_piece = [&](int buf, int t, int kk) { return *(const half8v *)(lds[buf][1] + tile_value(32 * t + col, 2 * kk + h2)); };

    // A tile's logits to probabilities and their product with its values: x[t][8 kk + j] is the logit of token 32 t + 16 kk + 8 h2 + j.
    auto weigh = [&](floatx16 (&x)[2], int buf) {
        float most = x[0][0];
#pragma unroll
        for (int i = 1; i < 32; i++) most = fmaxf(most, x[i / 16][i % 16]);
        {
            const auto e = __builtin_amdgcn_permlane32_swap(__float_as_uint(most), __float_as_uint(most), false, false);
            most = fmaxf(__uint_as_float(e[0]), __uint_as_float(e[1])) * a.scale;
        }
        if (__any(most > top + kLag)) {
            const float grown = fmaxf(top, most - kAbove), shrink = __builtin_amdgcn_exp2f(top - grown);
            top = grown;
            sum *= shrink;
#pragma unroll
            for (int t = 0; t < DT; t++) o[t] *= shrink;
        }
        half8v p[2];
        auto probabilities = [&](int kk) {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                p[kk % 2][j] = (_Float16)__builtin_amdgcn_exp2f(fmaf(x[kk / 2][8 * (kk % 2) + j], a.scale, -top));
                if (j % 2) sum = __builtin_amdgcn_fdot2(half2v{p[kk % 2][j - 1], p[kk % 2][j]}, half2v{(_Float16)1.0f, (_Float16)1.0f}, sum, false);
            }
        };
        half8v v[DT], ahead[DT];
#pragma unroll
        for (int t = 0; t < DT; t++) v[t] = value_piece(buf, t, 0);
        probabilities(0);
#pragma unroll
        for (int kk = 0; kk < 4; kk++) {  // (a step's reads and probabilities between the products of the one before)
#pragma unroll
            for (int t = 0; t < DT; t++) {
                if (kk < 3) ahead[t] = value_piece(buf, t, kk + 1);
                o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[t], p[kk % 2], o[t], 0, 0, 0);
            }
            if (kk < 3) {
                probabilities(kk + 1);
                __builtin_amdgcn_sched_group_barrier(0x100, DT, 0);
#pragma unroll
                for (int t = 0; t < DT; t++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    __builtin_amdgcn_sched_group_barrier(0x402, 24 / DT, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int t = 0; t < DT; t++) v[t] = ahead[t];
        }
    };

    int tile = it.begin, buf = 0;
    const int packed_tiles = min(it.end, packed_blocks / 2);  // up to there both blocks of a tile are packed
    if (tile < packed_tiles) {
        // Tiles of codes whose successor is one of codes too: no masks, nothing under a condition, and the codes of the next tile
        // become values between the products of this one's keys.  One loop for the waves that turn keys and one for those that
        // turn values.
        auto run = [&](auto is_value) {
            constexpr bool V = is_value.value;
            constexpr int B = V ? VB : KB, N = lane_words(D, B);
            const Exponents<B> e;
            uint32_t w[N], sd[D / 64];
            auto page_of = [&](int tile) { return table[(2 * min(tile, packed_tiles - 1) + which) >> a.blocks_log2]; };
            auto load = [&](int tile, int page) {
                const int in_page = (2 * min(tile, packed_tiles - 1) + which) & (per_page - 1);
                const uint32_t *at = a.packed + ((((int64_t)page * a.kv_heads + head) << a.blocks_log2) + in_page) * block_words(D, KB, VB);
                load_words<N>(at + (V ? D * KB : 0), lane, w);
                load_words<D / 64>(at + D * (KB + VB) + (V ? D : 0), lane, sd);
            };
            const _Float16 *side_at = (const _Float16 *)sides[wave] + 8 * g;
            auto start = [&]() {
                store_words<D / 64>(sides[wave], lane, sd);
                __builtin_amdgcn_wave_barrier();  // (a wave's LDS operations are done in order)
            };
            struct Side {
                half8v scale, zero;
            };
            auto side_of = [&](int p) {
                const int set = V ? p / 2 : p % (D / 32);
                return Side{*(const half8v *)(side_at + 32 * set), *(const half8v *)(side_at + D + 32 * set)};
            };
            auto turn = [&](int p, int buf, const Side &side) {
                const half8v x = piece_values<B, N>(w, p, side.scale, side.zero, e);
                const int at = V ? tile_value(16 * p + m, 4 * which + g)
                                 : tile_key<D>(kBlock * which + 8 * (m / 4) + 4 * (p / (D / 32)) + m % 4, 4 * (p % (D / 32)) + g);
                *(half8v *)(lds[buf][V] + at) = x;
            };
            load(tile, page_of(tile));
            int page = page_of(tile + 1);
            start();
#pragma unroll
            for (int p = 0; p < NP; p++) turn(p, 0, side_of(p));
            load(tile + 1, page);
            page = page_of(tile + 2);
            __syncthreads();
            for (; tile < packed_tiles - 1; tile++) {
                start();
                if (wave_last >= 0) {
                    floatx16 x[2] = {floatx16{}, floatx16{}};
                    half8v k[2] = {key_piece(buf, 0, 0), key_piece(buf, 1, 0)};
                    Side side = side_of(0);
#pragma unroll
                    for (int s = 0; s < KS; s++) {  // (the LDS is read a step ahead)
                        half8v k_ahead[2];
                        Side side_ahead;
                        if (s + 1 < KS) {
                            side_ahead = side_of(s + 1);
                            k_ahead[0] = key_piece(buf, 0, s + 1), k_ahead[1] = key_piece(buf, 1, s + 1);
                        }
#pragma unroll
                        for (int t = 0; t < 2; t++) x[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[t], q[s], x[t], 0, 0, 0);
                        turn(s, buf ^ 1, side);
                        __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 9, 0);
                        __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(0x002, 9, 0);
                        __builtin_amdgcn_sched_barrier(0);
                        if (s + 1 < KS) k[0] = k_ahead[0], k[1] = k_ahead[1], side = side_ahead;
                    }
                    load(tile + 2, page);
                    page = page_of(tile + 3);
                    weigh(x, buf);
                } else {
#pragma unroll
                    for (int p = 0; p < NP; p++) turn(p, buf ^ 1, side_of(p));
                    load(tile + 2, page);
                    page = page_of(tile + 3);
                }
                buf ^= 1;
                __syncthreads();
            }
        };
        if (matrix) run(std::true_type());
        else run(std::false_type());
    } else {
        fetch(tile);
        __syncthreads();
        place(tile, 0);
        __syncthreads();
    }
    // the last of them, and those with tokens in fp16
    if (tile + 1 < it.end) fetch(tile + 1);
    for (; tile < it.end; tile++) {
        if (tile + 1 < it.end) place(tile + 1, buf ^ 1);  // (that buffer was last read before the barrier that ended the turn before)
        if (tile + 2 < it.end) fetch(tile + 2);
        const int k0 = tile * kTileKeys;
        if (k0 <= wave_last) {
            floatx16 x[2] = {floatx16{}, floatx16{}};
#pragma unroll
            for (int s = 0; s < KS; s++) {
#pragma unroll
                for (int t = 0; t < 2; t++) x[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(key_piece(buf, t, s), q[s], x[t], 0, 0, 0);
                if (s % 4 == 3) __builtin_amdgcn_sched_barrier(0);  // (all reads of a tile ahead of its products would spill)
            }
            if (k0 + kTileKeys - 1 > wave_first) {
#pragma unroll
                for (int i = 0; i < 32; i++)
                    if (k0 + 32 * (i / 16) + 16 * (i % 16 / 8) + 8 * h2 + i % 8 > limit) x[i / 16][i % 16] = -__builtin_inff();
            }
            weigh(x, buf);
        }
        buf ^= 1;
        __syncthreads();
    }
    if (__builtin_expect(beyond.any, 0)) {
#pragma unroll
        for (int t = 0; t < DT; t++) {
#pragma unroll
            for (int i = 0; i < 16; i++) o[t][i] += beyond.of(32 * t + 8 * (i / 4) + 4 * h2 + i % 4, limit);
        }
    }
    if (own >= it.rows) return;
    {
        const auto e = __builtin_amdgcn_permlane32_swap(__float_as_uint(sum), __float_as_uint(sum), false, false);
        sum = __uint_as_float(e[0]) + __uint_as_float(e[1]);
    }
    if (it.part >= 0) {
        const int64_t to = head * a.part_rows + it.part + own;
#pragma unroll
        for (int t = 0; t < DT; t++) {
#pragma unroll
            for (int i = 0; i < 4; i++)
                *(floatx4 *)(a.part + to * D + 32 * t + 8 * i + 4 * h2) = floatx4{o[t][4 * i], o[t][4 * i + 1], o[t][4 * i + 2], o[t][4 * i + 3]};
        }
        if (h2 == 0) a.part_ml[to] = make_float2(top, sum);
        return;
    }
    typedef _Float16 half4v __attribute__((ext_vector_type(4)));
    const float inv = 1.0f / sum;
    _Float16 *to = a.out + (int64_t)(q_start + token) * a.o_ts + (int64_t)(head * a.group + r % a.group) * a.o_hs + 4 * h2;
#pragma unroll
    for (int t = 0; t < DT; t++) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            half4v w;
#pragma unroll
            for (int j = 0; j < 4; j++) w[j] = (_Float16)(o[t][4 * i + j] * inv);
            *(half4v *)(to + 32 * t + 8 * i) = w;
        }
    }
}

// The spans of one sequence's rows together; the item's `begin` is the number of spans, `end` the rows between them.  A row's D sums
// are four to a lane; a row is a group of lanes, or where there are many spans all groups of the block, each for every GROUPS-th of
// them.  Eight spans' sums and maxima are asked for at once, the maximum runs along: one wait on memory, which is what bounds it
// (3 us for a few rows; 19392 rows in two or three spans, 25 MB, 9 us).
constexpr int kJoinAhead = 8;

template <int D>
__global__ void __launch_bounds__(256) paged_join(PagedArgs a)
{
    constexpr int LANES = D / 4, GROUPS = 256 / LANES;
    typedef _Float16 half4v __attribute__((ext_vector_type(4)));
    __shared__ floatx4 sums[GROUPS][LANES];
    __shared__ float2 stats[GROUPS];
    const int group = threadIdx.x / LANES, c = threadIdx.x % LANES;
    const int head = blockIdx.x % a.kv_heads;
    const PagedItem it = item_of(a.items, blockIdx.x / a.kv_heads);
    const int spans = it.begin;
    const bool shared = spans > kJoinAhead;
    const int step = shared ? GROUPS : 1, first_span = shared ? group : 0, rows = shared ? 1 : GROUPS;
    for (int r0 = blockIdx.y * rows; r0 < it.rows; r0 += gridDim.y * rows) {
        const int r = shared ? r0 : min(r0 + group, it.rows - 1);
        const int64_t first = head * a.part_rows + it.part + r;
        float top = -1e30f, total = 0.0f;
        floatx4 o = {};
        for (int i0 = first_span; i0 < spans; i0 += step * kJoinAhead) {
            float2 ml[kJoinAhead];
            floatx4 x[kJoinAhead];
#pragma unroll
            for (int i = 0; i < kJoinAhead; i++) {
                const int64_t at = first + (int64_t)min(i0 + i * step, spans - 1) * it.end;
                ml[i] = a.part_ml[at];
                x[i] = *(const floatx4 *)(a.part + at * D + 4 * c);
            }
            float most = top;
#pragma unroll
            for (int i = 0; i < kJoinAhead; i++) most = fmaxf(most, ml[i].x);  // (past the end: the last one's again)
            const float shrink = __builtin_amdgcn_exp2f(top - most);
            top = most, total *= shrink, o *= shrink;
#pragma unroll
            for (int i = 0; i < kJoinAhead; i++) {
                if (i0 + i * step < spans) {
                    const float w = __builtin_amdgcn_exp2f(ml[i].x - most);
                    total = fmaf(ml[i].y, w, total);
                    o += x[i] * w;
                }
            }
        }
        if (shared) {
            sums[group][c] = o;
            if (c == 0) stats[group] = make_float2(top, total);
            __syncthreads();
            float most = -1e30f;
#pragma unroll
            for (int i = 0; i < GROUPS; i++) most = fmaxf(most, stats[i].x);
            o = floatx4{}, total = 0.0f;
#pragma unroll
            for (int i = 0; i < GROUPS; i++) {
                const float w = __builtin_amdgcn_exp2f(stats[i].x - most);
                total = fmaf(stats[i].y, w, total);
                o += sums[i][c] * w;
            }
            __syncthreads();
        }
        if (shared ? group != 0 : r0 + group >= it.rows) continue;
        const float inv = 1.0f / total;
        const int row = it.row0 + r;
        half4v w;
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (_Float16)(o[j] * inv);
        *(half4v *)(a.out + (int64_t)(it.q_start + row / a.group) * a.o_ts + (int64_t)(head * a.group + row % a.group) * a.o_hs + 4 * c) = w;
    }
}

namespace {

constexpr int64_t kFewMost = 32;    // rows of a sequence and kv head that go to paged_few
constexpr int64_t kFewUnit = 4;     // blocks of tokens, one to a wave: what its launch is cut by ...
constexpr int64_t kFewLeast = 2;    // ... of which a column has that many at least
// Blocks of paged_few that the chip holds at once: three to a CU by their registers (sixteen rows), or two (32).
int64_t few_resident(int64_t rows) { return rows > 16 ? 512 : 768; }

// The same of paged_tile, and the tiles' worth of time that a block of it takes beside its tiles.
constexpr int64_t kTileResident = 512, kTileStart = 3;

int64_t up(int64_t n, int64_t m) { return (n + m - 1) / m * m; }

struct Span {
    int32_t word[6];
    int64_t cost;
    int32_t items = 0, next = 0;
};

// Items dealt to columns of equal cost, cut where a column ends.
struct Deal {
    int64_t units = 0, columns = 0;  // of all items together; columns to deal to
    std::vector<Span> list;
    std::vector<int32_t> starts;     // the first item of each column
    int64_t dealt = 0, column_end = 0;

    // `length` blocks, of which kFewUnit make a unit
    void add(int64_t seq, int64_t rows, int64_t length)
    {
        const int64_t count = (length + kFewUnit - 1) / kFewUnit;
        for (int64_t at = 0; at < count;) {
            if (dealt == column_end) {
                starts.push_back((int32_t)list.size());
                column_end = units * (int64_t)starts.size() / columns;
                continue;
            }
            const int64_t here = std::min(count - at, column_end - dealt);
            list.push_back({{(int32_t)seq, 0, (int32_t)rows, (int32_t)(at * kFewUnit), (int32_t)std::min((at + here) * kFewUnit, length), -1}, here});
            at += here, dealt += here;
        }
    }

    // The first item of every column, then the others.
    void close()
    {
        std::vector<Span> firsts, others;
        for (size_t c = 0; c < starts.size(); c++) {
            const size_t from = starts[c], to = c + 1 < starts.size() ? starts[c + 1] : list.size();
            firsts.push_back(list[from]);
            firsts.back().items = (int32_t)(to - from);
            firsts.back().next = (int32_t)(starts.size() + others.size());
            others.insert(others.end(), list.begin() + from + 1, list.begin() + to);
        }
        list = std::move(firsts);
        list.insert(list.end(), others.begin(), others.end());
    }
};

// Tiles that a block of paged_tile takes at most, from the lengths of the 128-row problems of one kv head.  Spans such that all
// blocks are resident in one round (two, three, four), or problems left whole and dealt as blocks end; whichever is estimated to
// end first, in units of a tile's time in a block that shares its CU with another (1.8 us; alone 1.35).  What is cut costs the
// spans' sums, written and read again.  (Without that, and with one speed, two chunks of 1000 tokens over 16000 and 10667, 32 heads over 8:
// 256 spans and 546 us instead of 64 and 500.)
constexpr double kTileAlone = 0.75, kJoinTiles = 1.5, kSpanTiles = 0.006;

int64_t tile_span(std::vector<int64_t> lengths, int64_t kv_heads)
{
    std::sort(lengths.begin(), lengths.end(), std::greater<int64_t>());
    int64_t total = 0;
    const int64_t longest = lengths[0], cus = kTileResident / 2;
    for (int64_t n : lengths) total += n;
    const auto blocks = [&](int64_t span) {
        int64_t n = 0;
        for (int64_t l : lengths) n += (l + span - 1) / span;
        return n * kv_heads;
    };
    const auto joins = [&](int64_t span) {
        int64_t n = 0;
        for (int64_t l : lengths) n += l > span ? (l + span - 1) / span : 0;
        return n ? kJoinTiles + kSpanTiles * (double)(n * kv_heads) : 0.0;
    };
    const int64_t whole = blocks(longest);
    int64_t best = longest;
    double least = (double)total * kv_heads / kTileResident + longest / 2.0 + kTileStart * (double)((whole + kTileResident - 1) / kTileResident);
    if (whole <= kTileResident) {  // (the longest with the longest of those that are dealt in the second turn, then alone)
        const int64_t beside = whole > cus ? lengths[cus / kv_heads] : 0;
        least = longest * kTileAlone + beside * (1.0 - kTileAlone) + kTileStart;
    }
    for (int64_t rounds = 1; rounds <= 4; rounds++) {
        int64_t low = 1, high = longest;  // the shortest spans whose blocks fit
        while (low < high) {
            const int64_t mid = (low + high) / 2;
            if (blocks(mid) <= rounds * kTileResident) high = mid;
            else low = mid + 1;
        }
        if (blocks(low) > rounds * kTileResident) continue;
        const double time = (double)rounds * (low + kTileStart) + joins(low);
        if (time < least) least = time, best = low;
    }
    return best;
}

int batch_check(const kvmix_paged_batch_t *b)
{
    if (!b) return KVMIX_ERR_NULL;
    if (b->sequences < 0 || b->heads <= 0 || b->kv_heads <= 0 || b->table_stride < 0) return KVMIX_ERR_SHAPE;
    if (b->heads % b->kv_heads != 0) return KVMIX_ERR_HEADS;
    if ((b->head_dim != 64 && b->head_dim != 128) || !page_size_ok(b->page_size) || b->kv_heads > kMostHeads || b->heads > (1 << 20) ||
        b->sequences > (1 << 20) || (__int128)b->sequences * b->table_stride > (1 << 28))
        return KVMIX_ERR_UNSUPPORTED;
    if (b->sequences && (!b->kv_lens || !b->packed_lens || !b->q_lens || (!b->table && b->table_stride))) return KVMIX_ERR_NULL;
    return KVMIX_OK;
}

int make_plan(const kvmix_paged_batch_t *b, int32_t *words, int64_t capacity, kvmix_paged_plan_t *plan)
{
    const int64_t G = b->heads / b->kv_heads, P = b->page_size, kMostTokens = int64_t(1) << 30;
    *plan = kvmix_paged_plan_t{};
    plan->heads = b->heads, plan->kv_heads = b->kv_heads, plan->head_dim = b->head_dim, plan->page_size = P;
    plan->table_stride = b->table_stride;
    Deal few;
    std::vector<int64_t> lengths;  // of the problems of 128 rows, in tiles
    plan->few_rows = 16;
    for (int64_t s = 0; s < b->sequences; s++) {
        const int64_t kv = b->kv_lens[s], pk = b->packed_lens[s], n = b->q_lens[s];
        if (n < 0 || n > kv || pk < 0 || pk % P != 0 || pk > kv - n || (kv + P - 1) / P > b->table_stride) return KVMIX_ERR_LENGTHS;
        if (kv > kMostTokens || n * G > kMostTokens || plan->tokens + n > kMostTokens) return KVMIX_ERR_UNSUPPORTED;
        const int32_t *row = b->table + s * b->table_stride;
        for (int64_t i = 0; i * P < kv; i++) {
            if (row[i] < 0) return KVMIX_ERR_PAGE;
            int64_t &most = i * P < pk ? plan->packed_pages : plan->row_pages;
            most = std::max<int64_t>(most, row[i] + int64_t(1));
        }
        plan->tokens += n;
        if (n * G <= kFewMost) {
            few.units += n ? (kv + kFewUnit * kBlock - 1) / (kFewUnit * kBlock) : 0;
            if (n * G > 16) plan->few_rows = kFewMost;
            plan->few_tokens = std::max(plan->few_tokens, n);
        } else {
            for (int64_t r = 0; r < n * G; r += kTileRows)
                lengths.push_back((kv - n + std::min(n * G - 1, r + kTileRows - 1) / G) / kTileKeys + 1);
        }
    }
    if ((__int128)plan->row_pages * P > kMost32) return KVMIX_ERR_UNSUPPORTED;
    // One round of blocks: as many columns as the chip holds blocks, each of the same number of units, whatever sequences they
    // are of.  (Spans of sequences as the items, the longest first, left a second round of a few: of 1048 blocks of which 1024
    // fit 85 us instead of 77.)
    few.columns = std::min(std::max<int64_t>(few_resident(plan->few_rows) / b->kv_heads, 1), (few.units + kFewLeast - 1) / kFewLeast);
    const int64_t span = lengths.empty() ? 1 : tile_span(lengths, b->kv_heads);

    std::vector<Span> tiles, joins;
    int64_t part = 0;
    // the spans list[first ..) of one problem
    auto joined = [&](std::vector<Span> &list, size_t first) {
        const int64_t spans = (int64_t)(list.size() - first);
        if (spans < 2) return;
        const Span &one = list[first];
        const int64_t at_once = spans > kJoinAhead ? 1 : 1024 / b->head_dim;  // rows of a block of paged_join
        plan->join_blocks = std::max<int64_t>(plan->join_blocks, (one.word[2] + at_once - 1) / at_once);
        joins.push_back({{one.word[0], one.word[1], one.word[2], (int32_t)spans, one.word[2], (int32_t)part}, 0});
        for (int64_t i = 0; i < spans; i++, part += one.word[2]) list[first + i].word[5] = (int32_t)part;
    };
    size_t problem = 0;
    for (int64_t s = 0; s < b->sequences; s++) {
        const int64_t kv = b->kv_lens[s], n = b->q_lens[s], rows = n * G;
        if (n == 0) continue;
        if (rows <= kFewMost) {
            const size_t first = few.list.size();
            few.add(s, rows, (kv + kBlock - 1) / kBlock);
            joined(few.list, first);
        } else {
            for (int64_t r = 0; r < rows; r += kTileRows) {
                const int64_t length = lengths[problem++], spans = (length + span - 1) / span, even = (length + spans - 1) / spans;
                const size_t first = tiles.size();
                for (int64_t from = 0; from < length; from += even) {
                    const int64_t to = std::min(from + even, length);
                    tiles.push_back({{(int32_t)s, (int32_t)r, (int32_t)std::min<int64_t>(kTileRows, rows - r), (int32_t)from, (int32_t)to, -1}, to - from});
                }
                joined(tiles, first);
            }
        }
        if (part > kMostTokens) return KVMIX_ERR_UNSUPPORTED;
    }
    few.close();
    // (what ends a launch is short then)
    std::stable_sort(tiles.begin(), tiles.end(), [](const Span &x, const Span &y) { return x.cost > y.cost; });
    if (few.list.size() > (size_t)kMost32 || std::max({few.starts.size(), tiles.size(), joins.size()}) * (__int128)b->kv_heads > kMostBlocks) return KVMIX_ERR_UNSUPPORTED;
    plan->few = (int64_t)few.list.size(), plan->tiles = (int64_t)tiles.size(), plan->joins = (int64_t)joins.size(), plan->part_rows = part;
    plan->few_columns = (int64_t)few.starts.size();
    int64_t at = 0;
    auto take = [&](int64_t n) {
        const int64_t was = at;
        at += up(n, 4);
        return was;
    };
    plan->slots_at = take(plan->tokens);
    for (int64_t s = 0; s < b->sequences; s++) {
        const int64_t kv = b->kv_lens[s], n = b->q_lens[s];
        plan->stores += n ? (kv - 1) / kBlock - (kv - n) / kBlock + 1 : 0;
    }
    if ((__int128)plan->stores * b->kv_heads > 4 * kMostBlocks) return KVMIX_ERR_UNSUPPORTED;
    plan->store_at = take(plan->stores * kStoreWords);
    plan->table_at = take(b->sequences * b->table_stride);
    plan->few_at = take(plan->few * kItemWords);
    plan->tile_at = take(plan->tiles * kItemWords);
    plan->join_at = take(plan->joins * kItemWords);
    plan->words = at;
    if (at > kMost32) return KVMIX_ERR_UNSUPPORTED;
    if (!words) return KVMIX_OK;
    if (capacity < at) return KVMIX_ERR_WORKSPACE;
    std::fill(words, words + at, 0);
    std::vector<int32_t> starts(b->sequences);
    int64_t token = 0, store = plan->store_at;
    for (int64_t s = 0; s < b->sequences; s++) {
        const int64_t kv = b->kv_lens[s], n = b->q_lens[s];
        starts[s] = (int32_t)token;
        const int32_t *pages = b->table + s * b->table_stride;
        for (int64_t t = kv - n; t < kv;) {  // block by block
            const int64_t end = std::min(kv, t / kBlock * kBlock + kBlock);
            const int32_t record[kStoreWords] = {(int32_t)token, (int32_t)(pages[t / P] * P + t % P), (int32_t)(end - t), 0};
            store = std::copy(record, record + kStoreWords, words + store) - words;
            for (; t < end; t++) words[plan->slots_at + token++] = (int32_t)(pages[t / P] * P + t % P);
        }
    }
    if (b->sequences && b->table_stride) std::copy(b->table, b->table + b->sequences * b->table_stride, words + plan->table_at);
    auto write = [&](const std::vector<Span> &list, int64_t to) {
        for (const Span &s : list) {
            const int32_t q = s.word[0];
            const int32_t of_seq[6] = {starts[q], (int32_t)b->q_lens[q], (int32_t)b->kv_lens[q], (int32_t)b->packed_lens[q], s.items, s.next};
            std::copy(s.word, s.word + 6, words + to);
            std::copy(of_seq, of_seq + 6, words + to + 6);
            to += kItemWords;
        }
    };
    write(few.list, plan->few_at), write(tiles, plan->tile_at), write(joins, plan->join_at);
    return KVMIX_OK;
}

int attention_check(const kvmix_paged_pool_t *p, const kvmix_paged_plan_t *plan, const kvmix_paged_attn_t *c)
{
    int rc = pool_check(p);
    if (rc == KVMIX_OK) rc = plan && c ? bits_check(p) : KVMIX_ERR_NULL;
    if (rc != KVMIX_OK) return rc;
    if (plan->kv_heads != p->kv_heads || plan->head_dim != p->head_dim || plan->page_size != p->page_size) return KVMIX_ERR_SHAPE;
    if (plan->row_pages > p->row_pages || plan->packed_pages > p->packed_pages) return KVMIX_ERR_PAGE;
    if (!(c->scale > 0.0f) || c->scale > 0x1p40f)  // (no logit of fp16 numbers is beyond 1e25 then)
        return KVMIX_ERR_UNSUPPORTED;
    for (int64_t s : {c->q_token_stride, c->q_head_stride, c->out_token_stride, c->out_head_stride})
        if (s % 8 != 0) return KVMIX_ERR_UNSUPPORTED;
    if (((uintptr_t)c->q | (uintptr_t)c->out) % 16 != 0 || (uintptr_t)c->list % 4 != 0) return KVMIX_ERR_UNSUPPORTED;
    return KVMIX_OK;
}

}  // namespace
}  // namespace kvmix

using namespace kvmix;

extern "C" int kvmix_paged_plan(const kvmix_paged_batch_t *batch, int32_t *words, int64_t capacity, kvmix_paged_plan_t *plan)
{
    const int rc = batch_check(batch);
    if (rc != KVMIX_OK) return rc;
    if (!plan) return KVMIX_ERR_NULL;
    try {
        return make_plan(batch, words, capacity, plan);
    } catch (...) {  // (lists that do not fit in memory; no exception leaves a C entry)
        return KVMIX_ERR_MEMORY;
    }
}

extern "C" int64_t kvmix_paged_attention_workspace_bytes(const kvmix_paged_plan_t *plan)
{
    return plan ? plan->kv_heads * plan->part_rows * (plan->head_dim * 4 + 8) : 0;
}

extern "C" int kvmix_paged_attention(const kvmix_paged_pool_t *p, const kvmix_paged_plan_t *plan, const kvmix_paged_attn_t *c, void *workspace,
                                     int64_t workspace_bytes, kvmix_stream_t stream)
{
    const int rc = attention_check(p, plan, c);
    if (rc != KVMIX_OK) return rc;
    if (plan->tokens == 0) return KVMIX_OK;
    if (!c->q || !c->out || !c->list || (plan->row_pages && !p->rows) || (plan->packed_pages && !p->packed)) return KVMIX_ERR_NULL;
    if (plan->part_rows && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < kvmix_paged_attention_workspace_bytes(plan)))
        return KVMIX_ERR_WORKSPACE;
    PagedArgs a;
    a.q = (const _Float16 *)c->q, a.out = (_Float16 *)c->out;
    a.q_ts = c->q_token_stride, a.q_hs = c->q_head_stride, a.o_ts = c->out_token_stride, a.o_hs = c->out_head_stride;
    a.rows = (const _Float16 *)p->rows, a.packed = (const uint32_t *)p->packed;
    const PlanWords list = (PlanWords)c->list;
    a.table = list + plan->table_at, a.items = nullptr;
    a.table_stride = (int)plan->table_stride, a.kv_heads = (int)plan->kv_heads, a.group = (int)(plan->heads / plan->kv_heads);
    a.blocks_log2 = __builtin_ctzll((uint64_t)plan->page_size / kBlock);
    a.scale = c->scale * kLog2e;
    a.part = (float *)workspace, a.part_rows = plan->part_rows;
    a.part_ml = (float2 *)((float *)workspace + plan->kv_heads * plan->part_rows * plan->head_dim);
    hipStream_t st = (hipStream_t)stream;
    with_dim(p->head_dim, [&](auto D) {
        with_bits(p->k_bits, [&](auto KB) {
            with_bits(p->v_bits, [&](auto VB) {
                if (plan->tiles) {
                    a.items = list + plan->tile_at;
                    paged_tile<D.value, KB.value, VB.value><<<(unsigned)(plan->tiles * plan->kv_heads), 256, 0, st>>>(a);
                }
                if (plan->few) {
                    a.items = list + plan->few_at;
                    const unsigned grid = (unsigned)(plan->few_columns * plan->kv_heads);
                    if (plan->few_rows > 16) paged_few<D.value, KB.value, VB.value, 2, true><<<grid, 256, 0, st>>>(a);
                    else if (plan->few_tokens > 1) paged_few<D.value, KB.value, VB.value, 1, true><<<grid, 256, 0, st>>>(a);
                    else paged_few<D.value, KB.value, VB.value, 1, false><<<grid, 256, 0, st>>>(a);
                }
            });
        });
        if (plan->joins) {
            a.items = list + plan->join_at;
            paged_join<D.value><<<dim3((unsigned)(plan->joins * plan->kv_heads), (unsigned)plan->join_blocks), 256, 0, st>>>(a);
        }
    });
    return launch_status();
}
