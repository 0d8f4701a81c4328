// Low-rank adapters of many requests beside a projection that they share:  y_t = base_t + s_i B_i (A_i x_t), i the adapter of token t.
//
// Bound by memory: the weights of the adapters in use and the activations are read once, two operations for a value of them and rank.
// Two launches, because every value of y wants all of x (and one where that is little):
//   shrink   u = A x.  A tile is up to 64 tokens of one adapter (kvmix_adapter_plan deals them out, whichever sequences they are of), a
//            block a tile and a stretch of k.  Ranks are the rows of v_mfma_f32_16x16x32, tokens its columns, so that a lane has eight k
//            of one row of A and of one token, sixteen bytes.  The four waves read 256 bytes of each row at once, exchange them in
//            the LDS and multiply a quarter of these each.  (Few tokens and ranks: each wave its own quarter, without the LDS.)  The
//            waves' sums come together in the LDS, those of the stretches (there are several where there are few tiles) in
//   expand   y = base + s B u.  A block sums u of its tile and keeps it in the LDS, then takes 128 columns of y at a time, a quarter of them
//            to a wave.  u is kept as the sum of two numbers of 16 bits: next to a token's largest it is exact to 2^-22 (bf16: 2^-16), where it
//            rounds to fp16 alone it would be off by 2^-11 before the sum over the ranks.  In fp16 it is kept times a power of two that
//            brings the token's largest just below 2^14.  bf16 has all of fp32's exponents: what is below 2^-8 is brought up to there, so that
//            second parts keep their digits and 128 products with the largest of B stay below 2^128, and what is beyond 2^126, which could
//            round to an infinity, down to there.  Rows of B are dealt to two matrix products so that a lane ends with eight columns of
//            one token that follow one another; through the LDS they come to where 256 bytes of a row of base are.
// Reads of rows in runs of 256 bytes by a wave are what counts: as the matrix products take them, 64 bytes of each of sixteen rows, the
// same bytes take 26 us instead of 19 (x) and 38 instead of 28 (base and y).  Both kernels read a step ahead of the one that is multiplied,
// and expand's first reads go out before it sums u.
// One token with an adapter of rank 8, k = n = 4096: 6.0 us, one launch and the reads of A by each of its 32 blocks.
// 8168 tokens of 6 adapters of rank 64, k = n = 4096, bf16: 44.6 us, 4.5 TB/s (a copy of as many bytes: 40); 1567 tokens of rank 32 from
// k = 11008 to n = 4096: 20 us; 64 tokens of 8 adapters of rank 16 to n = 12288: 8.6 us, that is two launches; of 40 adapters 11.4, of 64 11.9.
// Sums in fp32; y is rounded once.
#include <algorithm>
#include <new>
#include <type_traits>
#include <vector>

#include "kvmix_common.h"

namespace kvmix {

typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef const __attribute__((address_space(4))) int32_t *PlanWords;

constexpr int kTile = 64, kSub = 16;       // tokens of a tile, of a column of a matrix product
constexpr int kTileWords = 4;              // adapter or -1, first of the list, how many, the first token where they follow one another, else -1
constexpr int kWaves = 4, kStep = 32 * kWaves;  // (values of a row in a step of a block)
constexpr int64_t kMostRank = 128;

template <typename T>
struct Vec8 {
    typedef T type __attribute__((ext_vector_type(8)));
};

__device__ __forceinline__ floatx4 product(Vec8<_Float16>::type a, Vec8<_Float16>::type b, floatx4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(a, b, c, 0, 0, 0);
}

__device__ __forceinline__ floatx4 product(Vec8<__bf16>::type a, Vec8<__bf16>::type b, floatx4 c)
{
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
}

struct AdapterArgs {
    const void *x, *a, *b, *base;
    void *out;
    int64_t x_ts, a_as, a_rs, b_as, b_ns, base_ts, out_ts;
    const float *scales;    // may be NULL: 1
    float *part;            // [splits][adapted tokens][padded rank]
    PlanWords tiles, rows;  // tiles; their tokens
    int64_t part_rows;
    int rank, padded, k, n, splits, rank_chunks, n_blocks, units;  // units: of 32 columns, of a wave of expand
};

// Every `step`th token of a tile from `from` on (where there is none, the last).
template <int ST>
__device__ __forceinline__ void rows_of(int (&row)[ST], const AdapterArgs &p, PlanWords tile, int from, int step)
{
    const int last = tile[2] - 1;
    if (tile[3] >= 0) {
#pragma unroll
        for (int s = 0; s < ST; s++) row[s] = tile[3] + min(step * s + from, last);
    } else {
#pragma unroll
        for (int s = 0; s < ST; s++) row[s] = p.rows[tile[1] + min(step * s + from, last)];
    }
}

// Waves meet; what each has written to the LDS is seen by all.  Reads of memory stay under way.
__device__ __forceinline__ void meet()
{
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

// ---------------------------------------------------------------------------------------------------------------------

// Steps 0 .. count - 1, each read into one of two places while the one before is used; `first` comes after the first reads.  (Three or
// four places gained nothing.)
template <typename L, typename U, typename F>
__device__ __forceinline__ void in_turn(int count, L load, U use, F first)
{
    if (count > 0) load(0, 0);
    first();
    int i = 0;
    for (; i + 3 <= count; i += 2) load(1, i + 1), use(0, i), load(0, i + 2), use(1, i + 1);
    if (i + 1 < count) load(1, i + 1);
    if (i < count) use(0, i);
    if (i + 1 < count) use(1, i + 1);
}

// Ranks [first, first + 16 RT) of a tile of up to sixteen tokens, over a quarter of the 32-wide units [begin, to) of k: every fourth UN of them,
// which are read at once.
template <int UN, typename T, int RT>
__device__ __forceinline__ void shrink_few(const T *const (&a)[RT], const T *x, int begin, int to, int k, int wave, int g, floatx4 (&acc)[RT][1])
{
    typedef typename Vec8<T>::type V;
    struct Units {
        V a[UN][RT], x[UN];
    } v[2];
    const int groups = max(0, (min(to, k / 32) - begin) / UN);
    auto load = [&](Units &v, int i) {
        const int at = 32 * (begin + UN * (wave + kWaves * i)) + 8 * g;
#pragma unroll
        for (int j = 0; j < UN; j++) {
            v.x[j] = *(const V *)(x + at + 32 * j);
#pragma unroll
            for (int r = 0; r < RT; r++) v.a[j][r] = *(const V *)(a[r] + at + 32 * j);
        }
    };
    auto multiply = [&](const Units &v) {
#pragma unroll
        for (int j = 0; j < UN; j++)
#pragma unroll
            for (int r = 0; r < RT; r++) acc[r][0] = product(v.a[j][r], v.x[j], acc[r][0]);
    };
    in_turn((groups - wave + kWaves - 1) / kWaves, [&](int d, int i) { load(v[d], i); }, [&](int d, int) { multiply(v[d]); }, [] {});
    for (int u = begin + UN * groups + wave; u < to; u += kWaves) {
        const bool in = 32 * u + 8 * g < k;  // (k in whole eights)
        const V xv = in ? *(const V *)(x + 32 * u + 8 * g) : V{};
#pragma unroll
        for (int r = 0; r < RT; r++) acc[r][0] = product(in ? *(const V *)(a[r] + 32 * u + 8 * g) : V{}, xv, acc[r][0]);
    }
}

// The same of more tokens, over whole steps of kStep of k through the LDS: a wave reads a quarter of the rows of A and x, 256 bytes of each at once, and
// multiplies one of a step's four units.  A row's pieces of sixteen bytes are exchanged by its number, so that no lanes meet in a bank.
template <bool STREAM, typename T, int RT, int ST>
__device__ __forceinline__ void shrink_staged(const T *const (&a)[RT], const T *const (&x)[ST], void *lds, int begin, int to, int k, int wave, int m,
                                              int g, floatx4 (&acc)[RT][ST])
{
    typedef typename Vec8<T>::type V;
    typedef V Rows[16];
    Rows *buffer = (Rows *)lds;  // two steps: rows of A, then of x
    struct Step {
        V a[RT], x[ST];
    } v[2];
    auto load = [&](Step &v, int i) {
        const int at = begin + kStep * i + 8 * m;
#pragma unroll
        for (int r = 0; r < RT; r++) v.a[r] = *(const V *)(a[r] + min(at, k - 8));
#pragma unroll
        for (int s = 0; s < ST; s++) {
            const V *from = (const V *)(x[s] + min(at, k - 8));
            v.x[s] = STREAM ? __builtin_nontemporal_load(from) : *from;
        }
        if (begin + kStep * i + kStep > k && at >= k) {  // (k in whole eights)
#pragma unroll
            for (int r = 0; r < RT; r++) v.a[r] = V{};
#pragma unroll
            for (int s = 0; s < ST; s++) v.x[s] = V{};
        }
    };
    auto multiply = [&](const Step &v, int i) {
        Rows *rows_a = buffer + i % 2 * 16 * (RT + ST), *rows_x = rows_a + 16 * RT;
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const int row = wave * 4 * RT + g + 4 * r;
            rows_a[row][m ^ row % 16] = v.a[r];
        }
#pragma unroll
        for (int s = 0; s < ST; s++) {
            const int row = wave * 4 * ST + g + 4 * s;
            rows_x[row][m ^ row % 16] = v.x[s];
        }
        meet();  // (who is here has multiplied what lay in the other half)
        V xv[ST];
#pragma unroll
        for (int s = 0; s < ST; s++) xv[s] = rows_x[16 * s + m][4 * wave + g ^ m];
#pragma unroll
        for (int r = 0; r < RT; r++) {
            const V av = rows_a[16 * r + m][4 * wave + g ^ m];
#pragma unroll
            for (int s = 0; s < ST; s++) acc[r][s] = product(av, xv[s], acc[r][s]);
        }
    };
    in_turn((to - begin + kStep - 1) / kStep, [&](int d, int i) { load(v[d], i); }, [&](int d, int i) { multiply(v[d], i); }, [] {});
    meet();  // (the LDS is wanted for the sums)
}

// Not of sixteen tokens of a rank of 32 at most, which wait for the LDS longer than for their rows (40 tiles of rank 8, k 11008: 8.5 instead of
// 10.9 us with the other kernel; one of rank 64, k 4096: 7.2 and 6.6).
constexpr bool through_lds(int RT, int ST) { return RT > 2 || ST > 1; }

// STREAM: x is more than the caches of the dies keep.
template <typename T, int RT, bool STREAM>
__global__ void __launch_bounds__(256) adapter_shrink(AdapterArgs p)
{
    constexpr int LD = RT * 16, Q = RT * 4;
    // [waves][tokens][ranks]; the fours of ranks of token t in an order of its own, so that lanes meet in no bank
    extern __shared__ __attribute__((aligned(16))) float sums[];
    auto place = [](int row, int t, int four) { return row * LD + 4 * (four ^ t % Q); };
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), m = lane % 16, g = lane / 16;
    const int split = blockIdx.x % p.splits, nth = blockIdx.x / p.splits, chunk = nth % p.rank_chunks;
    const PlanWords tile = p.tiles + nth / p.rank_chunks * kTileWords;
    const int adapter = tile[0], first = tile[1], count = tile[2], subs = (count + kSub - 1) / kSub;
    const int steps = (p.k + kStep - 1) / kStep;
    const int begin = steps * split / p.splits * kStep, to = steps * (split + 1) / p.splits * kStep;  // (2^17 steps, 16 stretches at most)
    auto run = [&](auto st) {
        constexpr int ST = decltype(st)::value;
        const T *a[RT], *x[ST];
        int row[ST];
        floatx4 acc[RT][ST] = {};
        constexpr bool staged = through_lds(RT, ST);
        rows_of(row, p, tile, staged ? wave * 4 * ST + g : m, staged ? 4 : kSub);
#pragma unroll
        for (int s = 0; s < ST; s++) x[s] = (const T *)p.x + row[s] * p.x_ts;
#pragma unroll
        for (int r = 0; r < RT; r++)  // (what lies beyond the rank is not kept)
            a[r] = (const T *)p.a + adapter * p.a_as + min(chunk * RT * 16 + (staged ? wave * 4 * RT + g + 4 * r : 16 * r + m), p.rank - 1) * p.a_rs;
        if constexpr (staged) shrink_staged<STREAM>(a, x, sums, begin, to, p.k, wave, m, g, acc);
        else shrink_few<4>(a, x[0], begin / 32, min(to, p.k + 31) / 32, p.k, wave, g, acc);
#pragma unroll
        for (int s = 0; s < ST; s++)
            if (s < subs)
#pragma unroll
                for (int r = 0; r < RT; r++) *(floatx4 *)(sums + place((wave * subs + s) * kSub + m, m, 4 * r + g)) = acc[r][s];
    };
    if (subs == 1) run(std::integral_constant<int, 1>());
    else if (subs == 2) run(std::integral_constant<int, 2>());
    else run(std::integral_constant<int, 4>());
    __syncthreads();
    for (int i = threadIdx.x; i < count * Q; i += 256) {
        const int t = i / Q, c = i % Q, rank = (chunk * Q + c) * 4;
        floatx4 s = *(const floatx4 *)(sums + place(t, t % kSub, c));
#pragma unroll
        for (int w = 1; w < kWaves; w++) s += *(const floatx4 *)(sums + place(w * subs * kSub + t, t % kSub, c));
        if (rank < p.padded) *(floatx4 *)(p.part + (split * p.part_rows + first + t) * p.padded + rank) = s;
    }
}

// ---------------------------------------------------------------------------------------------------------------------

// RX: the rank, rounded up to 16, 32, 64 or 128.  TOKENS: of a tile at most, 16 or 64 (what the LDS holds says how many blocks a CU takes: 40
// adapters of rank 64 to n = 22016, one token each, 34 instead of 38 us).  WHOLE: every block makes all of u itself, of tiles of up to
// sixteen tokens, and there is no other launch.  STREAM: base and y are more than the caches of the dies keep, and are read and written as
// what nobody wants again soon.
template <typename T, int RX, int TOKENS, bool WHOLE, bool STREAM>
__global__ void __launch_bounds__(256) adapter_expand(AdapterArgs p)
{
    typedef typename Vec8<T>::type V;
    constexpr int NF = RX >= 32 ? RX / 32 : 1, LD = 2 * RX + 8, L = RX / 4;  // pieces of a row of B; of u: its two parts; lanes to a token
    constexpr int COLUMNS = 32 * kWaves;                                     // of y, in a step of the block
    __shared__ alignas(16) T u[TOKENS][LD];
    __shared__ float power[TOKENS];
    __shared__ alignas(16) float sums[WHOLE ? kWaves * kSub : TOKENS][COLUMNS + 4];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave), m = lane % 16, g = lane / 16;
    const PlanWords tile = p.tiles + blockIdx.x / p.n_blocks * kTileWords;
    const int adapter = tile[0], first = tile[1], count = tile[2], subs = (count + kSub - 1) / kSub;
    const int begin = blockIdx.x % p.n_blocks * p.units * COLUMNS, steps = (min(p.n - begin, p.units * COLUMNS) + COLUMNS - 1) / COLUMNS;
    if (adapter < 0) {  // (tokens without one: to be copied)
        constexpr int ST = kTile / kSub;
        int row[ST];
        rows_of(row, p, tile, wave * 4 * ST + g, 4);
        for (int i = 0; i < steps; i++) {
            const int column = begin + COLUMNS * i + 8 * m;
            if (column >= p.n) break;
            V y[ST];
#pragma unroll
            for (int s = 0; s < ST; s++) y[s] = *(const V *)((const T *)p.base + row[s] * p.base_ts + column);
#pragma unroll
            for (int s = 0; s < ST; s++)
                if (wave * 4 * ST + g + 4 * s < count) *(V *)((T *)p.out + row[s] * p.out_ts + column) = y[s];
        }
        return;
    }
    auto sum = [&](auto st) {
        constexpr int P = (decltype(st)::value * kSub * L + 255) / 256, AHEAD = P >= 4 ? 2 : P == 2 ? 4 : 8;  // turns of the block
        const int c = threadIdx.x % L, t0 = threadIdx.x / L;
        floatx4 s[P] = {};
        if constexpr (WHOLE) {
            constexpr int RT = RX / 16;
            const T *a[RT];
            int row[1];
            rows_of(row, p, tile, m, kSub);
#pragma unroll
            for (int r = 0; r < RT; r++) a[r] = (const T *)p.a + adapter * p.a_as + min(16 * r + m, p.rank - 1) * p.a_rs;
            floatx4 acc[RT][1] = {};
            shrink_few<RT <= 2 ? 4 : 2>(a, (const T *)p.x + row[0] * p.x_ts, 0, (p.k + 31) / 32, p.k, wave, g, acc);
#pragma unroll
            for (int r = 0; r < RT; r++) *(floatx4 *)&sums[wave * kSub + m][16 * r + 4 * g] = acc[r][0];
            meet();
#pragma unroll
            for (int w = 0; w < kWaves; w++) s[0] += *(const floatx4 *)&sums[w * kSub + t0 % kSub][4 * c];
        } else {
            const float *at[P];
#pragma unroll
            for (int j = 0; j < P; j++) at[j] = p.part + (int64_t)(first + min(t0 + 256 / L * j, count - 1)) * p.padded + (4 * c < p.rank ? 4 * c : 0);
            for (int i = 0; i < p.splits; i += AHEAD) {  // (AHEAD stretches' reads under way; of none: the last one's again, not added)
                floatx4 q[AHEAD][P];
#pragma unroll
                for (int h = 0; h < AHEAD; h++)
#pragma unroll
                    for (int j = 0; j < P; j++) q[h][j] = *(const floatx4 *)(at[j] + min(i + h, p.splits - 1) * p.part_rows * p.padded);
                __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                for (int h = 0; h < AHEAD; h++)
#pragma unroll
                    for (int j = 0; j < P; j++) s[j] += i + h < p.splits ? q[h][j] : floatx4{0.0f, 0.0f, 0.0f, 0.0f};
            }
        }
#pragma unroll
        for (int j = 0; j < P; j++)
            if (t0 + 256 / L * j >= count || 4 * c >= p.rank) s[j] = floatx4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < P; j++) {
            const int t = t0 + 256 / L * j;
            float most = 0.0f;
#pragma unroll
            for (int r = 0; r < 4; r++) most = fmaxf(most, fabsf(s[j][r]) < __builtin_inff() ? fabsf(s[j][r]) : 0.0f);
#pragma unroll
            for (int o = L / 2; o; o /= 2) most = fmaxf(most, __shfl_xor(most, o));
            // (the power of numbers below 2^-100 is that of 2^-100; infinities go through as they are, and their second part is nothing)
            const int top = most > 0.0f ? max(__builtin_amdgcn_frexp_expf(most), -100) : 0;
            const int e = std::is_same<T, _Float16>::value ? top - 14 : max(min(top + 8, 0), top - 126);
            typedef T four __attribute__((ext_vector_type(4)));
            four high, low;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float v = ldexpf(s[j][r], -e);
                const T h = (T)v;
                high[r] = h, low[r] = fabsf(v) < __builtin_inff() ? (T)(v - (float)h) : (T)0.0f;
            }
            if (t < kSub * decltype(st)::value) {
                *(four *)&u[t][4 * c] = high;
                *(four *)&u[t][RX + 4 * c] = low;
                if (c == 0) power[t] = ldexpf(1.0f, e);
            }
        }
        meet();
    };
    const float scale = p.scales ? p.scales[adapter] : 1.0f;
    auto run = [&](auto st) {
        constexpr int ST = decltype(st)::value;
        struct Unit {
            V w[2][NF], y[ST];  // rows of B, values of base
        } v[2];
        const T *from[ST];
        T *to[ST];
        int row[ST];
        const int t0 = wave * 4 * ST + g;  // a wave reads and writes every fourth of 4 ST tokens, 256 bytes of each at once
        rows_of(row, p, tile, t0, 4);
#pragma unroll
        for (int s = 0; s < ST; s++) from[s] = (const T *)p.base + row[s] * p.base_ts, to[s] = (T *)p.out + row[s] * p.out_ts;
        auto load = [&](Unit &v, int i) {
            const int column = begin + COLUMNS * i;
#pragma unroll
            for (int h = 0; h < 2; h++)
#pragma unroll
                for (int f = 0; f < NF; f++) {  // (what lies beyond is not kept; of u beyond the rank: nothing)
                    const int row = min(column + 32 * wave + 8 * (m / 4) + 4 * h + m % 4, p.n - 1), r = (32 * f + 8 * g) % RX;
                    v.w[h][f] = *(const V *)((const T *)p.b + adapter * p.b_as + row * p.b_ns + (r < p.rank ? r : 0));
                }
#pragma unroll
            for (int s = 0; s < ST; s++) {
                const V *at = (const V *)(from[s] + min(column + 8 * m, p.n - 8));
                v.y[s] = STREAM ? __builtin_nontemporal_load(at) : *at;
            }
        };
        auto store = [&](Unit &v, int i) {
#pragma unroll
            for (int s = 0; s < ST; s++) {
                const int t = kSub * s + m;
                floatx4 acc[2] = {};
#pragma unroll
                for (int f = 0; f < RX / 16; f++) {
                    const V x = *(const V *)&u[t][32 * f + 8 * g];
                    acc[0] = product(v.w[0][f % NF], x, acc[0]);
                    acc[1] = product(v.w[1][f % NF], x, acc[1]);
                }
                const float two = power[t];
#pragma unroll
                for (int h = 0; h < 2; h++) *(floatx4 *)&sums[t][32 * wave + 8 * g + 4 * h] = acc[h] * two;
            }
            meet();
            const int column = begin + COLUMNS * i + 8 * m;
#pragma unroll
            for (int s = 0; s < ST; s++) {
                const int t = t0 + 4 * s;
                V y = v.y[s];
#pragma unroll
                for (int h = 0; h < 2; h++) {
                    const floatx4 d = *(const floatx4 *)&sums[t][8 * m + 4 * h];
#pragma unroll
                    for (int c = 0; c < 4; c++) y[4 * h + c] = (T)fmaf(d[c], scale, (float)y[4 * h + c]);
                }
                if (t >= count || column >= p.n) continue;
                if constexpr (STREAM) __builtin_nontemporal_store(y, (V *)(to[s] + column));
                else *(V *)(to[s] + column) = y;
            }
            meet();
        };
        in_turn(steps, [&](int d, int i) { load(v[d], i); }, [&](int d, int i) { store(v[d], i); }, [&] { sum(st); });
    };
    if (TOKENS == kSub || subs == 1) run(std::integral_constant<int, 1>());
    else if constexpr (TOKENS > kSub) {
        if (subs == 2) run(std::integral_constant<int, 2>());
        else run(std::integral_constant<int, 4>());
    }
}

// ---------------------------------------------------------------------------------------------------------------------

namespace {

constexpr int64_t kMostTokens = int64_t(1) << 30;
constexpr int64_t kMostBlocks = (1 << 24) - 1;  // of 256 threads: a launch of 2^32 threads or more runs modulo 2^32, without an error

int make_adapter_plan(const int64_t *adapters, const int64_t *counts, int64_t sequences, int64_t n_adapters, int32_t *words, int64_t capacity,
                      kvmix_adapter_plan_t *plan)
{
    *plan = kvmix_adapter_plan_t{};
    std::vector<int64_t> of(n_adapters + 1);  // tokens of each adapter, of none last
    for (int64_t s = 0; s < sequences; s++) {
        if (counts[s] < 0) return KVMIX_ERR_SHAPE;
        if (adapters[s] >= n_adapters) return KVMIX_ERR_ADAPTER;
        if (counts[s] > kMostTokens - plan->tokens) return KVMIX_ERR_UNSUPPORTED;
        plan->tokens += counts[s];
        of[adapters[s] < 0 ? n_adapters : adapters[s]] += counts[s];
        if (counts[s]) plan->adapters = std::max(plan->adapters, adapters[s] + 1);
    }
    for (int64_t i = 0; i <= n_adapters; i++) {
        (i < n_adapters ? plan->tiles : plan->bare) += (of[i] + kTile - 1) / kTile;
        if (i < n_adapters) plan->rows += of[i], plan->most = std::max(plan->most, std::min<int64_t>(of[i], kTile));
    }
    plan->rows_at = (plan->tiles + plan->bare) * kTileWords;
    plan->words = plan->rows_at + plan->tokens;
    if (!words) return KVMIX_OK;
    if (capacity < plan->words) return KVMIX_ERR_WORKSPACE;
    std::vector<int64_t> next(n_adapters + 1);  // where each adapter's tokens go
    int32_t *tile = words;
    int64_t first = 0;
    for (int64_t i = 0; i <= n_adapters; i++) {
        next[i] = plan->rows_at + first;
        const int64_t tiles = (of[i] + kTile - 1) / kTile, even = tiles ? ((of[i] + tiles - 1) / tiles + kSub - 1) / kSub * kSub : 0;
        for (int64_t t = 0; t < tiles; t++, tile += kTileWords) {
            tile[0] = i < n_adapters ? (int32_t)i : -1, tile[1] = (int32_t)(first + t * even);
            tile[2] = (int32_t)std::min(even, of[i] - t * even);
        }
        first += of[i];
    }
    int32_t token = 0;
    for (int64_t s = 0; s < sequences; s++)
        for (int64_t t = 0; t < counts[s]; t++) words[next[adapters[s] < 0 ? n_adapters : adapters[s]]++] = token++;
    for (tile = words; tile < words + plan->rows_at; tile += kTileWords) {
        const int32_t *rows = words + plan->rows_at + tile[1];
        tile[3] = rows[tile[2] - 1] - rows[0] == tile[2] - 1 ? rows[0] : -1;  // (they ascend)
    }
    return KVMIX_OK;
}

int64_t padded_rank(int64_t rank) { return (rank + 15) / 16 * 16; }

int64_t rank_chunks(int64_t rank) { return (rank + 63) / 64; }

// Pieces of the columns of y, and how many steps each has.
struct ExpandPlan {
    int64_t tiles, units, blocks;
};

ExpandPlan expand_plan(const kvmix_adapter_plan_t *plan, const kvmix_adapters_t *c)
{
    const int64_t tiles = plan->tiles + (c->out == c->base ? 0 : plan->bare), columns = (c->n + 31) / 32;
    const int64_t units = std::max<int64_t>(1, std::min<int64_t>(8, tiles * columns / (kWaves * 384)));
    return {tiles, units, (columns + kWaves * units - 1) / (kWaves * units)};
}

// One launch instead of two: where the tiles are of few tokens, a block finds a CU of its own and has at most 64 KB of A to read (4096 of
// rank 8): up to there a call gains more than a graph's node loses.  One token, n = 4096, called one after the other and in a graph: k 2048,
// rank 16 5.0 instead of 7.4 us, 5.0 instead of 5.6; k 4096, rank 8 5.9 instead of 7.0, 5.8 instead of 5.5; k 4096, rank 16 7.1 instead of 7.3,
// 7.1 instead of 5.7 (eight tokens 7.7 instead of 7.4).  Twice as many blocks as CUs: 9 instead of 5.8 in a graph.
bool whole_u(const kvmix_adapter_plan_t *plan, const kvmix_adapters_t *c)
{
    const int64_t blocks = (plan->tiles + plan->bare) * ((c->n + 32 * kWaves - 1) / (32 * kWaves));
    return plan->tiles && plan->most <= kSub && c->rank <= 64 && c->k * c->rank <= 32768 && blocks <= 256;
}

// y of more than the eight dies' caches hold (32 MB) goes by them.  8168 tokens at rank 64 (k = n = 4096): 44.5 instead of 53 us among calls with
// other inputs, 55.7 instead of 53.8 between a kernel that writes base and one that reads y; n = 12288: 95 instead of 101 there.  12 MB
// of y: 20.6 instead of 19.9.
bool streams(const kvmix_adapter_plan_t *plan, const kvmix_adapters_t *c) { return plan->tokens > ((1 << 25) / 2) / c->n; }

// x of more than twice that: 4096 tokens of k = 11008 (90 MB) 46 instead of 49.7 us between a kernel that writes base and one that reads y, 16384 of
// 4096 (134 MB) 96 instead of 108; 8168 of 4096 (67 MB) 55 instead of 57, but 47.6 instead of 44.6 among calls with other inputs.
bool streams_x(const kvmix_adapter_plan_t *plan, const kvmix_adapters_t *c) { return plan->tokens > ((1 << 26) / 2) / c->k; }

// Stretches of k: a block for every CU, but no less than four steps.  Twice as many blocks read x no faster, and the sums that expand has to
// gather are twice as many: 128, 256 and 512 blocks take 24.9, 21.6 and 24.0 us for 1546 tokens of rank 32 from k = 11008, 54.0, 47.7 and
// 49.7 for 7972 of rank 64 from 4096.
constexpr int64_t kStretches = 256;

int64_t splits_of(const kvmix_adapter_plan_t *plan, int64_t rank, int64_t k)
{
    const int64_t blocks = std::max<int64_t>(plan->tiles * rank_chunks(rank), 1);
    return std::max<int64_t>(1, std::min<int64_t>({kStretches / blocks, k / 512, 16}));
}

bool whole(int64_t v) { return v % 8 == 0; }

int adapters_check(const kvmix_adapter_plan_t *plan, const kvmix_adapters_t *c)
{
    if (!plan || !c) return KVMIX_ERR_NULL;
    if (c->dtype != KVMIX_F16 && c->dtype != KVMIX_BF16) return KVMIX_ERR_DTYPE;
    if (c->adapters < 0 || c->rank <= 0 || c->k <= 0 || c->n <= 0) return KVMIX_ERR_SHAPE;
    if (plan->adapters > c->adapters) return KVMIX_ERR_ADAPTER;
    if (c->rank > kMostRank || c->k > (1 << 24) || c->n > (1 << 24) || !whole(c->rank) || !whole(c->k) || !whole(c->n) || !whole(c->x_token_stride) ||
        !whole(c->a_adapter_stride) || !whole(c->a_rank_stride) || !whole(c->b_adapter_stride) || !whole(c->b_row_stride) || !whole(c->base_token_stride) ||
        !whole(c->out_token_stride) || ((uintptr_t)c->x | (uintptr_t)c->a | (uintptr_t)c->b | (uintptr_t)c->base | (uintptr_t)c->out) % 16)
        return KVMIX_ERR_UNSUPPORTED;
    return KVMIX_OK;
}

template <typename F>
void with_rank(int64_t rank, F f)
{
    if (rank <= 16) f(std::integral_constant<int, 16>());
    else if (rank <= 32) f(std::integral_constant<int, 32>());
    else if (rank <= 64) f(std::integral_constant<int, 64>());
    else f(std::integral_constant<int, 128>());
}

}  // namespace
}  // namespace kvmix

using namespace kvmix;

extern "C" int kvmix_adapter_plan(const int64_t *adapters, const int64_t *counts, int64_t sequences, int64_t n_adapters, int32_t *words, int64_t capacity,
                                  kvmix_adapter_plan_t *plan)
{
    if (!plan || (sequences > 0 && (!adapters || !counts))) return KVMIX_ERR_NULL;
    if (sequences < 0 || n_adapters < 0) return KVMIX_ERR_SHAPE;
    if (n_adapters > (1 << 20) || sequences > kMostTokens) return KVMIX_ERR_UNSUPPORTED;
    try {
        return make_adapter_plan(adapters, counts, sequences, n_adapters, words, capacity, plan);
    } catch (const std::bad_alloc &) {
        return KVMIX_ERR_MEMORY;
    }
}

extern "C" int64_t kvmix_add_adapters_workspace_bytes(const kvmix_adapter_plan_t *plan, const kvmix_adapters_t *c)
{
    if (adapters_check(plan, c) != KVMIX_OK || whole_u(plan, c)) return 0;
    return splits_of(plan, c->rank, c->k) * plan->rows * padded_rank(c->rank) * (int64_t)sizeof(float);
}

extern "C" int kvmix_add_adapters(const kvmix_adapter_plan_t *plan, const int32_t *list, const kvmix_adapters_t *c, void *workspace, int64_t workspace_bytes,
                                  kvmix_stream_t stream)
{
    const int rc = adapters_check(plan, c);
    if (rc != KVMIX_OK) return rc;
    if (plan->tokens == 0) return KVMIX_OK;
    if (!c->x || !c->base || !c->out || !list || (plan->rows && (!c->a || !c->b))) return KVMIX_ERR_NULL;
    if (c->out == c->base && c->out_token_stride != c->base_token_stride) return KVMIX_ERR_SHAPE;
    if (plan->tokens > 1 && c->out_token_stride < c->n) return KVMIX_ERR_SHAPE;
    const int64_t need = kvmix_add_adapters_workspace_bytes(plan, c);
    if (need && (!workspace || (uintptr_t)workspace % 16 || workspace_bytes < need)) return KVMIX_ERR_WORKSPACE;
    AdapterArgs p{};
    p.x = c->x, p.a = c->a, p.b = c->b, p.base = c->base, p.out = c->out;
    p.x_ts = c->x_token_stride, p.a_as = c->a_adapter_stride, p.a_rs = c->a_rank_stride, p.b_as = c->b_adapter_stride, p.b_ns = c->b_row_stride;
    p.base_ts = c->base_token_stride, p.out_ts = c->out_token_stride, p.scales = c->scales, p.part = (float *)workspace;
    p.tiles = (PlanWords)list, p.rows = (PlanWords)list + plan->rows_at, p.part_rows = plan->rows;
    p.rank = (int)c->rank, p.padded = (int)padded_rank(c->rank), p.k = (int)c->k, p.n = (int)c->n;
    p.splits = (int)splits_of(plan, c->rank, c->k), p.rank_chunks = (int)rank_chunks(c->rank);
    const ExpandPlan e = expand_plan(plan, c);
    p.units = (int)e.units, p.n_blocks = (int)e.blocks;
    const int64_t shrink = plan->tiles * p.rank_chunks * p.splits, expand = e.tiles * e.blocks;
    if (shrink > kMostBlocks || expand > kMostBlocks) return KVMIX_ERR_UNSUPPORTED;
    hipStream_t st = (hipStream_t)stream;
    auto run = [&](auto zero) {
        using T = decltype(zero);
        with_rank(c->rank, [&](auto RX) {
            constexpr int RT = RX.value >= 64 ? 4 : RX.value / 16;
            const size_t subs = (plan->most + kSub - 1) / kSub, sums = kWaves * subs * kSub * (RT * 16) * sizeof(float);
            const int ST = subs <= 1 ? 1 : subs == 2 ? 2 : 4;
            const size_t lds = std::max(sums, through_lds(RT, ST) ? 2 * kSub * (RT + ST) * 256 : size_t(0));
            if constexpr (RX.value <= 64) {  // (a larger rank would need k of 448 at most)
                if (whole_u(plan, c)) {
                    adapter_expand<T, RX.value, kSub, true, false><<<(unsigned)expand, 256, 0, st>>>(p);
                    return;
                }
            }
            if (shrink && streams_x(plan, c)) adapter_shrink<T, RT, true><<<(unsigned)shrink, 256, lds, st>>>(p);
            else if (shrink) adapter_shrink<T, RT, false><<<(unsigned)shrink, 256, lds, st>>>(p);
            if (!expand) return;
            if (ST == 1) adapter_expand<T, RX.value, kSub, false, false><<<(unsigned)expand, 256, 0, st>>>(p);
            else if (streams(plan, c)) adapter_expand<T, RX.value, kTile, false, true><<<(unsigned)expand, 256, 0, st>>>(p);
            else adapter_expand<T, RX.value, kTile, false, false><<<(unsigned)expand, 256, 0, st>>>(p);
        });
    };
    if (c->dtype == KVMIX_F16) run((_Float16)0);
    else run((__bf16)0.0f);
    return launch_status();
}
