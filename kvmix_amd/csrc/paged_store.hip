// The pages of a cache written, quantized, read back and copied (paged_common.h says what a page holds).  All of it is bound by
// memory, or by the launch where there is little of it.
#include <stdlib.h>

#include <algorithm>
#include <type_traits>

#include "paged_common.h"

namespace kvmix {

constexpr int kStorePairs = 400;  // (source, destination) pages, or single pages, that travel as kernel arguments
constexpr int kCopyPools = 32;

struct PagePairs {
    int2 at[kStorePairs];
};

// ---------------------------------------------------------------------------------------------------------------------
// append: the new tokens of one block of a page and one head per wave (the plan lists such blocks).  Keys are copied as they
// come; values go through the LDS, turned round: eight tokens that follow one another in a page are one piece of sixteen bytes
// (token by token, two bytes at a time, 83 instead of 62 us for 8 x 1021 tokens of 32 heads).  A single token's values touch D
// rows of 64 bytes: sixteen times the lines that it has to, for a store that is read at every step after it.  8 x 1021 tokens:
// 62 us for 268 MB moved, 4.3 TB/s (a large copy 4.75); 64 x 1 of 8 heads 4.8 us, a launch.

struct AppendArgs {
    const _Float16 *k, *v;
    int64_t k_ts, k_hs, v_ts, v_hs;
    _Float16 *rows;
    PlanWords blocks;
    int heads, units, page_log2;  // units: blocks of tokens by heads
};

template <int D>
__global__ void __launch_bounds__(256) paged_append(AppendArgs a)
{
    constexpr int C = D / 8;  // 16-byte pieces of a token
    constexpr int kTurns = kBlock * C / kWave;
    __shared__ _Float16 turned[4][kBlock][D + 2];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int unit = blockIdx.x * 4 + wave;
    if (unit >= a.units) return;  // (waves share nothing but the array, of which each has its own part)
    const int head = unit % a.heads;
    const PlanWords p = a.blocks + unit / a.heads * kStoreWords;
    const int64_t token = p[0];
    const int slot = p[1], n = p[2], place = slot & (kBlock - 1), page = slot >> a.page_log2, in_page = (slot & ((1 << a.page_log2) - 1)) - place;
    _Float16 *keys = a.rows + ((((int64_t)page * a.heads + head) * 2) << a.page_log2) * D + (int64_t)in_page * D;
    _Float16 *values = keys + ((int64_t)D << a.page_log2);
    const _Float16 *k = a.k + token * a.k_ts + head * a.k_hs, *v = a.v + token * a.v_ts + head * a.v_hs;
    half8v key[kTurns], value[kTurns];
#pragma unroll
    for (int i = 0; i < kTurns; i++) {
        const int t = (i * kWave + lane) / C, c = (i * kWave + lane) % C;
        if (t < n) {
            key[i] = *(const half8v *)(k + t * a.k_ts + 8 * c);
            value[i] = *(const half8v *)(v + t * a.v_ts + 8 * c);
        }
    }
#pragma unroll
    for (int i = 0; i < kTurns; i++) {
        const int t = (i * kWave + lane) / C, c = (i * kWave + lane) % C;
        if (t < n) {
            *(half8v *)(keys + (place + t) * D + 8 * c) = key[i];
#pragma unroll
            for (int j = 0; j < 4; j++) *(half2v *)&turned[wave][place + t][8 * c + 2 * j] = half2v{value[i][2 * j], value[i][2 * j + 1]};
        }
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS operations are done in order)
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    // eight tokens of one channel: as one piece, or the new ones of them
    const int first = place / 8, last = (place + n - 1) / 8;
    for (int i = lane; i < D * 4; i += kWave) {
        const int d = i / 4, g = i % 4;
        if (g < first || g > last) continue;
        if (8 * g >= place && 8 * g + 8 <= place + n) {
            half8v w;
#pragma unroll
            for (int j = 0; j < 8; j++) w[j] = turned[wave][8 * g + j][d];
            *(half8v *)(values + d * kBlock + 8 * g) = w;
        } else {
            for (int t = max(8 * g, place); t < min(8 * g + 8, place + n); t++) values[d * kBlock + t] = turned[wave][t][d];
        }
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// The pieces of one matrix of a block of an fp16 page, in the packed order: keys piece u * D / 32 + s, values piece t.

template <int D, bool KEYS>
__device__ __forceinline__ half8v row_piece(const _Float16 *page_head, int page, int block, int lane, int piece)
{
    const int m = lane % 16, g = lane / 16;
    if constexpr (KEYS) {
        const int u = piece / (D / 32), s = piece % (D / 32);
        return *(const half8v *)(page_head + (int64_t)(block * kBlock + 8 * (m / 4) + 4 * u + m % 4) * D + 32 * s + 8 * g);
    } else {
        return *(const half8v *)(page_head + (int64_t)page * D + (int64_t)block * kBlock * D + (16 * piece + m) * kBlock + 8 * g);
    }
}

struct QuantizeArgs {
    const _Float16 *rows;
    uint32_t *packed;
    int heads, page;
    int k_bits, v_bits;
};

// (the builtins quiet both operands first, three operations for one)
__device__ __forceinline__ uint32_t pair_min(uint32_t a, uint32_t b)
{
    uint32_t o;
    asm("v_pk_min_f16 %0, %1, %2" : "=v"(o) : "v"(a), "v"(b));
    return o;
}

__device__ __forceinline__ uint32_t pair_max(uint32_t a, uint32_t b)
{
    uint32_t o;
    asm("v_pk_max_f16 %0, %1, %2" : "=v"(o) : "v"(a), "v"(b));
    return o;
}

// One halving step over the lanes of a row of sixteen whose numbers differ in the bits of MASK (15, 7, 3, 1: mirrors of the row,
// of its halves, of quarters and of pairs): the lane with MASK's highest bit clear gets the lower half of v over the pair.
template <int MASK, bool MAX, int N>
__device__ __forceinline__ void halve_pairs(uint32_t *v, int lane)
{
    constexpr int control = MASK == 15 ? 0x140 : MASK == 7 ? 0x141 : MASK == 3 ? 0x1b : 0xb1;
    const bool up = (lane & (MASK + 1) / 2) != 0;
#pragma unroll
    for (int i = 0; i < N / 2; i++) {
        const uint32_t keep = up ? v[N / 2 + i] : v[i], send = up ? v[i] : v[N / 2 + i];
        const uint32_t other = __builtin_amdgcn_update_dpp(0, send, control, 0xf, 0xf, true);
        v[i] = MAX ? pair_max(keep, other) : pair_min(keep, other);
    }
}

// A wave's groups, 32 tokens' or channels': minimum, reciprocal of the scale, scale; and a matrix's words as they are put together.
struct GroupTable {
    float at[4][4][8];  // [row of lanes][pair of groups][minimum, reciprocal, minimum, reciprocal, scale, scale]
};

// A quarter of one matrix of one block per wave (half at D = 64): the groups of 32 channels (keys) or tokens (values), of each of
// which a lane has two values and the sixteen lanes of a row the rest.  Extremes are found by halving, so that each lane ends with
// the two groups whose scales it works out for the row.  With a matrix to a wave, every lane working out all its groups and a
// branch for every two codes, 120 pages of 32 heads took 54 instead of 51 us; without the last two 42, but four pages of 8 heads 10.7
// instead of 6.3: that much code in a line takes longer to arrive than to run.  The codes are those of kvmix_quant_pack_last_dim
// with KVMIX_SCALE_RECIPROCAL, bit for bit.
template <int D, int BITS, bool KEYS>
__device__ __forceinline__ void quantize_set(const _Float16 *from, int page, int block, int set, uint32_t *words, _Float16 *side, int lane, GroupTable &table)
{
    constexpr int S = D / 32, N = lane_words(D, BITS), R = run_words(N);
    constexpr int QMAX = (1 << BITS) - 1;
    const int g = lane / 16;
    half8v x[2];
#pragma unroll
    for (int w = 0; w < 2; w++) x[w] = row_piece<D, KEYS>(from, page, block, lane, KEYS ? w * S + set : 2 * set + w);
    uint32_t lo[4], hi[4];
    const uint4v a = __builtin_bit_cast(uint4v, x[0]), b = __builtin_bit_cast(uint4v, x[1]);
#pragma unroll
    for (int j = 0; j < 4; j++) lo[j] = pair_min(a[j], b[j]), hi[j] = pair_max(a[j], b[j]);
    halve_pairs<15, false, 4>(lo, lane), halve_pairs<15, true, 4>(hi, lane);
    halve_pairs<7, false, 2>(lo, lane), halve_pairs<7, true, 2>(hi, lane);
    // (one left: the lanes of a quarter all get it)
    lo[0] = pair_min(lo[0], __builtin_amdgcn_update_dpp(0, lo[0], 0x1b, 0xf, 0xf, true));
    hi[0] = pair_max(hi[0], __builtin_amdgcn_update_dpp(0, hi[0], 0x1b, 0xf, 0xf, true));
    lo[0] = pair_min(lo[0], __builtin_amdgcn_update_dpp(0, lo[0], 0xb1, 0xf, 0xf, true));
    hi[0] = pair_max(hi[0], __builtin_amdgcn_update_dpp(0, hi[0], 0xb1, 0xf, 0xf, true));
    const int mine = lane % 16 / 4;
    {
        const half2v l = __builtin_bit_cast(half2v, lo[0]), h = __builtin_bit_cast(half2v, hi[0]);
        half2v scales;
        float fast[4], exact[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            const float mn = (float)l[i], range = (float)h[i] - mn, scale = range / (float)QMAX;
            fast[2 * i] = mn, fast[2 * i + 1] = quantize_rcp(scale), exact[i] = scale;
            scales[i] = (_Float16)scale_for_output(range, scale, 1.0f / (float)QMAX, KVMIX_SCALE_RECIPROCAL);
        }
        if (lane % 4 == 0) {
            *(floatx4 *)table.at[g][mine] = floatx4{fast[0], fast[1], fast[2], fast[3]};
            table.at[g][mine][4] = exact[0], table.at[g][mine][5] = exact[1];
            _Float16 *at = side + 32 * set + 8 * g + 2 * mine;
            *(half2v *)at = scales;
            *(uint32_t *)(at + D) = lo[0];
        }
    }
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS operations are done in order)
    uint32_t q[2][8];
    bool near = false;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const floatx4 f = *(const floatx4 *)table.at[g][p];
#pragma unroll
        for (int i = 0; i < 2; i++) {
#pragma unroll
            for (int w = 0; w < 2; w++) {
                // (as quantize_code_fast, but for the limit: a quotient above it is near)
                const float u = fmaf((float)x[w][2 * p + i] - f[2 * i], f[2 * i + 1], 0.5f);
                near |= !(fabsf(__builtin_amdgcn_fractf(u) - 0.5f) <= 0.5f - 0.000030517578125f);
                q[w][2 * p + i] = (uint32_t)u;
            }
        }
    }
    if (__builtin_expect(near, 0)) {
#pragma unroll 1
        for (int p = 0; p < 4; p++) {  // (values and codes by selection: a loop over registers)
#pragma unroll
            for (int i = 0; i < 2; i++) {
#pragma unroll
                for (int w = 0; w < 2; w++) {
                    const half8v y = x[w];
                    const float v = (float)(p == 0 ? y[i] : p == 1 ? y[2 + i] : p == 2 ? y[4 + i] : y[6 + i]);
                    const uint32_t c = quantize_code(v, table.at[g][p][2 * i], table.at[g][p][4 + i], QMAX);
#pragma unroll
                    for (int k = 0; k < 4; k++) q[w][2 * k + i] = k == p ? c : q[w][2 * k + i];
                }
            }
        }
    }
    auto put = [&](int word, uint32_t bits) { atomicOr(&words[word / R * kWave * R + lane * R + word % R], bits); };
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const int piece = KEYS ? w * S + set : 2 * set + w;
        if constexpr (BITS != 3) {  // a piece is a part of one word
            uint32_t part = 0;
#pragma unroll
            for (int p = 0; p < 4; p++) part |= (q[w][2 * p] | q[w][2 * p + 1] << 16) << (BITS * p);
            put(piece * BITS / 4, part << (piece * BITS % 4 * 4));
        } else {
#pragma unroll
            for (int p = 0; p < 4; p++) {
                const uint32_t c = q[w][2 * p] | q[w][2 * p + 1] << 16;
                const int t = 4 * piece + p;
                if (t < 5 * N) {
                    put(t / 5, c << (t % 5 * 3));
                } else {
#pragma unroll
                    for (int i = 0; i < 3; i++) put(3 * (t - 5 * N) + i, (c >> i & 0x00010001u) << 15);
                }
            }
        }
    }
}

template <int D>
__global__ void __launch_bounds__(256) paged_quantize(QuantizeArgs a, PagePairs pairs)
{
    constexpr int S = D / 32, M = 4 / S;  // waves to a matrix, matrices to a block
    __shared__ GroupTable tables[4];
    __shared__ __attribute__((aligned(16))) uint32_t words[M][kWave * lane_words(D, 4)];
    const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int2 pair = pairs.at[blockIdx.y];  // (at once with the other arguments, which come from far)
    const int unit = blockIdx.x * M + wave / S, set = wave % S;
    const int blocks = a.page / kBlock, values = unit % 2, block = unit / 2 % blocks, head = unit / 2 / blocks;
    const _Float16 *from = a.rows + ((int64_t)pair.x * a.heads + head) * 2 * a.page * D;
    uint32_t *to = a.packed + (((int64_t)pair.y * a.heads + head) * blocks + block) * block_words(D, a.k_bits, a.v_bits);
    _Float16 *side = (_Float16 *)(to + D * (a.k_bits + a.v_bits));
    uint32_t *mine = words[wave / S];
    for (int i = set * kWave + lane; i < kWave * lane_words(D, 4) / 4; i += S * kWave) ((uint4v *)mine)[i] = uint4v{0, 0, 0, 0};
    __syncthreads();
    if (values) with_bits(a.v_bits, [&](auto B) { quantize_set<D, B.value, false>(from, a.page, block, set, mine, side + 2 * D, lane, tables[wave]); });
    else with_bits(a.k_bits, [&](auto B) { quantize_set<D, B.value, true>(from, a.page, block, set, mine, side, lane, tables[wave]); });
    __syncthreads();
    const int bits = values ? a.v_bits : a.k_bits;
    to += values ? D * a.k_bits : 0;
    for (int i = set * kWave + lane; i < D * bits / 4; i += S * kWave) ((uint4v *)to)[i] = ((const uint4v *)mine)[i];
}

// ---------------------------------------------------------------------------------------------------------------------
// read: the values of pages, token by token: [pages, P, heads, D].  A block of one head per wave pair, keys and values.  Bound by its
// writes: 120 pages of 32 heads, 3/2 bits, 25 us (126 MB written, 28 read: 6.1 TB/s); four pages of 8 heads 3.8, a launch; 120 fp16 pages 42 us
// (252 MB, 6.0 TB/s).

struct ReadArgs {
    const void *pool;
    _Float16 *k, *v;
    int heads, page, units;
    int k_bits, v_bits;
};

template <int D, bool ROWS>
__global__ void __launch_bounds__(256) paged_read(ReadArgs a, PagePairs ids)
{
    constexpr int NP = D / 16;
    __shared__ _Float16 turned[4][kBlock][D + 8];
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, m = lane % 16, g = lane / 16;
    const int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + wave);
    if (unit >= a.units) return;  // (waves share nothing but the array, of which each has its own part)
    const int nth = blockIdx.y;
    const int2 two = ids.at[nth / 2];
    const int64_t id = nth % 2 ? two.y : two.x;
    const int blocks = a.page / kBlock, values = unit % 2, block = unit / 2 % blocks, head = unit / 2 / blocks;
    half8v x[NP];
    if constexpr (ROWS) {
        const _Float16 *from = (const _Float16 *)a.pool + (id * a.heads + head) * 2 * a.page * D;
#pragma unroll
        for (int p = 0; p < NP; p++) x[p] = values ? row_piece<D, false>(from, a.page, block, lane, p) : row_piece<D, true>(from, a.page, block, lane, p);
    } else {
        const uint32_t *from = (const uint32_t *)a.pool + ((id * a.heads + head) * blocks + block) * block_words(D, a.k_bits, a.v_bits);
        const _Float16 *side = (const _Float16 *)(from + D * (a.k_bits + a.v_bits)) + (values ? 2 * D : 0) + 8 * g;
        with_bits(values ? a.v_bits : a.k_bits, [&](auto B) {
            constexpr int N = lane_words(D, B.value);
            uint32_t w[N];
            load_words<N>(values ? from + D * a.k_bits : from, lane, w);
            const Exponents<B.value> e;
#pragma unroll
            for (int p = 0; p < NP; p++) {
                const int s = values ? p / 2 : p % (D / 32);
                x[p] = piece_values<B.value, N>(w, p, *(const half8v *)(side + 32 * s), *(const half8v *)(side + D + 32 * s), e);
            }
        });
    }
    const int64_t token0 = (int64_t)nth * a.page + block * kBlock;
    if (!values) {
#pragma unroll
        for (int p = 0; p < NP; p++) {
            const int u = p / (D / 32), s = p % (D / 32);
            *(half8v *)(a.k + ((token0 + 8 * (m / 4) + 4 * u + m % 4) * a.heads + head) * D + 32 * s + 8 * g) = x[p];
        }
        return;
    }
#pragma unroll
    for (int p = 0; p < NP; p++) {
#pragma unroll
        for (int j = 0; j < 8; j++) turned[wave][8 * g + j][16 * p + m] = x[p][j];
    }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();  // (a wave's LDS operations are done in order)
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int i = 0; i < kBlock * D / 8 / kWave; i++) {
        const int at = i * kWave + lane, t = at / (D / 8), c = at % (D / 8);
        *(half8v *)(a.v + ((token0 + t) * a.heads + head) * D + 8 * c) = *(const half8v *)&turned[wave][t][8 * c];
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// copy: pages of up to kCopyPools pools, the same pairs in all of them, 16 KiB to a block: four loads of sixteen bytes in flight per
// thread, then their stores.  2.9 GB moved in 701 pages of 32 pools 579 us, 5.1 TB/s; 134 MB in 32 us with its launch.

constexpr int kCopyPieces = 4;  // of 16 bytes per thread
constexpr uint32_t kCopyBytes = 256 * 16 * kCopyPieces;

struct CopyArgs {
    uint8_t *pool[kCopyPools];
    uint32_t bytes[kCopyPools];      // of a page
    uint32_t blocks[kCopyPools];     // up to and with this pool
    int pools;
};

__global__ void __launch_bounds__(256) paged_copy(CopyArgs a, PagePairs pairs)
{
    const uint32_t at = blockIdx.x;
    const int2 pair = pairs.at[blockIdx.y];
    int p = 0;
    while (at >= a.blocks[p]) p++;
    const uint32_t piece = at - (p ? a.blocks[p - 1] : 0);
    const uint32_t bytes = a.bytes[p];
    const uint8_t *src = a.pool[p] + (int64_t)pair.x * bytes;
    uint8_t *dst = a.pool[p] + (int64_t)pair.y * bytes;
    if (__builtin_expect(bytes % 16 != 0, 0)) {  // (pages that begin between pieces of sixteen bytes)
        for (uint32_t off = piece * kCopyBytes + threadIdx.x * 8; off < (piece + 1) * kCopyBytes && off < bytes; off += 256 * 8)
            *(uint2v *)(dst + off) = *(const uint2v *)(src + off);
        return;
    }
    uint4v v[kCopyPieces];
#pragma unroll
    for (int i = 0; i < kCopyPieces; i++) {
        const uint32_t off = piece * kCopyBytes + (i * 256 + threadIdx.x) * 16;
        if (off < bytes) v[i] = *(const uint4v *)(src + off);
    }
#pragma unroll
    for (int i = 0; i < kCopyPieces; i++) {
        const uint32_t off = piece * kCopyBytes + (i * 256 + threadIdx.x) * 16;
        if (off < bytes) *(uint4v *)(dst + off) = v[i];
    }
}

// ---------------------------------------------------------------------------------------------------------------------

}  // namespace kvmix

using namespace kvmix;

namespace {

// Whether no page is written twice by these pairs, nor (`read_too`) written and read.
int pairs_apart(const int32_t *pairs, int64_t count, bool read_too)
{
    int32_t *written = (int32_t *)malloc((size_t)count * sizeof(int32_t));
    if (!written) return KVMIX_ERR_MEMORY;
    for (int64_t i = 0; i < count; i++) written[i] = pairs[2 * i + 1];
    std::sort(written, written + count);
    bool apart = std::adjacent_find(written, written + count) == written + count;
    for (int64_t i = 0; read_too && apart && i < count; i++) apart = !std::binary_search(written, written + count, pairs[2 * i]);
    free(written);
    return apart ? KVMIX_OK : KVMIX_ERR_PAGE_ORDER;
}

}  // namespace

extern "C" int kvmix_paged_append(const kvmix_paged_pool_t *p, const kvmix_paged_plan_t *plan, const int32_t *list, const void *k,
                                  int64_t k_token_stride, int64_t k_head_stride, const void *v, int64_t v_token_stride, int64_t v_head_stride,
                                  kvmix_stream_t stream)
{
    const int rc = pool_check(p);
    if (rc != KVMIX_OK) return rc;
    if (!plan) return KVMIX_ERR_NULL;
    if (plan->page_size != p->page_size) return KVMIX_ERR_SHAPE;
    if (plan->row_pages > p->row_pages) return KVMIX_ERR_PAGE;
    if (k_token_stride % 8 || k_head_stride % 8 || v_token_stride % 8 || v_head_stride % 8 || ((uintptr_t)k | (uintptr_t)v) % 16) return KVMIX_ERR_UNSUPPORTED;
    if (plan->stores == 0) return KVMIX_OK;
    if (!k || !v || !list || !p->rows) return KVMIX_ERR_NULL;
    if ((__int128)plan->stores * p->kv_heads > 4 * kMostBlocks) return KVMIX_ERR_UNSUPPORTED;  // (four units to a block)
    const AppendArgs a = {(const _Float16 *)k, (const _Float16 *)v, k_token_stride, k_head_stride, v_token_stride, v_head_stride, (_Float16 *)p->rows,
                          (PlanWords)list + plan->store_at, (int)p->kv_heads, (int)(plan->stores * p->kv_heads),
                          __builtin_ctzll((uint64_t)p->page_size)};
    const unsigned grid = (unsigned)((plan->stores * p->kv_heads + 3) / 4);
    with_dim(p->head_dim, [&](auto D) { paged_append<D.value><<<grid, 256, 0, (hipStream_t)stream>>>(a); });
    return launch_status();
}

extern "C" int kvmix_paged_quantize(const kvmix_paged_pool_t *p, const int32_t *pairs, int64_t count, kvmix_stream_t stream)
{
    int rc = pool_check(p);
    if (rc == KVMIX_OK) rc = bits_check(p);
    if (rc != KVMIX_OK) return rc;
    if (count < 0) return KVMIX_ERR_SHAPE;
    if (count == 0) return KVMIX_OK;
    if (!pairs || !p->rows || !p->packed) return KVMIX_ERR_NULL;
    for (int64_t i = 0; i < count; i++)
        if (pairs[2 * i] < 0 || pairs[2 * i] >= p->row_pages || pairs[2 * i + 1] < 0 || pairs[2 * i + 1] >= p->packed_pages) return KVMIX_ERR_PAGE;
    rc = pairs_apart(pairs, count, false);
    if (rc != KVMIX_OK) return rc;
    const int64_t per = p->kv_heads * (p->page_size / kBlock) * 2;
    for (int64_t first = 0; first < count; first += kStorePairs) {
        const int n = (int)(count - first < kStorePairs ? count - first : kStorePairs);
        PagePairs list{};
        for (int i = 0; i < n; i++) list.at[i] = make_int2(pairs[2 * (first + i)], pairs[2 * (first + i) + 1]);
        const QuantizeArgs a = {(const _Float16 *)p->rows, (uint32_t *)p->packed, (int)p->kv_heads, (int)p->page_size, p->k_bits, p->v_bits};
        const dim3 grid((unsigned)(per / (128 / p->head_dim)), (unsigned)n);
        with_dim(p->head_dim, [&](auto D) { paged_quantize<D.value><<<grid, 256, 0, (hipStream_t)stream>>>(a, list); });
        if (launch_status() != KVMIX_OK) return KVMIX_ERR_LAUNCH;
    }
    return KVMIX_OK;
}

extern "C" int kvmix_paged_read(const kvmix_paged_pool_t *p, int packed, const int32_t *pages, int64_t count, void *k, void *v, kvmix_stream_t stream)
{
    int rc = pool_check(p);
    if (rc == KVMIX_OK && packed) rc = bits_check(p);
    if (rc != KVMIX_OK) return rc;
    if (count < 0) return KVMIX_ERR_SHAPE;
    if (count == 0) return KVMIX_OK;
    if (!pages || !k || !v || !(packed ? p->packed : p->rows)) return KVMIX_ERR_NULL;
    if (((uintptr_t)k | (uintptr_t)v) % 16) return KVMIX_ERR_UNSUPPORTED;
    for (int64_t i = 0; i < count; i++)
        if (pages[i] < 0 || pages[i] >= (packed ? p->packed_pages : p->row_pages)) return KVMIX_ERR_PAGE;
    const int64_t per = p->kv_heads * (p->page_size / kBlock) * 2, most = 2 * kStorePairs, size = p->page_size * p->kv_heads * p->head_dim;
    for (int64_t first = 0; first < count; first += most) {
        const int n = (int)(count - first < most ? count - first : most);
        PagePairs list{};
        for (int i = 0; i < n; i++) (i % 2 ? list.at[i / 2].y : list.at[i / 2].x) = pages[first + i];
        const ReadArgs a = {packed ? p->packed : p->rows, (_Float16 *)k + first * size, (_Float16 *)v + first * size, (int)p->kv_heads,
                            (int)p->page_size, (int)per, p->k_bits, p->v_bits};
        const dim3 grid((unsigned)((per + 3) / 4), (unsigned)n);
        with_dim(p->head_dim, [&](auto D) {
            if (packed) paged_read<D.value, false><<<grid, 256, 0, (hipStream_t)stream>>>(a, list);
            else paged_read<D.value, true><<<grid, 256, 0, (hipStream_t)stream>>>(a, list);
        });
        if (launch_status() != KVMIX_OK) return KVMIX_ERR_LAUNCH;
    }
    return KVMIX_OK;
}

extern "C" int kvmix_paged_copy(void *const *pools, const int64_t *page_bytes, int64_t n_pools, int64_t pages, const int32_t *pairs, int64_t count,
                                kvmix_stream_t stream)
{
    if (n_pools < 0 || count < 0 || pages < 0) return KVMIX_ERR_SHAPE;
    if (n_pools == 0 || count == 0) return KVMIX_OK;
    if (!pools || !page_bytes || !pairs) return KVMIX_ERR_NULL;
    for (int64_t i = 0; i < n_pools; i++) {
        if (page_bytes[i] < 0) return KVMIX_ERR_SHAPE;
        if (page_bytes[i] % 8 != 0 || page_bytes[i] > (1 << 28) || (uintptr_t)pools[i] % 16 != 0) return KVMIX_ERR_UNSUPPORTED;
        if (!pools[i] && page_bytes[i]) return KVMIX_ERR_NULL;
    }
    // Pairs are done in no particular order: a page is written once at most, and no page that is written is read.
    if (pages > kMost32) return KVMIX_ERR_UNSUPPORTED;
    for (int64_t i = 0; i < 2 * count; i++)
        if (pairs[i] < 0 || pairs[i] >= pages) return KVMIX_ERR_PAGE;
    const int rc = pairs_apart(pairs, count, true);
    if (rc != KVMIX_OK) return rc;
    for (int64_t p0 = 0; p0 < n_pools; p0 += kCopyPools) {
        CopyArgs a{};
        a.pools = (int)(n_pools - p0 < kCopyPools ? n_pools - p0 : kCopyPools);
        uint32_t blocks = 0;
        for (int i = 0; i < a.pools; i++) {
            a.pool[i] = (uint8_t *)pools[p0 + i];
            a.bytes[i] = (uint32_t)page_bytes[p0 + i];
            blocks += (uint32_t)((page_bytes[p0 + i] + kCopyBytes - 1) / kCopyBytes);
            a.blocks[i] = blocks;
        }
        if (blocks == 0) continue;
        for (int64_t first = 0; first < count; first += kStorePairs) {
            const int64_t n = count - first < kStorePairs ? count - first : kStorePairs;
            PagePairs list{};
            for (int64_t i = 0; i < n; i++) list.at[i] = make_int2(pairs[2 * (first + i)], pairs[2 * (first + i) + 1]);
            paged_copy<<<dim3(blocks, (unsigned)n), 256, 0, (hipStream_t)stream>>>(a, list);
            if (launch_status() != KVMIX_OK) return KVMIX_ERR_LAUNCH;
        }
    }
    return KVMIX_OK;
}
