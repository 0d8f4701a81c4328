// What the kernels of the paged cache share: where things lie in a page, and codes to values and back.
//
// A page holds P tokens (a multiple of 32) of one layer, for every kv head.  Blocks of 32 tokens are the unit of everything:
//   fp16 page      keys [P][D], then per block the values as [D][32] (what a matrix instruction wants of them is eight tokens
//                  of one channel, so they are turned round when they are stored, once, and not at every read)
//   packed page    per block D * (KB + VB + 2) words: key codes, value codes, then 4 D halves: the keys' scale and minimum per
//                  channel, the values' per token, [D / 32 groups][32 tokens]
// Codes lie in the order of the lanes of v_mfma_f32_16x16x32: lane 16 g + m has pieces of eight codes, of the keys piece
// u * D / 32 + s = channels 32 s + 8 g + (0..7) of token 8 (m / 4) + 4 u + m % 4, of the values piece t = tokens 8 g + (0..7) of
// channel 16 t + m.  With the keys' rows in that order the logits that a lane holds after q.K^T are those of tokens 8 g +
// (0..7): they are its operand of p.V as they stand.  The D / 16 pieces of a lane fill D * bits / 64 words; a wave reads them
// as whole runs of 16 (8, 4) bytes per lane.  Codes lie in the word so that two of them come out as a pair of halves with one
// or two instructions: the pair's first code in the low half, its second at the same place in the high half.
#pragma once

#include <type_traits>

#include "kvmix_common.h"

namespace kvmix {

typedef _Float16 half2v __attribute__((ext_vector_type(2)));
typedef _Float16 half8v __attribute__((ext_vector_type(8)));
typedef float floatx4 __attribute__((ext_vector_type(4)));
typedef uint32_t uint4v __attribute__((ext_vector_type(4)));
typedef uint32_t uint2v __attribute__((ext_vector_type(2)));

constexpr int kBlock = 32;      // tokens
constexpr int kStoreWords = 4;  // new tokens of one block of a page: the first one's number, its page * page_size + place, how many; one of no use

// The plan's words: nobody writes them while a kernel runs, so they are read through the scalar cache (as ordinary memory every
// look at a page table waited for all loads in flight).
typedef const __attribute__((address_space(4))) int32_t *PlanWords;

__host__ __device__ constexpr int lane_words(int D, int bits) { return D * bits / 64; }
__host__ __device__ constexpr int run_words(int words) { return words % 4 == 0 ? 4 : words % 2 == 0 ? 2 : 1; }
__host__ __device__ constexpr int block_words(int D, int kb, int vb) { return D * (kb + vb + 2); }

// A lane's words of one matrix of a block.
template <int N>
__device__ __forceinline__ void load_words(const uint32_t *at, int lane, uint32_t *w)
{
    constexpr int R = run_words(N);
#pragma unroll
    for (int i = 0; i < N / R; i++) {
        const uint32_t *p = at + i * kWave * R + lane * R;
        if constexpr (R == 4) {
            const uint4v v = *(const uint4v *)p;
#pragma unroll
            for (int j = 0; j < 4; j++) w[4 * i + j] = v[j];
        } else if constexpr (R == 2) {
            const uint2v v = *(const uint2v *)p;
            w[2 * i] = v[0], w[2 * i + 1] = v[1];
        } else {
            w[i] = *p;
        }
    }
}

template <int N>
__device__ __forceinline__ void store_words(uint32_t *at, int lane, const uint32_t *w)
{
    constexpr int R = run_words(N);
#pragma unroll
    for (int i = 0; i < N / R; i++) {
        uint32_t *p = at + i * kWave * R + lane * R;
        if constexpr (R == 4) *(uint4v *)p = uint4v{w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]};
        else if constexpr (R == 2) *(uint2v *)p = uint2v{w[2 * i], w[2 * i + 1]};
        else *p = w[i];
    }
}

// Pairs of codes to a word.  Three-bit pairs past 5 N of a lane's N words take the top bits of three words' halves, one bit from each.
__host__ __device__ constexpr int word_pairs(int bits) { return bits == 3 ? 5 : 16 / bits; }

// Pair `t` as two halves that hold the codes exactly.  A field at bit s of a half, under the exponent of 2^(10 - s), is the code
// plus 2^(10 - s): the bits are masked in place, in one operation with the exponent (v_and_or_b32 takes one scalar and no
// literal: the exponents are kept in registers, Exponents below), and that is subtracted.
template <int BITS>
struct Exponents {
    // fields lie in the ten bits of a half's fraction, or are shifted there
    static constexpr int shift = BITS == 4 ? 8 : BITS == 3 ? 9 : 10;
    static constexpr int count = (10 - BITS) / BITS + 1;
    uint32_t at[count];

    __device__ __forceinline__ Exponents()
    {
#pragma unroll
        for (int i = 0; i < count; i++) {
            const uint32_t e = (0x6400u - 0x400u * (i * BITS)) * 0x00010001u;
            asm volatile("v_mov_b32 %0, %1" : "=v"(at[i]) : "s"(e));
        }
    }
};

template <int BITS, int N>
__device__ __forceinline__ half2v code_pair(const uint32_t *w, int t, const Exponents<BITS> &e)
{
    constexpr uint32_t ones = 0x00010001u;
    constexpr uint32_t mask = (1u << BITS) - 1;
    constexpr int per = word_pairs(BITS);
    if (t >= N * per) {  // (3 bits only)
        const int r = 3 * (t - N * per);
        const uint32_t c = (w[r] >> 15 & ones) | (w[r + 1] >> 14 & 2 * ones) | (w[r + 2] >> 13 & 4 * ones) | e.at[0];
        return __builtin_bit_cast(half2v, c) - half2v{(_Float16)1024.0f, (_Float16)1024.0f};
    }
    int s = t % per * BITS;
    uint32_t v = w[t / per], c;
    if (s + BITS > 10) v >>= Exponents<BITS>::shift, s -= Exponents<BITS>::shift;
    asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(c) : "v"(v), "s"(mask * ones << s), "v"(e.at[s / BITS]));
    const _Float16 base = (_Float16)(float)(1 << (10 - s));
    return __builtin_bit_cast(half2v, c) - half2v{base, base};
}

// Piece `piece` of a lane's words: its codes, and its values code * scale + zero, each rounded once, to fp16.
template <int BITS, int N>
__device__ __forceinline__ half8v piece_codes(const uint32_t *w, int piece, const Exponents<BITS> &e)
{
    half8v out;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const half2v c = code_pair<BITS, N>(w, 4 * piece + p, e);
        out[2 * p] = c[0], out[2 * p + 1] = c[1];
    }
    return out;
}

// The codes of a piece of two- or four-bit codes in the order 0 4 1 5 2 6 3 7, by the conversions of small floating-point formats,
// two codes to an operation: two bits as four-bit numbers of the format e2m1, whose 0 .. 3 are 0, 1/2, 1, 3/2 (eleven
// operations for sixteen codes instead of seventeen), four bits as bytes of the format e4m3, whose 0 .. 15 are these numbers times 2^-9
// (seven operations for eight codes instead of nine).
__device__ __forceinline__ half8v turned(half8v v) { return __builtin_shufflevector(v, v, 0, 4, 1, 5, 2, 6, 3, 7); }
__device__ __forceinline__ half8v turned_back(half8v v) { return __builtin_shufflevector(v, v, 0, 2, 4, 6, 1, 3, 5, 7); }

template <int BITS>
__device__ __forceinline__ half8v piece_codes_turned(const uint32_t *w, int piece)
{
    static_assert(BITS == 2 || BITS == 4, "");
    if constexpr (BITS == 4) {
        const uint32_t even = w[piece] & 0x0f0f0f0fu, odd = w[piece] >> 4 & 0x0f0f0f0fu;
        const half2v a = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, false), b = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(even, 512.0f, true);
        const half2v c = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, false), d = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(odd, 512.0f, true);
        return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    } else {
        const uint32_t even = w[piece / 2] & 0x33333333u, odd = w[piece / 2] >> 2 & 0x33333333u;
        const half2v a = piece % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 2.0f, 1) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 2.0f, 0);
        const half2v b = piece % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 2.0f, 3) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(even, 2.0f, 2);
        const half2v c = piece % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 2.0f, 1) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 2.0f, 0);
        const half2v d = piece % 2 ? __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 2.0f, 3) : __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(odd, 2.0f, 2);
        return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
    }
}

template <int BITS, int N>
__device__ __forceinline__ half8v piece_values(const uint32_t *w, int piece, half8v scale, half8v zero, const Exponents<BITS> &e)
{
    return __builtin_elementwise_fma(piece_codes<BITS, N>(w, piece, e), scale, zero);
}

constexpr int64_t kMost32 = 0x7fffffff;
constexpr int64_t kMostBlocks = (1 << 24) - 1;  // of 256 threads: a launch of 2^32 threads or more runs modulo 2^32, without an error
constexpr int64_t kMostHeads = 4096;

inline bool page_size_ok(int64_t n) { return n >= kBlock && n <= 1024 && (n & (n - 1)) == 0; }

// Sizes that every call on pages shares.
inline int pool_check(const kvmix_paged_pool_t *p)
{
    if (!p) return KVMIX_ERR_NULL;
    if (p->kv_heads <= 0 || p->row_pages < 0 || p->packed_pages < 0) return KVMIX_ERR_SHAPE;
    if ((p->head_dim != 64 && p->head_dim != 128) || !page_size_ok(p->page_size) || p->kv_heads > kMostHeads)
        return KVMIX_ERR_UNSUPPORTED;
    if ((__int128)p->row_pages * p->page_size > kMost32 || p->packed_pages > kMost32) return KVMIX_ERR_UNSUPPORTED;
    if (((uintptr_t)p->rows | (uintptr_t)p->packed) % 16 != 0) return KVMIX_ERR_UNSUPPORTED;
    return KVMIX_OK;
}

inline int bits_check(const kvmix_paged_pool_t *p)
{
    return p->k_bits < 1 || p->k_bits > 4 || p->v_bits < 1 || p->v_bits > 4 ? KVMIX_ERR_BITS : KVMIX_OK;
}

template <typename F>
void with_dim(int64_t D, F f)
{
    if (D == 128) f(std::integral_constant<int, 128>());
    else f(std::integral_constant<int, 64>());
}

template <typename F>
__host__ __device__ __forceinline__ void with_bits(int bits, F f)
{
    if (bits == 1) f(std::integral_constant<int, 1>());
    else if (bits == 2) f(std::integral_constant<int, 2>());
    else if (bits == 3) f(std::integral_constant<int, 3>());
    else f(std::integral_constant<int, 4>());
}

}  // namespace kvmix
