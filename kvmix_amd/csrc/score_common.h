// What the kernels over rows of logits share: values in pieces of sixteen bytes, and the order of the most likely tokens.
#pragma once

#include "kvmix_common.h"

namespace kvmix {

typedef uint32_t uint4v __attribute__((ext_vector_type(4)));

constexpr int kTopMost = 64, kCandidates = 1024;
constexpr float kLog2e = 1.44269504088896340736f, kLn2 = 0.693147180559945309417f;

template <typename T>
__device__ __forceinline__ float to_float(T v)
{
    return (float)v;
}

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
    for (int j = 1; j < (int)(16 / sizeof(T)); j++) most = fmaxf(most, to_float(w.t[j]));
    return most;
}

// order of the most likely: larger value first, then lower index; NaN is larger than anything
__device__ __forceinline__ uint32_t value_key(float v)
{
    const uint32_t b = __float_as_uint(v + 0.0f);  // (-0 is 0)
    return v != v ? 0xffffffffu : b & 0x80000000u ? ~b : b | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }

__device__ __forceinline__ uint64_t full_key(float v, int index) { return (uint64_t)value_key(v) << 32 | (uint32_t)~index; }

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

template <typename F>
inline void with_type(int dtype, F f)
{
    if (dtype == KVMIX_F16) f((_Float16)0);
    else if (dtype == KVMIX_F32) f(0.0f);
    else f((__bf16)0.0f);
}

}  // namespace kvmix
