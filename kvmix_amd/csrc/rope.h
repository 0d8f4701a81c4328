// The rotary embedding of one value with fp16 tables, as the fp16 tensor expression x * cos + rotate_half(x) * sin rounds it.
#pragma once

#include "kvmix_common.h"

namespace kvmix {

// The products are pinned in registers as fp16 bit patterns before they are added: left to itself
// the compiler contracts fp16 product + sum into one mixed-precision fma, and the product's rounding
// to fp16 -- which the tensor expression has -- is lost.
__device__ __forceinline__ float rounded_product(float a, float b)
{
    uint32_t bits = f32_to_h16(a * b);
    asm volatile("" : "+v"(bits));
    return h16_to_f32((uint16_t)bits);
}

__device__ __forceinline__ uint16_t rope_one(uint16_t x, uint16_t other, uint16_t c, uint16_t s, bool negate_other)
{
    const float a = rounded_product(h16_to_f32(x), h16_to_f32(c));
    const float o = negate_other ? -h16_to_f32(other) : h16_to_f32(other);
    const float b = rounded_product(o, h16_to_f32(s));
    return f32_to_h16(a + b);
}

}  // namespace kvmix
