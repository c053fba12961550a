// The warp-level MMA of 16-bit operands and the two-part form of f32 operands (lora.cu, moe_w8.cu).
#pragma once
#include <type_traits>

#include "common.cuh"

namespace eq {

// c[16 x 8] += a[16 x 16] b[16 x 8].  Lane 4 g + j: a0 / a1 rows g / g + 8 at k = 2j, 2j + 1, a2 / a3 the same rows at k = 2j + 8, 2j + 9;
// b0 / b1 column g at those k; c rows g (c0, c1) and g + 8 (c2, c3), columns 2j, 2j + 1.
template <typename T>
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    if (std::is_same<T, __half>::value)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Value and remainder of v in 16 bits each: together 16 (bf16) or 22 (f16) bits of it.  A value that is not finite has no remainder.
template <typename T>
__device__ __forceinline__ void split16(float v, T& hi, T& lo) {
    hi = from_float<T>(v);
    const float back = to_float(hi);
    lo = from_float<T>(fabsf(back) <= 3.4028234e38f ? v - back : 0.f);
}

}  // namespace eq
