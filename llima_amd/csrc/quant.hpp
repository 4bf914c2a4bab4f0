// quant.hpp -- values in e4m3 with a scale: m = max(max |x|, 2^-100), scale = m / 448,
// q = e4m3(448 x / m), to nearest, ties to even (gfx950).
#pragma once

#include "common.hpp"

namespace llima {

#define Q8_TINY 7.8886090522101181e-31f                      // 2^-100

// The greatest of non-negative floats by their bits: NaN above infinity above every number.
__device__ __forceinline__ uint32_t q8_abs(float f) { return __float_as_uint(f) & 0x7FFFFFFFu; }
__device__ __forceinline__ uint32_t q8_umax(uint32_t a, uint32_t b) { return a > b ? a : b; }

// What the values of one maximum share: 448 x / m is taken as (0.875 c x) / (c m / 512), the
// same value with no overflow and no subnormal number on the way: c is 2^100 below m = 1.
struct Q8Divisor {
    float f, r, e;                                           // 0.875 c; 1 / d, d = c m / 512; d, or 0 when it is infinite
    __device__ __forceinline__ explicit Q8Divisor(float m) {
        const float c = m < 1.0f ? 1.2676506002282294e30f : 1.0f;
        const float d = m * (c * 0.001953125f);
        f = 0.875f * c;
        r = 1.0f / d;                                        // rounded to nearest: the quotient below is too
        e = d < __builtin_inff() ? d : 0.0f;
    }
    // f x / d rounded to nearest: the estimate's remainder is exact, and with r the nearest
    // to 1 / d one correction by it gives the nearest quotient (Markstein): next to the borders
    // between e4m3 values, for every divisor, no quotient differs from the division's.  The remainder is
    // taken with its sign turned, since that of a zero is then added as the opposite of the estimate's
    // sign and -0 stays -0.  An infinite m gives 0 of x's sign for a number and NaN for an infinity, a NaN m NaN.
    __device__ __forceinline__ float operator()(float x) const {
        const float n = x * f, q = n * r;
        return __builtin_fmaf(-__builtin_fmaf(q, e, -n), r, q);
    }
};

__device__ __forceinline__ uint2 q8_pack8(const float (&v)[8], float m) {
    const Q8Divisor div(m);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) q[i] = div(v[i]);
    int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
    lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
    int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
    hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
    return make_uint2((uint32_t)lo, (uint32_t)hi);
}

}  // namespace llima
