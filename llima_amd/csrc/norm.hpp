// norm.hpp -- pieces of 8 values of a row in bf16, fp16 or fp32, and the checks of rows
// that the norm kernels share (gfx950).
#pragma once

#include <hip/hip_fp16.h>

#include "common.hpp"
#include "../../include/llima_sampler.h"

namespace llima {

#define NRM_BLK 128

// 8 values of a row as fp32 (16 bytes of a 16-bit type, 32 of fp32), and back
// rounded to nearest, ties to even.
template <int DT> struct NormType;
template <> struct NormType<LLIMA_BF16> {
    static constexpr int E = 2;
    typedef llima_u32x4 Raw;
    static __device__ __forceinline__ void open(const Raw& q, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            v[2 * i] = __uint_as_float(q[i] << 16);
            v[2 * i + 1] = __uint_as_float(q[i] & 0xFFFF0000u);
        }
    }
    static __device__ __forceinline__ void load(const void* p, float (&v)[8]) { open(*(const Raw*)p, v); }
    static __device__ __forceinline__ void store(void* p, const float (&v)[8]) {
        typedef float f2 __attribute__((ext_vector_type(2)));
        typedef __bf16 h2 __attribute__((ext_vector_type(2)));
        llima_u32x4 q;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f2 a = {v[2 * i], v[2 * i + 1]};
            q[i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(a, h2));
        }
        *(llima_u32x4*)p = q;
    }
    static __device__ __forceinline__ float round(float f) { return (float)(__bf16)f; }
};
template <> struct NormType<LLIMA_F16> {
    static constexpr int E = 2;
    typedef _Float16 Raw __attribute__((ext_vector_type(8)));
    static __device__ __forceinline__ void open(const Raw& q, float (&v)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = (float)q[i];
    }
    static __device__ __forceinline__ void load(const void* p, float (&v)[8]) { open(*(const Raw*)p, v); }
    static __device__ __forceinline__ void store(void* p, const float (&v)[8]) {
        typedef _Float16 h8 __attribute__((ext_vector_type(8)));
        h8 q;
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = (_Float16)v[i];
        *(h8*)p = q;
    }
    static __device__ __forceinline__ float round(float f) { return (float)(_Float16)f; }
};
template <> struct NormType<LLIMA_F32> {
    static constexpr int E = 4;
    struct Raw { float4 a, b; };
    static __device__ __forceinline__ void open(const Raw& q, float (&v)[8]) {
        const float4 a = q.a, b = q.b;
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    static __device__ __forceinline__ void load(const void* p, float (&v)[8]) { open(*(const Raw*)p, v); }
    static __device__ __forceinline__ void store(void* p, const float (&v)[8]) {
        ((float4*)p)[0] = make_float4(v[0], v[1], v[2], v[3]);
        ((float4*)p)[1] = make_float4(v[4], v[5], v[6], v[7]);
    }
    static __device__ __forceinline__ float round(float f) { return f; }
};

// A launch holds fewer than 2^32 threads.
#define NRM_ROWS (1 << 23)

static inline bool nrm_aligned(const void* p) { return (uintptr_t)p % 16 == 0; }

static inline int nrm_check(const void* x, int32_t dtype, int32_t B, int32_t H, int64_t stride) {
    if (dtype != LLIMA_BF16 && dtype != LLIMA_F16 && dtype != LLIMA_F32) return LLIMA_E_INVAL;
    if (B < 0 || H <= 0 || H % 8 != 0 || H > 65536) return LLIMA_E_INVAL;
    const int64_t e = dtype == LLIMA_F32 ? 4 : 2;
    if (B > 0 && (!x || !nrm_aligned(x) || stride * e % 16 != 0 || (B > 1 && stride < H))) return LLIMA_E_INVAL;
    return LLIMA_OK;
}

}  // namespace llima
