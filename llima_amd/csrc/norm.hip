// norm.hip -- root-mean-square norm with the residual's addition, and rows and
// LM head weights as 8-bit values with a scale per block of 128 (gfx950).
//
//   r = round(x + residual)                     (x itself without a residual)
//   y = (r * f) * (w + offset),  f = fp32(1 / sqrt(mean(r^2) + eps))
//   out = round(y), or per block of 128 values of a row
//         m = max(max |y|, 2^-100),  scale = m / 448,  q = e4m3(448 y / m)
//
// The mean is summed in 64 bits and f rounded once from it, y is three fp32
// products, and 448 y / m one product and the IEEE division's quotient (as
// Q8Divisor takes it: 8192 x 5760 bf16 rows 31 -> 25 us): every step is a
// defined operation, so the outputs do not depend on how a row is spread over
// lanes (a sum of 16-bit squares is exact in 64 bits but for the last place),
// and a tie of the 8-bit rounding stays one.  Rounding to 8 bits is what the
// caller asks for: relative 2^-4 of a value, 2^-10 of its block's maximum at
// most below the normal range.  A block holding a NaN or an infinity has that
// as its scale (and NaN where an infinity stood, 0 where a number did, or NaN
// throughout for a NaN).
#include "norm.hpp"
#include "quant.hpp"

namespace llima {

struct NormParams {
    const void* x;
    const void* residual;                                    // or null
    const void* weight;                                      // null: no norm (quantize only)
    void* out;
    float* scales;                                           // [B][ceil(H / 128)] (8-bit output)
    void* out_residual;                                      // or null
    int64_t x_stride, res_stride;                            // elements between rows
    int32_t B, H, NK;
    float eps, offset;
};

// One workgroup of 64 NWV threads per row; thread t holds the pieces of 8
// values t + 64 NWV j, j < NP, of the row in registers between the two passes
// over them (the sum, the output).  16 lanes hold a block of 128.
// With NP = 0 (rows past 8192 values) the row is read again in the second pass.
//
// Bound: reading x and the residual and writing both results once (8000 x 5760
// bf16: 369 MB in 73 us, 5.0 TB/s; a large copy 5.1).  The sum's 64-bit products are
// hidden under that.  16 x 4096 to 8 bits: 4.6 us, launch and latency.
template <int DT, int NWV, int NP, bool Q8, bool NORM>
__global__ __launch_bounds__(64 * NWV) void rms_rows(NormParams P) {
    using T = NormType<DT>;
    constexpr int NT = 64 * NWV;
    __shared__ double part[NWV];
    const int t = (int)threadIdx.x, b = (int)blockIdx.x, np = P.H / 8;
    const uint8_t* x = (const uint8_t*)P.x + (int64_t)b * P.x_stride * T::E;
    const uint8_t* res = P.residual ? (const uint8_t*)P.residual + (int64_t)b * P.res_stride * T::E : nullptr;
    uint8_t* rout = P.out_residual ? (uint8_t*)P.out_residual + (size_t)b * P.H * T::E : nullptr;
    auto fetch = [&](int p, float (&v)[8]) {                 // r of piece p, p < np
        T::load(x + (size_t)p * 8 * T::E, v);
        if (res) {
            float a[8];
            T::load(res + (size_t)p * 8 * T::E, a);
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = T::round(v[i] + a[i]);
        }
    };
    float v[NP > 0 ? NP : 1][8];
    double s = 0.0;
    if constexpr (NP > 0) {
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int p = t + NT * j;
            if (p < np) {
                fetch(p, v[j]);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) v[j][i] = 0.0f;
            }
        }
    }
    float f = 1.0f;
    if constexpr (NORM) {
        if constexpr (NP > 0) {
#pragma unroll
            for (int j = 0; j < NP; ++j)
#pragma unroll
                for (int i = 0; i < 8; ++i) s = __builtin_fma((double)v[j][i], (double)v[j][i], s);
        } else {
            for (int p = t; p < np; p += NT) {
                float w[8];
                fetch(p, w);
#pragma unroll
                for (int i = 0; i < 8; ++i) s = __builtin_fma((double)w[i], (double)w[i], s);
            }
        }
#pragma unroll
        for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
        if constexpr (NWV > 1) {
            if ((t & 63) == 0) part[t >> 6] = s;
            __syncthreads();
            s = part[0];
#pragma unroll
            for (int w = 1; w < NWV; ++w) s += part[w];
        }
        f = (float)(1.0 / __builtin_sqrt(s / (double)P.H + (double)P.eps));
    }
    auto put = [&](int p, float (&w)[8]) {
        const bool in = p < np;
        if (rout && in) T::store(rout + (size_t)p * 8 * T::E, w);
        if constexpr (NORM) {
            float g[8];
            T::load((const uint8_t*)P.weight + (size_t)(in ? p : 0) * 8 * T::E, g);
#pragma unroll
            for (int i = 0; i < 8; ++i) w[i] = w[i] * f * (g[i] + P.offset);
        }
        if constexpr (Q8) {
            uint32_t m = 0;
            if (in) {
#pragma unroll
                for (int i = 0; i < 8; ++i) m = q8_umax(m, q8_abs(w[i]));
            }
#pragma unroll
            for (int o = 8; o >= 1; o >>= 1) m = q8_umax(m, (uint32_t)__shfl_xor((int)m, o, 64));
            m = q8_umax(m, __float_as_uint(Q8_TINY));
            const float mf = __uint_as_float(m);
            if (in) {
                *(uint2*)((uint8_t*)P.out + (size_t)b * P.H + (size_t)p * 8) = q8_pack8(w, mf);
                if ((p & 15) == 0) P.scales[(size_t)b * P.NK + p / 16] = mf / 448.0f;
            }
        } else {
            if (in) T::store((uint8_t*)P.out + ((size_t)b * P.H + (size_t)p * 8) * T::E, w);
        }
    };
    if constexpr (NP > 0) {
#pragma unroll
        for (int j = 0; j < NP; ++j) put(t + NT * j, v[j]);
    } else {
        for (int p0 = 0; p0 < np; p0 += NT) {                // whole waves: the block maximum takes all lanes
            const int p = p0 + t;
            float w[8] = {0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f, 0.0f};
            if (p < np) fetch(p, w);
            put(p, w);
        }
    }
}

// One workgroup per block of 128 x 128 of an LM head weight [V][H] bf16: its
// maximum, scale and e4m3 values.  Thread t holds the pieces of 8 columns
// t % 16 of rows t / 16 + 16 j.
__global__ __launch_bounds__(LLIMA_WG) void fp8_blocks(const uint16_t* w, uint8_t* out, float* scales,
                                                       int V, int H, int NK) {
    __shared__ uint32_t part[LLIMA_WAVES];
    const int t = (int)threadIdx.x, kb = (int)blockIdx.x, vb = (int)blockIdx.y;
    const int h = kb * NRM_BLK + (t & 15) * 8, r0 = vb * NRM_BLK + (t >> 4);
    float v[8][8];
    uint32_t m = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int n = r0 + 16 * j;
        if (n < V && h < H) {                                // H % 8 == 0: a piece is inside or outside
            NormType<LLIMA_BF16>::load(w + (size_t)n * H + h, v[j]);
#pragma unroll
            for (int i = 0; i < 8; ++i) m = q8_umax(m, q8_abs(v[j][i]));
        }
    }
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) m = q8_umax(m, (uint32_t)__shfl_xor((int)m, o, 64));
    if ((t & 63) == 0) part[t >> 6] = m;
    __syncthreads();
    m = q8_umax(q8_umax(part[0], part[1]), q8_umax(part[2], part[3]));
    m = q8_umax(m, __float_as_uint(Q8_TINY));
    const float mf = __uint_as_float(m);
    if (t == 0) scales[(size_t)vb * NK + kb] = mf / 448.0f;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const int n = r0 + 16 * j;
        if (n < V && h < H) *(uint2*)(out + (size_t)n * H + h) = q8_pack8(v[j], mf);
    }
}

template <int DT, int NWV, bool Q8, bool NORM>
static void nrm_launch_np(const NormParams& P, hipStream_t st) {
    const int np = (P.H / 8 + 64 * NWV - 1) / (64 * NWV);
    const dim3 g((uint32_t)P.B), blk(64 * NWV);              // B <= NRM_ROWS
    switch (np) {
        case 1: hipLaunchKernelGGL((rms_rows<DT, NWV, 1, Q8, NORM>), g, blk, 0, st, P); break;
        case 2: hipLaunchKernelGGL((rms_rows<DT, NWV, 2, Q8, NORM>), g, blk, 0, st, P); break;
        case 3: hipLaunchKernelGGL((rms_rows<DT, NWV, 3, Q8, NORM>), g, blk, 0, st, P); break;
        case 4: hipLaunchKernelGGL((rms_rows<DT, NWV, 4, Q8, NORM>), g, blk, 0, st, P); break;
        default: hipLaunchKernelGGL((rms_rows<DT, NWV, 0, Q8, NORM>), g, blk, 0, st, P); break;
    }
}

template <int DT, bool Q8, bool NORM>
static int nrm_launch(const NormParams& P, hipStream_t st) {
    const size_t e = NormType<DT>::E, row = (size_t)P.H * e;
    for (int64_t b0 = 0; b0 < P.B; b0 += NRM_ROWS) {
        NormParams Q = P;
        Q.B = P.B - b0 < NRM_ROWS ? (int)(P.B - b0) : NRM_ROWS;
        Q.x = (const uint8_t*)P.x + b0 * P.x_stride * (int64_t)e;
        if (P.residual) Q.residual = (const uint8_t*)P.residual + b0 * P.res_stride * (int64_t)e;
        if (P.out_residual) Q.out_residual = (uint8_t*)P.out_residual + b0 * row;
        Q.out = (uint8_t*)P.out + b0 * (Q8 ? (size_t)P.H : row);
        if (Q8) Q.scales = P.scales + b0 * P.NK;
        nrm_launch_np<DT, 4, Q8, NORM>(Q, st);
    }
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}

template <bool Q8, bool NORM>
static int nrm_dispatch(const NormParams& P, int32_t dtype, hipStream_t st) {
    if (dtype == LLIMA_BF16) return nrm_launch<LLIMA_BF16, Q8, NORM>(P, st);
    if (dtype == LLIMA_F16) return nrm_launch<LLIMA_F16, Q8, NORM>(P, st);
    return nrm_launch<LLIMA_F32, Q8, NORM>(P, st);
}

}  // namespace llima

using namespace llima;

extern "C" int llima_add_rms_norm(const void* x, const void* residual, const void* weight,
                                  int32_t dtype, int32_t B, int32_t H, int64_t x_stride,
                                  int64_t residual_stride, float eps, float weight_offset,
                                  void* out, float* out_scales, void* out_residual, void* stream) {
    int st0 = nrm_check(x, dtype, B, H, x_stride);
    if (st0 != LLIMA_OK) return st0;
    if (!(eps >= 0.0f) || __builtin_isinf(eps) || !(weight_offset == weight_offset) || __builtin_isinf(weight_offset))
        return LLIMA_E_INVAL;
    if (residual && (st0 = nrm_check(residual, dtype, B, H, residual_stride)) != LLIMA_OK) return st0;
    if (out_residual && !residual) return LLIMA_E_INVAL;
    if (B > 0 && (!weight || !out || !nrm_aligned(weight) || !nrm_aligned(out) || !nrm_aligned(out_residual)))
        return LLIMA_E_INVAL;
    if (B == 0) return LLIMA_OK;
    NormParams P = {};
    P.x = x; P.residual = residual; P.weight = weight; P.out = out;
    P.scales = out_scales; P.out_residual = out_residual;
    P.x_stride = x_stride; P.res_stride = residual_stride;
    P.B = B; P.H = H; P.NK = (H + NRM_BLK - 1) / NRM_BLK;
    P.eps = eps; P.offset = weight_offset;
    return out_scales ? nrm_dispatch<true, true>(P, dtype, (hipStream_t)stream)
                      : nrm_dispatch<false, true>(P, dtype, (hipStream_t)stream);
}

extern "C" int llima_quantize_rows(const void* x, int32_t dtype, int32_t B, int32_t H,
                                   int64_t x_stride, void* out, float* out_scales, void* stream) {
    const int st0 = nrm_check(x, dtype, B, H, x_stride);
    if (st0 != LLIMA_OK) return st0;
    if (B > 0 && (!out || !out_scales || !nrm_aligned(out))) return LLIMA_E_INVAL;
    if (B == 0) return LLIMA_OK;
    NormParams P = {};
    P.x = x; P.out = out; P.scales = out_scales;
    P.x_stride = x_stride;
    P.B = B; P.H = H; P.NK = (H + NRM_BLK - 1) / NRM_BLK;
    return nrm_dispatch<true, false>(P, dtype, (hipStream_t)stream);
}

extern "C" int llima_lm_head_quantize(const void* weight, int32_t V, int32_t H, void* out,
                                      float* out_scales, void* stream) {
    if (V <= 0 || H <= 0 || H % 64 != 0 || H > 65536) return LLIMA_E_INVAL;
    if (!weight || !out || !out_scales || !nrm_aligned(weight) || !nrm_aligned(out)) return LLIMA_E_INVAL;
    const int NK = (H + NRM_BLK - 1) / NRM_BLK, NVB = (V + NRM_BLK - 1) / NRM_BLK;
    // 65535 rows of workgroups at most in a launch
    for (int v0 = 0; v0 < NVB; v0 += 65535) {
        const int n = NVB - v0 < 65535 ? NVB - v0 : 65535;
        const size_t r0 = (size_t)v0 * NRM_BLK;
        hipLaunchKernelGGL(fp8_blocks, dim3((uint32_t)NK, (uint32_t)n), dim3(LLIMA_WG), 0, (hipStream_t)stream,
                           (const uint16_t*)weight + r0 * H, (uint8_t*)out + r0 * H, out_scales + (size_t)v0 * NK,
                           (int)(V - (int64_t)r0), H, NK);
    }
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}
