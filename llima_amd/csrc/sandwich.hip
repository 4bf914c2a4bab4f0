// sandwich.hip -- the norms on both sides of the residual stream: a block's output is
// normalised, gated and added to the scaled stream, and the stream normalised for the next
// block, in one pass (gfx950).
//
//   p = (x f1) (post + offset)                  (x itself without post)
//   r = round(rs residual + (p gate) gs)        (p gs without gate)
//   y = (r f2) (pre + offset),  rounded or in 8 bits with a scale per block of 128
//   f = fp32(1 / sqrt(mean of squares + eps)), the mean in 64 bits
//
// Every product and sum is one fp32 operation in this order, as in rms_rows: the outputs do
// not depend on how a row is spread over lanes.
//
// Bound: reading x, the residual and a gate per token once, writing r and y once.  8000 rows of
// 5760 in bf16: 369 MB in 71 us, 5.2 TB/s, what a copy reaches.  16 rows of 4096 into 8 bits:
// 4.9 us, one wait for memory and two exchanges of sums.
// One workgroup per row, since a row's factor needs all of it and it fits the registers.  Outputs
// that pass by L2 too are slower (69 -> 72 us), and the next operator reads them.
#include "norm.hpp"
#include "quant.hpp"

namespace llima {

struct SandwichParams {
    const void *x, *residual, *gate, *post, *pre;            // gate, post: or null
    void* out;
    float* scales;                                           // [B][ceil(H / 128)] (8-bit output)
    void* out_residual;
    int64_t x_stride, res_stride, gate_stride;               // elements between rows (gate: 0 for one row)
    int32_t B, H, NK;
    float eps, offset, rs, gs;
};

// A piece that nobody reads again: it passes by L2 (8000 x 5760 bf16, whole calls: 71.7 -> 70.8 us).
template <class Raw> __device__ __forceinline__ Raw sw_once(const void* p) {
    Raw r;
#pragma unroll
    for (int i = 0; i < (int)(sizeof(Raw) / 16); ++i)
        ((llima_u32x4*)&r)[i] = __builtin_nontemporal_load((const llima_u32x4*)p + i);
    return r;
}

// 1 / sqrt of the mean of the squares whose sums the threads hold, rounded once to fp32.
template <int NWV>
__device__ __forceinline__ float sw_factor(double s, double* part, int H, float eps) {
#pragma unroll
    for (int o = 32; o >= 1; o >>= 1) s += __shfl_xor(s, o, 64);
    const int t = (int)threadIdx.x;
    if ((t & 63) == 0) part[t >> 6] = s;
    __syncthreads();
    s = part[0];
#pragma unroll
    for (int w = 1; w < NWV; ++w) s += part[w];
    return (float)(1.0 / __builtin_sqrt(s / (double)H + (double)eps));
}

// One workgroup of 64 NWV threads per row; thread t holds the pieces of 8 values t + 64 NWV j,
// j < NP, from the first read to the last write.  Everything that the row needs is requested
// before the first sum, so that a row waits for memory once and for two exchanges.  With NP = 0
// (rows past 16384 values) the inputs are read twice, and r where the thread wrote it.
template <int DT, int NWV, int NP, bool Q8>
__global__ __launch_bounds__(64 * NWV) void sandwich_rows(SandwichParams P) {
    using T = NormType<DT>;
    constexpr int NT = 64 * NWV, NA = NP > 0 ? NP : 1;
    __shared__ double part[2][NWV];
    const int t = (int)threadIdx.x, b = (int)blockIdx.x, np = P.H / 8;
    const uint8_t* x = (const uint8_t*)P.x + (int64_t)b * P.x_stride * T::E;
    const uint8_t* res = (const uint8_t*)P.residual + (int64_t)b * P.res_stride * T::E;
    const uint8_t* gate = (const uint8_t*)P.gate + (int64_t)b * P.gate_stride * T::E;
    uint8_t* rout = (uint8_t*)P.out_residual + (size_t)b * P.H * T::E;
    auto at = [](const void* base, int p) { return (const uint8_t*)base + (size_t)p * 8 * T::E; };
    // r of a piece from its x, in place
    auto stream = [&](float (&v)[8], float f, const float (&w)[8], const float (&g)[8], const float (&a)[8]) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (P.post) v[i] = v[i] * f * (w[i] + P.offset); // uniform
            if (P.gate) v[i] = v[i] * g[i];                  // uniform
            v[i] = T::round(a[i] * P.rs + v[i] * P.gs);
        }
    };
    auto put = [&](int p, float (&v)[8], float f, const float (&w)[8]) {
        const bool in = p < np;
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = v[i] * f * (w[i] + P.offset);
        if constexpr (Q8) {
            uint32_t m = 0;
            if (in) {
#pragma unroll
                for (int i = 0; i < 8; ++i) m = q8_umax(m, q8_abs(v[i]));
            }
#pragma unroll
            for (int o = 8; o >= 1; o >>= 1) m = q8_umax(m, (uint32_t)__shfl_xor((int)m, o, 64));
            const float mf = __uint_as_float(q8_umax(m, __float_as_uint(Q8_TINY)));
            if (in) {
                *(uint2*)((uint8_t*)P.out + (size_t)b * P.H + (size_t)p * 8) = q8_pack8(v, mf);
                if ((p & 15) == 0) P.scales[(size_t)b * P.NK + p / 16] = mf / 448.0f;
            }
        } else {
            if (in) T::store((uint8_t*)P.out + ((size_t)b * P.H + (size_t)p * 8) * T::E, v);
        }
    };
    auto squares = [](const float (&v)[8], double s) {
#pragma unroll
        for (int i = 0; i < 8; ++i) s = __builtin_fma((double)v[i], (double)v[i], s);
        return s;
    };
    double s = 0.0;
    float f = 1.0f;
    if constexpr (NP > 0) {
        typename T::Raw rx[NA], ra[NA], rg[NA] = {}, r1[NA] = {}, r2[NA];
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            const int p = t + NT * j < np ? t + NT * j : np - 1;
            rx[j] = sw_once<typename T::Raw>(at(x, p));
            ra[j] = sw_once<typename T::Raw>(at(res, p));
            if (P.post) r1[j] = *(const typename T::Raw*)at(P.post, p);   // uniform
            if (P.gate) rg[j] = *(const typename T::Raw*)at(gate, p);     // uniform
            r2[j] = *(const typename T::Raw*)at(P.pre, p);
        }
        float v[NA][8];
#pragma unroll
        for (int j = 0; j < NP; ++j) T::open(rx[j], v[j]);
        if (P.post) {                                        // uniform
#pragma unroll
            for (int j = 0; j < NP; ++j)
                if (t + NT * j < np) s = squares(v[j], s);
            f = sw_factor<NWV>(s, part[0], P.H, P.eps);
        }
        s = 0.0;
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            float w[8], g[8], a[8];
            T::open(r1[j], w);
            T::open(rg[j], g);
            T::open(ra[j], a);
            stream(v[j], f, w, g, a);
            if (t + NT * j < np) {
                T::store(rout + (size_t)(t + NT * j) * 8 * T::E, v[j]);
                s = squares(v[j], s);
            }
        }
        f = sw_factor<NWV>(s, part[1], P.H, P.eps);
#pragma unroll
        for (int j = 0; j < NP; ++j) {
            float w[8];
            T::open(r2[j], w);
            put(t + NT * j, v[j], f, w);
        }
    } else {
        if (P.post) {                                        // uniform
            for (int p = t; p < np; p += NT) {
                float v[8];
                T::load(at(x, p), v);
                s = squares(v, s);
            }
            f = sw_factor<NWV>(s, part[0], P.H, P.eps);
        }
        s = 0.0;
        for (int p = t; p < np; p += NT) {
            float v[8], w[8] = {}, g[8] = {}, a[8];
            T::load(at(x, p), v);
            T::load(at(res, p), a);
            if (P.post) T::load(at(P.post, p), w);
            if (P.gate) T::load(at(gate, p), g);
            stream(v, f, w, g, a);
            T::store(rout + (size_t)p * 8 * T::E, v);
            s = squares(v, s);
        }
        f = sw_factor<NWV>(s, part[1], P.H, P.eps);
        for (int p0 = 0; p0 < np; p0 += NT) {                // whole waves: the block maximum takes all lanes
            const int p = p0 + t < np ? p0 + t : np - 1;
            float v[8] = {}, w[8];
            if (p0 + t < np) T::load(rout + (size_t)p * 8 * T::E, v);
            T::load(at(P.pre, p), w);
            put(p0 + t, v, f, w);
        }
    }
}

template <int DT, bool Q8>
static void sw_launch_np(const SandwichParams& P, hipStream_t st) {
    const dim3 g((uint32_t)P.B);                             // B <= NRM_ROWS
    const int np = P.H / 8;
    if (np <= 256) hipLaunchKernelGGL((sandwich_rows<DT, 4, 1, Q8>), g, dim3(256), 0, st, P);
    else if (np <= 512) hipLaunchKernelGGL((sandwich_rows<DT, 4, 2, Q8>), g, dim3(256), 0, st, P);
    else if (np <= 768) hipLaunchKernelGGL((sandwich_rows<DT, 4, 3, Q8>), g, dim3(256), 0, st, P);
    else if (np <= 1024) hipLaunchKernelGGL((sandwich_rows<DT, 4, 4, Q8>), g, dim3(256), 0, st, P);
    else if (np <= 2048) hipLaunchKernelGGL((sandwich_rows<DT, 16, 2, Q8>), g, dim3(1024), 0, st, P);
    else hipLaunchKernelGGL((sandwich_rows<DT, 16, 0, Q8>), g, dim3(1024), 0, st, P);
}

template <int DT, bool Q8>
static int sw_launch(const SandwichParams& P, hipStream_t st) {
    const size_t e = NormType<DT>::E, row = (size_t)P.H * e;
    for (int64_t b0 = 0; b0 < P.B; b0 += NRM_ROWS / 4) {     // (1024 threads a row)
        SandwichParams Q = P;
        Q.B = P.B - b0 < NRM_ROWS / 4 ? (int)(P.B - b0) : NRM_ROWS / 4;
        Q.x = (const uint8_t*)P.x + b0 * P.x_stride * (int64_t)e;
        Q.residual = (const uint8_t*)P.residual + b0 * P.res_stride * (int64_t)e;
        if (P.gate) Q.gate = (const uint8_t*)P.gate + b0 * P.gate_stride * (int64_t)e;
        Q.out_residual = (uint8_t*)P.out_residual + b0 * row;
        Q.out = (uint8_t*)P.out + b0 * (Q8 ? (size_t)P.H : row);
        if (Q8) Q.scales = P.scales + b0 * P.NK;
        sw_launch_np<DT, Q8>(Q, st);
    }
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}

}  // namespace llima

using namespace llima;

extern "C" int llima_sandwich_norm(const llima_sandwich_norm_args* a, void* stream) {
    if (!a) return LLIMA_E_INVAL;
    int ok = nrm_check(a->x, a->dtype, a->B, a->H, a->x_stride);
    if (ok == LLIMA_OK) ok = nrm_check(a->residual, a->dtype, a->B, a->H, a->residual_stride);
    if (ok == LLIMA_OK && a->gate) ok = nrm_check(a->gate, a->dtype, a->gate_stride ? a->B : a->B < 1 ? a->B : 1, a->H, a->gate_stride);
    if (ok != LLIMA_OK) return ok;
    const float f[] = {a->eps, a->weight_offset, a->residual_scale, a->gate_scale};
    for (float v : f)
        if (!(v == v) || __builtin_isinf(v)) return LLIMA_E_INVAL;
    if (a->eps < 0.0f) return LLIMA_E_INVAL;
    if (a->B == 0) return LLIMA_OK;
    if (!a->pre_weight || !a->out || !a->out_residual) return LLIMA_E_INVAL;
    if (!nrm_aligned(a->post_weight) || !nrm_aligned(a->pre_weight) || !nrm_aligned(a->out) || !nrm_aligned(a->out_residual))
        return LLIMA_E_INVAL;
    SandwichParams P = {};
    P.x = a->x; P.residual = a->residual; P.gate = a->gate; P.post = a->post_weight; P.pre = a->pre_weight;
    P.out = a->out; P.scales = a->out_scales; P.out_residual = a->out_residual;
    P.x_stride = a->x_stride; P.res_stride = a->residual_stride; P.gate_stride = a->gate ? a->gate_stride : 0;
    P.B = a->B; P.H = a->H; P.NK = (a->H + NRM_BLK - 1) / NRM_BLK;
    P.eps = a->eps; P.offset = a->weight_offset; P.rs = a->residual_scale; P.gs = a->gate_scale;
    hipStream_t st = (hipStream_t)stream;
    const bool q8 = P.scales != nullptr;
    if (a->dtype == LLIMA_BF16) return q8 ? sw_launch<LLIMA_BF16, true>(P, st) : sw_launch<LLIMA_BF16, false>(P, st);
    if (a->dtype == LLIMA_F16) return q8 ? sw_launch<LLIMA_F16, true>(P, st) : sw_launch<LLIMA_F16, false>(P, st);
    return q8 ? sw_launch<LLIMA_F32, true>(P, st) : sw_launch<LLIMA_F32, false>(P, st);
}
