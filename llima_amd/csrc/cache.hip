// cache.hip -- an 8-bit KV cache: keys and values quantised as they are written, and read
// back in 16 bits (gfx950).
//
//   per token and key head:  m = max(max |x|, 2^-100),  scale = m / 448,
//                            q = e4m3(448 x / m),  back: round(q scale)
//
// One scale for a head's D values: the attention over the cache multiplies a key's score
// and a value's weight by it once, and 4 bytes stand beside 64 to 256.
#include "attention.hpp"
#include "quant.hpp"

namespace llima {

struct CacheParams {
    const uint8_t *k, *v;                                    // written from (write); or null
    uint8_t *ok, *ov;                                        // read into (read); or null
    uint8_t *kq, *vq;                                        // the cache's values
    float *ksc, *vsc;                                        // and scales
    const int32_t *nodes, *counts, *lens, *table;            // nodes, counts, table: or null
    int32_t* new_lens;
    int64_t ks[4], vs[4];                                    // layer, batch, token and head strides (bytes; 16-bit side)
    int64_t kqs[4], vqs[4];                                  // layer, page, token and head strides (bytes)
    int64_t kss[4], vss[4];                                  // the same of the scales (elements)
    int64_t ns, ts, cap;
    int32_t B, N, L, Hkv;
    int32_t page, pages;
    uint32_t page_mul, page_shift, row_mul, row_shift;       // / page; / Hkv
    int32_t tok, chunks;                                     // tokens of a workgroup; workgroups of a sequence
};

// The maximum of non-negative floats' bits over N adjacent lanes, in all of them.
template <int N>
__device__ __forceinline__ uint32_t ca_max(uint32_t m) {
    m = q8_umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0xB1, 0xF, 0xF, false));   // lane ^ 1
    m = q8_umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x4E, 0xF, 0xF, false));   // lane ^ 2
    m = q8_umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x141, 0xF, 0xF, false));  // 7 - lane of 8
    if constexpr (N >= 16) m = q8_umax(m, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)m, 0x140, 0xF, 0xF, false));   // 15 - lane of 16
    if constexpr (N >= 32) {
        const auto s = __builtin_amdgcn_permlane16_swap(m, m, false, false);
        m = q8_umax(s[0], s[1]);
    }
    return m;
}

// The largest magnitude of 8 values, as bits of fp32.  16-bit floats without their sign are in
// the order of the numbers they are, NaN above infinity.
typedef uint16_t ca_h2 __attribute__((ext_vector_type(2)));
template <int DT> __device__ __forceinline__ uint32_t ca_top8(const llima_u32x4& q) {
    ca_h2 m = __builtin_bit_cast(ca_h2, q[0] & 0x7FFF7FFFu);
#pragma unroll
    for (int i = 1; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(ca_h2, q[i] & 0x7FFF7FFFu));
    return __float_as_uint(at_f32<DT>(m[0] > m[1] ? m[0] : m[1]));
}

// m / 448 rounded to nearest (as Q8Divisor's quotients).
__device__ __forceinline__ float ca_scale(float m) {
    constexpr float r = 1.0f / 448.0f;
    const float q = m * r;
    return m < __builtin_inff() ? __builtin_fmaf(__builtin_fmaf(-q, 448.0f, m), r, q) : q;
}

template <int DT> __device__ __forceinline__ void ca_load8(const llima_u32x4& q, float (&v)[8]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = at_f32<DT>((uint16_t)q[i]);
        v[2 * i + 1] = at_f32<DT>((uint16_t)(q[i] >> 16));
    }
}

// Every page of tokens [from, to) of sequence b in range (the same in all threads).  Each workgroup of a
// sequence looks at all of them.  In pages of 256 that costs nothing; reading 131072 tokens of 8 heads
// of 128 takes 164 us without a table, 190 in pages of 64, 241 in pages of 16 and 933 in pages of 1.
__device__ __forceinline__ bool ca_pages_ok(const CacheParams& P, int b, int from, int to) {
    bool ok = true;
    if (P.table && to > from) {                              // uniform
        const int e1 = (int)at_page(P.page_mul, P.page_shift, to - 1);
        for (int e = (int)at_page(P.page_mul, P.page_shift, from) + (int)threadIdx.x; e <= e1; e += LLIMA_WG) {
            const int p = P.table[b * P.ts + e];
            ok = ok && p >= 0 && p < P.pages;
        }
    }
    return ok;
}

// Token at of sequence b: its page and place in it.
__device__ __forceinline__ void ca_place(const CacheParams& P, int b, int at, uint32_t& p, uint32_t& o) {
    p = (uint32_t)b;
    o = (uint32_t)at;
    if (P.table) {                                           // uniform
        const uint32_t e = at_page(P.page_mul, P.page_shift, at);
        o = (uint32_t)at - e * (uint32_t)P.page;
        p = (uint32_t)P.table[b * P.ts + e];
    }
}

// i s.  W: strides past 32 bits (one multiplication instead of three where there are none: the
// addresses' products took as long as the rest of a row).
template <bool W> __device__ __forceinline__ int64_t ca_mul(uint32_t i, int64_t s) {
    if constexpr (W) return (int64_t)i * s;
    else return (int64_t)((uint64_t)i * (uint32_t)s);
}

// One workgroup per `tok` places of a sequence and layer; D / 8 lanes take a row of D values
// each: 16 bytes in, 8 out, the maximum over the row's lanes.  The first rows are requested
// before the sequence's whole path and room are checked (every workgroup of a sequence comes
// to the same answer, and nothing is written before it), keys and values together, so that
// half of them are still on their way while the others are computed.
// Bound: the inputs' bytes, two thirds of all, for prompts (8 of up to 4096 tokens, 81 MB moved: 20 us, the
// rate of a copy); an accepted path or a decoded token is latency (a node, a page, a row: 4.7 us).  Stores or loads that
// pass by L2 are slower here (20.8 -> 22.9 us).
template <int DT, int D, bool W>
__global__ __launch_bounds__(LLIMA_WG) void cache_write8(CacheParams P) {
    constexpr int U = D / 8, RW = LLIMA_WG / U, F = 4;       // lanes of a row; rows of a pass; passes in flight
    const int c = (int)(blockIdx.x % (uint32_t)P.chunks), b = (int)(blockIdx.x / (uint32_t)P.chunks), t = (int)threadIdx.x;
    const int64_t layer = blockIdx.y;
    const int len = P.lens[b], cnt = P.counts ? P.counts[b] : P.L;
    bool ok = len >= 0 && cnt >= 0 && cnt <= P.L && len <= P.cap && (int64_t)len + cnt <= P.cap;
    const int j0 = c * P.tok, j1 = j0 + P.tok < cnt ? j0 + P.tok : cnt;
    const int rows = j0 < cnt ? (j1 - j0) * P.Hkv : 0, u = t % U;   // (behind the count the product may pass 32 bits)
    llima_u32x4 y[2][F];
    uint32_t h[F], p[F], o[F];                               // head, page and place in it (a wait for a load behind
    auto load = [&](int i0) {                                // a store is one for the store, so these come first too)
#pragma unroll
        for (int f = 0; f < F; ++f) {                        // the last row again behind it
            const int i = i0 + f * RW < rows ? i0 + f * RW : rows - 1, e = (int)at_page(P.row_mul, P.row_shift, i), j = j0 + e;
            h[f] = (uint32_t)(i - e * P.Hkv);
            ca_place(P, b, len + j, p[f], o[f]);
            int node = j;
            if (P.nodes) {                                   // uniform
                node = P.nodes[b * P.ns + j];
                node = node >= 0 && node < P.N ? node : 0;   // (not written then)
            }
            y[0][f] = *(const llima_u32x4*)(P.k + layer * P.ks[0] + b * P.ks[1] + ca_mul<W>((uint32_t)node, P.ks[2]) + ca_mul<W>(h[f], P.ks[3]) + u * 16);
            y[1][f] = *(const llima_u32x4*)(P.v + layer * P.vs[0] + b * P.vs[1] + ca_mul<W>((uint32_t)node, P.vs[2]) + ca_mul<W>(h[f], P.vs[3]) + u * 16);
        }
    };
    if (ok && rows > 0) load(t / U);                         // uniform
    if (ok) {                                                // uniform
        bool all = ca_pages_ok(P, b, len, len + cnt);
        if (P.nodes)
            for (int i = t; i < cnt; i += LLIMA_WG) {
                const int node = P.nodes[b * P.ns + i];
                all = all && node >= 0 && node < P.N;
            }
        ok = __syncthreads_and(all);
    }
    if (c == 0 && layer == 0 && t == 0) P.new_lens[b] = ok ? len + cnt : LLIMA_E_RANGE;
    if (!ok || rows == 0) return;                            // uniform
    for (int i0 = t / U;;) {
#pragma unroll
        for (int f = 0; f < F; ++f) {
            auto put = [&](const llima_u32x4& x, uint8_t* q, const int64_t* qs, float* s, const int64_t* ss) __attribute__((always_inline)) {
                float v[8];
                ca_load8<DT>(x, v);
                const float mf = __uint_as_float(q8_umax(ca_max<U>(ca_top8<DT>(x)), __float_as_uint(Q8_TINY)));
                const uint2 z = q8_pack8(v, mf);
                if (i0 + f * RW < rows) {
                    *(uint2*)(q + layer * qs[0] + ca_mul<W>(p[f], qs[1]) + ca_mul<W>(o[f], qs[2]) + ca_mul<W>(h[f], qs[3]) + u * 8) = z;
                    if (u == 0) s[layer * ss[0] + ca_mul<W>(p[f], ss[1]) + ca_mul<W>(o[f], ss[2]) + ca_mul<W>(h[f], ss[3])] = ca_scale(mf);
                }
            };
            put(y[0][f], P.kq, P.kqs, P.ksc, P.kss);
            put(y[1][f], P.vq, P.vqs, P.vsc, P.vss);
        }
        i0 += RW * F;
        if (i0 - t / U >= rows) break;                       // uniform
        load(i0);
    }
}

// One workgroup per `tok` tokens of a sequence and layer, D / 8 lanes a row: 8 bytes in, 16
// out.  Rows past the sequence's length are 0; a sequence with a bad length or page is NaN.
// Bound, but for very small pages: the outputs' bytes, five sixths of all (16 sequences of up to 8192 tokens: 638 MB).  Stores
// that pass by L2 leave it to the reads: whole calls 128 -> 125 us, 5.1 TB/s.
template <int DT, int D, bool W>
__global__ __launch_bounds__(LLIMA_WG) void cache_read8(CacheParams P) {
    constexpr int U = D / 8, RW = LLIMA_WG / U, F = 4;
    const int c = (int)(blockIdx.x % (uint32_t)P.chunks), b = (int)(blockIdx.x / (uint32_t)P.chunks), t = (int)threadIdx.x;
    const int64_t layer = blockIdx.y;
    const int len = P.lens[b];
    bool ok = len >= 0 && len <= P.cap;
    if (ok) ok = __syncthreads_and(ca_pages_ok(P, b, 0, len));   // uniform
    const int j0 = c * P.tok, j1 = j0 + P.tok < P.L ? j0 + P.tok : P.L;
    const int rows = (j1 - j0) * P.Hkv, u = t % U;
    for (int i0 = t / U; i0 < rows; i0 += RW * F) {
        uint32_t h[F], p[F], o[F];
        int j[F];
#pragma unroll
        for (int f = 0; f < F; ++f) {                        // the last row again behind it
            const int i = i0 + f * RW < rows ? i0 + f * RW : rows - 1, e = (int)at_page(P.row_mul, P.row_shift, i);
            j[f] = j0 + e;
            h[f] = (uint32_t)(i - e * P.Hkv);
            p[f] = o[f] = 0;
            if (ok && j[f] < len) ca_place(P, b, j[f], p[f], o[f]);
        }
        uint2 x[2][F];
        float sc[2][F];
        auto load = [&](uint2 (&x)[F], float (&sc)[F], const uint8_t* q, const int64_t* qs, const float* s, const int64_t* ss) __attribute__((always_inline)) {
#pragma unroll
            for (int f = 0; f < F; ++f) {
                x[f] = make_uint2(0u, 0u);
                sc[f] = ok ? 0.0f : __builtin_nanf("");
                if (ok && j[f] < len) {
                    x[f] = *(const uint2*)(q + layer * qs[0] + ca_mul<W>(p[f], qs[1]) + ca_mul<W>(o[f], qs[2]) + ca_mul<W>(h[f], qs[3]) + u * 8);
                    sc[f] = s[layer * ss[0] + ca_mul<W>(p[f], ss[1]) + ca_mul<W>(o[f], ss[2]) + ca_mul<W>(h[f], ss[3])];
                }
            }
        };
        load(x[0], sc[0], P.kq, P.kqs, P.ksc, P.kss);
        load(x[1], sc[1], P.vq, P.vqs, P.vsc, P.vss);
        auto put = [&](const uint2 (&x)[F], const float (&sc)[F], uint8_t* y, const int64_t* ys) __attribute__((always_inline)) {
#pragma unroll
            for (int f = 0; f < F; ++f) {
                const uint32_t w[2] = {x[f].x, x[f].y};
                llima_u32x4 z;
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], false), d = __builtin_amdgcn_cvt_pk_f32_fp8((int)w[i], true);
                    z[2 * i] = at_pack<DT>(a[0] * sc[f], a[1] * sc[f]);
                    z[2 * i + 1] = at_pack<DT>(d[0] * sc[f], d[1] * sc[f]);
                }
                if (i0 + f * RW < rows)
                    __builtin_nontemporal_store(z, (llima_u32x4*)(y + layer * ys[0] + b * ys[1] + ca_mul<W>((uint32_t)j[f], ys[2]) +
                                                                  ca_mul<W>(h[f], ys[3]) + u * 16));
            }
        };
        put(x[0], sc[0], P.ok, P.ks);
        put(x[1], sc[1], P.ov, P.vs);
    }
}

// Tokens of a workgroup: up to 8 passes of its rows (its checks of the path and pages are the same for 1 and
// for 8), fewer where that would leave less than 2048 workgroups, a device's eight to a CU.
static void ca_plan(CacheParams& P, int layers, int D) {
    const int64_t rw = LLIMA_WG / (D / 8), rows = (int64_t)layers * P.B * P.L * 2 * P.Hkv;
    int64_t passes = rows / (rw * 2048);
    passes = passes < 1 ? 1 : passes > 8 ? 8 : passes;
    const int64_t tok = passes * rw / (2 * P.Hkv);
    P.tok = tok < 1 ? 1 : (int)tok;
    P.chunks = (P.L + P.tok - 1) / P.tok;
}

template <int DT, bool WRITE>
static int ca_launch(const CacheParams& P, int layers, int D, hipStream_t st) {
    if ((int64_t)P.B * P.chunks >= 1 << 24) return LLIMA_E_INVAL;   // (a launch: fewer than 2^32 threads)
    const dim3 g((uint32_t)(P.B * P.chunks), (uint32_t)layers), w(LLIMA_WG);
    bool wide = false;                                       // (the layers' and, of k and v, the batch's strides are the workgroup's)
    for (const int64_t* s : {P.ks, P.vs, P.kqs, P.vqs, P.kss, P.vss})
        for (int i = 1; i < 4; ++i) wide = wide || s[i] > (int64_t)UINT32_MAX;
    auto go = [&](auto d, auto w64) {
        constexpr int DD = decltype(d)::value;
        constexpr bool WW = decltype(w64)::value;
        if constexpr (WRITE) hipLaunchKernelGGL((cache_write8<DT, DD, WW>), g, w, 0, st, P);
        else hipLaunchKernelGGL((cache_read8<DT, DD, WW>), g, w, 0, st, P);
    };
    auto at = [&](auto d) { wide ? go(d, std::true_type{}) : go(d, std::false_type{}); };
    if (D == 64) at(std::integral_constant<int, 64>{});
    else if (D == 128) at(std::integral_constant<int, 128>{});
    else at(std::integral_constant<int, 256>{});
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}

// The arguments that writing and reading share: sizes, the cache and its strides.
template <class Args>
static int ca_fill(const Args* a, CacheParams& P) {
    if (!a || (a->dtype != LLIMA_BF16 && a->dtype != LLIMA_F16)) return LLIMA_E_INVAL;
    if (a->layers <= 0 || a->layers > 65535 || a->B < 0 || a->Hkv <= 0 || a->Hkv > 1024) return LLIMA_E_INVAL;
    if (a->D != 64 && a->D != 128 && a->D != 256) return LLIMA_E_INVAL;
    if (a->page_size <= 0 || a->pages < 0 || a->max_blocks < 0) return LLIMA_E_INVAL;
    if (!a->block_table && (a->pages < a->B || a->max_blocks != 1)) return LLIMA_E_INVAL;
    if ((int64_t)a->page_size * a->max_blocks > AT_KEYS) return LLIMA_E_INVAL;
    if (!at_strides_ok(a->k_strides, 4, 8) || !at_strides_ok(a->v_strides, 4, 8) || !at_strides_ok(a->k_cache_strides, 4, 16) ||
        !at_strides_ok(a->v_cache_strides, 4, 16) || !at_strides_ok(a->k_scale_strides, 4, 1) || !at_strides_ok(a->v_scale_strides, 4, 1))
        return LLIMA_E_INVAL;
    if (a->block_table && a->table_stride < 0) return LLIMA_E_INVAL;
    if (a->B == 0) return LLIMA_OK;
    const bool cached = a->pages > 0 && a->max_blocks > 0;
    if (!a->cache_lens || !a->k || !a->v) return LLIMA_E_INVAL;
    if (cached && (!a->k_cache || !a->v_cache || !a->k_scales || !a->v_scales)) return LLIMA_E_INVAL;
    const void* ptrs[] = {a->k, a->v, a->k_cache, a->v_cache};
    for (const void* p : ptrs)
        if ((uintptr_t)p % 16) return LLIMA_E_INVAL;
    if ((uintptr_t)a->k_scales % 4 || (uintptr_t)a->v_scales % 4) return LLIMA_E_INVAL;
    P.kq = (uint8_t*)a->k_cache; P.vq = (uint8_t*)a->v_cache;
    P.ksc = (float*)a->k_scales; P.vsc = (float*)a->v_scales;
    P.lens = a->cache_lens; P.table = a->block_table;
    for (int i = 0; i < 4; ++i) {
        P.ks[i] = 2 * a->k_strides[i]; P.vs[i] = 2 * a->v_strides[i];
        P.kqs[i] = a->k_cache_strides[i]; P.vqs[i] = a->v_cache_strides[i];
        P.kss[i] = a->k_scale_strides[i]; P.vss[i] = a->v_scale_strides[i];
    }
    P.ts = a->table_stride;
    P.cap = cached ? (int64_t)a->page_size * a->max_blocks : 0;
    P.B = a->B; P.Hkv = a->Hkv;
    P.page = a->page_size; P.pages = a->pages;
    at_divisor(P.page, P.page_mul, P.page_shift);
    at_divisor(P.Hkv, P.row_mul, P.row_shift);
    return LLIMA_OK;
}

}  // namespace llima

using namespace llima;

extern "C" int llima_cache_write_fp8(const llima_cache_write_fp8_args* a, void* stream) {
    CacheParams P = {};
    if (a && (a->N <= 0 || a->L <= 0 || a->L > AT_KEYS || (!a->nodes && a->L != a->N) || a->nodes_stride < 0)) return LLIMA_E_INVAL;
    const int ok = ca_fill(a, P);
    if (ok != LLIMA_OK || a->B == 0) return ok;
    if (!a->new_lens) return LLIMA_E_INVAL;
    P.k = (const uint8_t*)a->k; P.v = (const uint8_t*)a->v;
    P.nodes = a->nodes; P.counts = a->counts; P.new_lens = a->new_lens;
    P.ns = a->nodes_stride;
    P.N = a->N; P.L = a->L;
    ca_plan(P, a->layers, a->D);
    return a->dtype == LLIMA_BF16 ? ca_launch<LLIMA_BF16, true>(P, a->layers, a->D, (hipStream_t)stream)
                                  : ca_launch<LLIMA_F16, true>(P, a->layers, a->D, (hipStream_t)stream);
}

extern "C" int llima_cache_read_fp8(const llima_cache_read_fp8_args* a, void* stream) {
    CacheParams P = {};
    if (a && (a->L < 0 || a->L > AT_KEYS)) return LLIMA_E_INVAL;
    const int ok = ca_fill(a, P);
    if (ok != LLIMA_OK || a->B == 0 || a->L == 0) return ok;
    P.ok = (uint8_t*)a->k; P.ov = (uint8_t*)a->v;
    P.L = a->L;
    ca_plan(P, a->layers, a->D);
    return a->dtype == LLIMA_BF16 ? ca_launch<LLIMA_BF16, false>(P, a->layers, a->D, (hipStream_t)stream)
                                  : ca_launch<LLIMA_F16, false>(P, a->layers, a->D, (hipStream_t)stream);
}
