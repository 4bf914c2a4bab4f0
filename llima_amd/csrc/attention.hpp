// attention.hpp -- what the attention kernels over a 16-bit and over an 8-bit KV cache
// share: the partition of the keys into equal shares, the partial sums and their
// join, and the checks of the arguments (gfx950).
#pragma once

#include <type_traits>

#include "common.hpp"
#include "../../include/llima_sampler.h"

namespace llima {

struct AttnParams {
    const void *q, *k, *v, *kc, *vc;
    void* out;
    const int32_t* lens;                                     // [B]
    const void* mask;                                        // [B][N][N] or null (m <= n)
    const int32_t* table;                                    // [B][max_blocks] or null
    float* part_o;                                           // [slots][Hkv][R][D]
    float2* part_ml;                                         // [slots][Hkv][R]
    int64_t qs[3], ks[3], vs[3], os[3];                      // batch, token and head strides (elements)
    int64_t kcs[3], vcs[3];                                  // page, token and head strides
    int64_t ms[2];                                           // mask: batch and row strides
    int64_t ts;                                              // table row stride
    int64_t cap;                                             // tokens a sequence has room for
    int32_t mask_f32;
    int32_t B, N, Hq, Hkv, G, R;                             // R = N G rows of a key head
    int32_t page, pages;                                     // tokens of a page; pages of the cache
    uint32_t page_mul, page_shift;                           // j / page = j page_mul >> page_shift, j < 2^30
    int32_t slots, parts;                                    // partial sums per key head at most; shares of the keys
    int32_t pairs;                                           // partial sums stand two to a share (at_slot)
    int32_t RG, RT;                                          // row groups, row tiles of a group
    float scale2;                                            // |scale| log2(e)
    int32_t flip;                                            // scale < 0
    int32_t mode;                                            // AT_TILE, AT_REQUEST or AT_LANE
};

#define AT_KEYS (1 << 30)              // keys of a sequence at most
#define AT_TILE 0
#define AT_REQUEST 1
#define AT_LANE 2

__device__ __forceinline__ uint32_t at_page(uint32_t mul, uint32_t shift, int j) {
    return (uint32_t)(((uint64_t)(uint32_t)j * mul) >> shift);
}

// The kernel's arguments, loaded anew where they are used: held in registers
// from the start, those of the parts that run seldom push out the others.
typedef const __attribute__((address_space(4))) AttnParams* AttnArgs;
__device__ __forceinline__ AttnArgs at_args() {
    AttnArgs a = (AttnArgs)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(a));
    return a;
}

__device__ __forceinline__ uint64_t readfirstlane64(uint64_t v) {
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
           (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)v);
}

typedef float at_acc __attribute__((ext_vector_type(16)));
typedef short at_s4 __attribute__((ext_vector_type(4)));
typedef short at_s8 __attribute__((ext_vector_type(8)));

template <int DT> __device__ __forceinline__ at_acc at_mfma(at_s8 a, at_s8 b, at_acc c) {
    if constexpr (DT == LLIMA_BF16) {
        typedef __bf16 t8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(t8, a), __builtin_bit_cast(t8, b), c, 0, 0, 0);
    } else {
        typedef _Float16 t8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(t8, a), __builtin_bit_cast(t8, b), c, 0, 0, 0);
    }
}

// Two fp32 rounded to the type (to nearest, ties to even).
template <int DT> __device__ __forceinline__ uint32_t at_pack(float a, float b) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 v = {a, b};
    if constexpr (DT == LLIMA_BF16) {
        typedef __bf16 t2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, t2));
    } else {
        typedef _Float16 t2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, t2));
    }
}

template <int DT> __device__ __forceinline__ float at_f32(uint16_t h) {
    if constexpr (DT == LLIMA_BF16) return __uint_as_float((uint32_t)h << 16);
    else return (float)__builtin_bit_cast(_Float16, h);
}

// Exponent all ones: an infinity or NaN of the type.
template <int DT> __device__ __forceinline__ bool at_special(uint16_t h) {
    constexpr uint32_t e = DT == LLIMA_BF16 ? 0x7F80u : 0x7C00u;
    return (h & e) == e;
}

// Sequence b's cached length; a length outside [0, cap] is 0 and bad.
__device__ __forceinline__ int at_len(const AttnParams& P, int b, bool& bad) {
    const int l = P.lens[b];
    bad = l < 0 || l > P.cap;
    return bad ? 0 : l;
}

// The partition of the keys: each sequence's are tiles of T, all sequences'
// tiles stand in a row, and P.parts workgroups (per key head and row group)
// take equal shares of it.  A share may hold parts of several sequences (at_slot:
// where a part leaves its sums).
// KeyTiles::count: a sequence's tiles; at_share: the length of a share (every lane of
// a wave calls it and gets the same).  len0: the length of sequence lane.
// A sequence counts for AT_EXTRA tiles more than it has, at its end: the time that
// its mask, its sums' exchange and the next sequence's start take (3 / 6 / 8: 24 ragged
// sequences of up to 16384 tokens, 16 nodes, 151 / 140 / 140 us; 48 of up to 3000, one
// node, 75 / 67 / 62; 100 of up to 500 49 / 52 / 59).
#define AT_EXTRA 6
template <int T>
struct KeyTiles {
    static constexpr int EXTRA = AT_EXTRA;
    static __device__ __forceinline__ int count(const AttnParams& P, int len) { return (len + P.N + T - 1) / T + AT_EXTRA; }
};

template <class TL>
__device__ __forceinline__ int64_t at_share(const AttnParams& P, int len0) {
    const int lane = (int)lane_id();
    if (P.B == 1)                                            // uniform; a step of one stream waits for this
        return ((uint32_t)__builtin_amdgcn_readfirstlane(TL::count(P, len0)) + (uint32_t)P.parts - 1u) / (uint32_t)P.parts;
    int64_t total = lane < P.B ? TL::count(P, len0) : 0;
    for (int b = 64 + lane; b < P.B; b += 64) {
        bool bad;
        total += TL::count(P, at_len(P, b, bad));
    }
    return ((int64_t)wave_sum_u64((uint64_t)total) + P.parts - 1) / P.parts;
}

// The slot of the partial sums that share x has of sequence b (begins: from the
// sequence's first tile on).  Slot x + b is one that no other pair has; with more
// sequences than shares, two slots to a share: its first sequence may come from the
// share before, its last may go on in the next, and the others it has whole.
__device__ __forceinline__ int at_slot(int pairs, int x, int b, bool begins) {
    return pairs ? 2 * x + (begins ? 1 : 0) : x + b;
}

// The sequence that has tile `at` of the row, its length, and its first tile's
// place in the row; false past the last tile.
template <class TL>
__device__ __forceinline__ bool at_find(const AttnParams& P, int64_t at, int len0, int& b, int& len,
                                        int64_t& first) {
    const int lane = (int)lane_id();
    if (P.B == 1) {                                          // uniform
        b = 0;
        len = __builtin_amdgcn_readfirstlane(len0);
        first = 0;
        return at < TL::count(P, len);
    }
    int64_t before = 0;
    for (int b0 = 0; b0 < P.B; b0 += 64) {
        bool bad;
        const bool in = b0 + lane < P.B;
        const int ln = !in ? 0 : b0 ? at_len(P, b0 + lane, bad) : len0;
        const uint32_t n = in ? (uint32_t)TL::count(P, ln) : 0u;   // 64 times 2^25 + 70 at most
        const uint32_t incl = wave_incl_scan_u32(n);
        const uint64_t past = ballot(in && before + incl > at);
        if (past) {
            const int l = __builtin_ctzll(past);
            b = b0 + l;
            first = before + readlane(incl - n, l);
            len = (int)readlane((uint32_t)ln, l);
            return true;
        }
        before += readlane63(incl);
    }
    return false;
}

// One over the sum l of a row's weights.  The largest weight is 1 (2^10 in fp16), so a sum of 0
// is a row that sees nothing, which is 0, or one whose visible scores are all minus
// infinity, which is NaN.
template <class Params>
__device__ __forceinline__ float at_inverse(const Params* P, float l, int b, int n, int len) {
    if (l != 0.0f) return 1.0f / l;
    bool sees = len > 0 || !P->mask;
    for (int m = 0; m < P->N && !sees; ++m) {
        const int64_t at = b * P->ms[0] + n * P->ms[1] + m;
        sees = P->mask_f32 ? ((const float*)P->mask)[at] > 0.0f : ((const uint8_t*)P->mask)[at] != 0;
    }
    return sees ? __builtin_nanf("") : 0.0f;
}

__device__ __forceinline__ void at_dma(const void* src, uint8_t* dst) {
    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                     (__attribute__((address_space(3))) void*)dst, 16, 0, 0);
}

// Joins the parts of each row (a sequence's node and query head), WPR waves a
// row, which take every WPR-th part each in rounds of 8 loads.  Four waves up to 1024 rows,
// one where they fill the device (the call, 16 nodes over 8192 tokens, four / one: 512 rows
// 26.8 / 29.0 us, 1024 30.3 / 31.5, 2048 40.6 / 38.6, 4096 76.4 / 70.3, 12288 203 / 179).
template <int DT, int D, class TL, int WPR>
__global__ __launch_bounds__(LLIMA_WG) void tree_attn_join(AttnParams P) {
    constexpr int E = D / 64;                                // values per lane
    static_assert(WPR == 1 || WPR == LLIMA_WAVES, "one row or four to a workgroup");
    __shared__ float so[WPR][D], sl[WPR];
    const int lane = (int)lane_id(), sub = (int)wave_id() % WPR;
    const int w = (int)(blockIdx.x * (LLIMA_WAVES / WPR) + wave_id() / WPR);
    if (w >= P.B * P.N * P.Hq) return;                       // (WPR = 1)
    const int b = w / (P.N * P.Hq), n = w / P.Hq % P.N, hq = w % P.Hq;
    bool bad;
    const int len0 = lane < P.B ? at_len(P, lane, bad) : 0;
    const int64_t share = at_share<TL>(P, len0);
    int64_t first = 0;                                       // the sequence's first tile
    if (b > 0) {                                             // uniform
        first = lane < b ? TL::count(P, len0) : 0;
        for (int i = 64 + lane; i < b; i += 64) first += TL::count(P, at_len(P, i, bad));
        first = (int64_t)wave_sum_u64((uint64_t)first);
    }
    const int len = b < 64 ? (int)readlane((uint32_t)len0, (uint32_t)b) : at_len(P, b, bad);
    const int64_t last = first + TL::count(P, len) - 1 - TL::EXTRA;
    const int x0 = (int)(first / share), np = (int)(last / share) - x0 + 1;
    if (np <= 1) return;                                     // the same for a row's waves
    const int h = hq / P.G, row = n * P.G + hq % P.G;
    const size_t slot = (size_t)P.Hkv * P.R, step = P.pairs ? 2 * slot : slot;
    const size_t at1 = (size_t)at_slot(P.pairs, x0 + 1, b, false) * slot + (size_t)h * P.R + row;
    const size_t at0 = (size_t)at_slot(P.pairs, x0, b, true) * slot + (size_t)h * P.R + row;
    auto place = [&](int c) { return c == 0 ? at0 : at1 + (size_t)(c - 1) * step; };
    float m = -__builtin_inff(), l = 0.0f, o[E];
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] = 0.0f;
    // the greatest maximum first (a lane per part), then one pass of weighted sums
    for (int c = lane; c < np; c += 64) m = __builtin_fmaxf(m, P.part_ml[place(c)].x);
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) m = __builtin_fmaxf(m, __shfl_xor(m, x, 64));
    const float mu = m > -__builtin_inff() ? m : 0.0f;
    for (int c0 = sub; c0 < np; c0 += 8 * WPR) {
        float2 ml[8];
        float po[8][E];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int c = c0 + i * WPR;
            const size_t at = place(c < np ? c : c0);
            ml[i] = P.part_ml[at];
#pragma unroll
            for (int e = 0; e < E; ++e) po[i][e] = P.part_o[at * D + lane * E + e];
        }
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            if (c0 + i * WPR < np) {                         // uniform
                const float a = __builtin_amdgcn_exp2f(ml[i].x - mu);
                l += ml[i].y * a;
#pragma unroll
                for (int e = 0; e < E; ++e) o[e] += po[i][e] * a;
            }
        }
    }
    if constexpr (WPR > 1) {
#pragma unroll
        for (int e = 0; e < E; ++e) so[sub][lane * E + e] = o[e];
        if (lane == 0) sl[sub] = l;
        __syncthreads();
        if (sub != 0) return;
        l = (sl[0] + sl[1]) + (sl[2] + sl[3]);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int d = lane * E + e;
            o[e] = (so[0][d] + so[1][d]) + (so[2][d] + so[3][d]);
        }
    }
    const float inv = at_inverse(&P, l, b, n, len);
#pragma unroll
    for (int e = 0; e < E; ++e) o[e] *= inv;
    uint16_t* op = (uint16_t*)P.out + b * P.os[0] + n * P.os[1] + hq * P.os[2] + lane * E;
    if constexpr (E == 1) op[0] = (uint16_t)at_pack<DT>(o[0], 0.0f);
#pragma unroll
    for (int e = 0; e + 1 < E; e += 2) *(uint32_t*)(op + e) = at_pack<DT>(o[e], o[e + 1]);
}

static inline bool at_sizes_ok(int32_t B, int32_t N, int32_t Hq, int32_t Hkv, int32_t D) {
    if (B < 0 || N <= 0 || N > 1024 || Hq <= 0 || Hkv <= 0 || Hq % Hkv != 0 || Hq > 1024) return false;
    if (D != 64 && D != 128 && D != 256) return false;
    return (int64_t)B * N * Hq < (1 << 26);                  // (the join's launch: fewer than 2^32 threads)
}

// Strides are multiples of `align` elements (16 bytes), so every row is aligned as
// its base pointer is.
static inline bool at_strides_ok(const int64_t* s, int n, int align) {
    for (int i = 0; i < n; ++i)
        if (s[i] < 0 || s[i] % align != 0) return false;
    return true;
}

// j / d = j mul >> shift for j < 2^30.  l = ceil(log2 d): mul = ceil(2^(30 + l) / d) <=
// 2^31 + 1 exceeds the quotient by less than d / 2^(30 + l) <= 2^-30 of j.
static inline void at_divisor(int32_t d, uint32_t& mul, uint32_t& shift) {
    uint32_t l = 0;
    while ((1ll << l) < d) ++l;
    mul = (uint32_t)(((1ull << (30 + l)) + d - 1) / (uint64_t)d);
    shift = 30 + l;
}

// The partial sums' slots of a plan, their bytes, and their places in the workspace.
static inline void at_slots(AttnParams& P) {
    P.pairs = P.parts < P.B;
    P.slots = P.pairs ? 2 * P.parts : P.parts + P.B;
}

static inline size_t at_parts_bytes(const AttnParams& P, int D) {
    const size_t rows = (size_t)P.slots * P.Hkv * P.R;
    return (rows * D * sizeof(float) + 255) / 256 * 256 + rows * sizeof(float2);
}

static inline void at_parts_at(AttnParams& P, int D, void* workspace) {
    const size_t rows = (size_t)P.slots * P.Hkv * P.R;
    P.part_o = (float*)workspace;
    P.part_ml = (float2*)((uint8_t*)workspace + (rows * D * sizeof(float) + 255) / 256 * 256);
}

// Checks the arguments and takes them over; cache strides are multiples of `align`
// elements (16 bytes).
static inline int at_fill(const llima_tree_attention_args* a, int align, AttnParams& P) {
    if (!a || !at_sizes_ok(a->B, a->N, a->Hq, a->Hkv, a->D)) return LLIMA_E_INVAL;
    if (a->dtype != LLIMA_BF16 && a->dtype != LLIMA_F16) return LLIMA_E_INVAL;
    if (!(a->scale == a->scale) || __builtin_isinf(a->scale)) return LLIMA_E_INVAL;
    if (a->page_size <= 0 || a->pages < 0 || a->max_blocks < 0) return LLIMA_E_INVAL;
    if (!a->block_table && (a->pages < a->B || a->max_blocks != 1)) return LLIMA_E_INVAL;
    if ((int64_t)a->page_size * a->max_blocks + a->N > AT_KEYS) return LLIMA_E_INVAL;
    if (a->mask_dtype != LLIMA_MASK_U8 && a->mask_dtype != LLIMA_MASK_F32) return LLIMA_E_INVAL;
    if (!at_strides_ok(a->q_strides, 3, 8) || !at_strides_ok(a->k_strides, 3, 8) || !at_strides_ok(a->v_strides, 3, 8) ||
        !at_strides_ok(a->out_strides, 3, 8) || !at_strides_ok(a->k_cache_strides, 3, align) ||
        !at_strides_ok(a->v_cache_strides, 3, align))
        return LLIMA_E_INVAL;
    if (a->mask && (a->mask_strides[0] < 0 || a->mask_strides[1] < 0)) return LLIMA_E_INVAL;
    if (a->block_table && a->table_stride < 0) return LLIMA_E_INVAL;
    if (a->B == 0) return LLIMA_OK;
    const bool cached = a->pages > 0 && a->max_blocks > 0;   // else no sequence may have a cached token
    if (!a->q || !a->k || !a->v || !a->out || !a->cache_lens || (cached && (!a->k_cache || !a->v_cache)))
        return LLIMA_E_INVAL;
    const void* ptrs[] = {a->q, a->k, a->v, a->out, a->k_cache, a->v_cache};
    for (const void* p : ptrs)
        if ((uintptr_t)p % 16) return LLIMA_E_INVAL;
    P.q = a->q; P.k = a->k; P.v = a->v; P.kc = a->k_cache; P.vc = a->v_cache; P.out = a->out;
    P.lens = a->cache_lens; P.mask = a->mask; P.table = a->block_table;
    for (int i = 0; i < 3; ++i) {
        P.qs[i] = a->q_strides[i]; P.ks[i] = a->k_strides[i]; P.vs[i] = a->v_strides[i];
        P.os[i] = a->out_strides[i]; P.kcs[i] = a->k_cache_strides[i]; P.vcs[i] = a->v_cache_strides[i];
    }
    P.ms[0] = a->mask_strides[0]; P.ms[1] = a->mask_strides[1];
    P.ts = a->table_stride;
    P.cap = cached ? (int64_t)a->page_size * a->max_blocks : 0;
    P.mask_f32 = a->mask_dtype == LLIMA_MASK_F32;
    P.B = a->B; P.N = a->N; P.Hq = a->Hq; P.Hkv = a->Hkv; P.G = a->Hq / a->Hkv;
    P.page = a->page_size; P.pages = a->pages;
    at_divisor(P.page, P.page_mul, P.page_shift);
    P.scale2 = __builtin_fabsf(a->scale) * 1.44269504088896340736f;
    P.flip = a->scale < 0.0f;
    return LLIMA_OK;
}

}  // namespace llima
