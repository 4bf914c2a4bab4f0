// attention_fp8.hip -- attention of drafted tokens (or of one new token) over an 8-bit KV
// cache under a tree mask (gfx950).
//
//   out[b][n][h] = sum_j p_j v_j,  p = softmax over the visible j of scale q . k_j
//   cached tokens:  k_j = kq_j ks_j,  v_j = vq_j vs_j  (e4m3 values, a scale per token and head)
//
// One pass over the keys with the running maximum and sum of the softmax (fp32, base 2).
// bf16 and fp16 hold every e4m3 value, so the values go into the 16-bit matrix cores by a
// conversion without rounding; a key's scale multiplies its score, a value's scale its
// weight, both in fp32.  The products are taken transposed in tiles of 16 rows:
// S^T = K Q^T leaves 4 keys of a query row in a lane (lane l: row l % 16, keys 4 (l / 16)
// + 0 .. 3), which are at once the operand of O^T = V^T P^T; V's transposing loads fetch the
// keys in that order.
//
// The waves of a workgroup share no tile: each takes its own keys for all rows (up to 64) of
// its row group, so that a value is read from memory, from LDS and converted once, and no
// wave waits for another before the end of a sequence's part, where their sums are joined.
//
// For the product with V a weight times its value's scale is rounded to fp16 whatever q's type
// (11 bits; in bf16 the outputs' error against 64 bits was 0.0023 of their size with weights in bf16, now
// 0.0017, that of the output's own rounding).  What a row's scores are taken less goes by these products, not
// by the weights: it moves only when one would pass 2^15, and then so far that the row's greatest is 2^7 (the
// sums are rescaled seldom, and a score's product with its key's scale and the difference are one
// operation).  So a product is rounded by its own size down to 2^-21 of its row's greatest, whatever the scales
// of keys that weigh nothing there, and by 2^-32 of the greatest below.  The weights alone, which
// are summed, run from 2^-120 to 2^100.  A lane's greatest score and greatest scale tell that nothing moves; the
// logarithms of single scales are taken only where they do not.
// The drafted tokens' values are of q's type, and so are their weights.
//
// Bound: up to one row tile (16 rows per key head) reading the cache's D + 4 bytes per key and
// value once.  64 sequences of one token, 755 MB: 117-126 us, 6.0-6.4 TB/s (requests into LDS alone
// reach 5.6 TB/s, 6.2 where they pass by L2).  From three row tiles on the issue: a tile of 32 keys takes
// a wave 340 vector operations with 48 matrix ones and 64 that widen K and V among them, and 129 scalar ones
// (33 nodes of 4 heads over 4 x 131072 tokens, 1.1 GB: 440-453 us; the vector units busy 67 % of the time, the
// matrix cores 35 %; requests alone 287).  16 nodes over 24 x up to 16384: 72 us, the memory's 50.  Short calls
// are a chain of latencies (1 x 1000 tokens: 8.7 us and 4.1 of the join).
//
// Why four waves with tiles of their own: waves that share a tile convert it once each or pass it on
// through LDS.  Eight waves for three and more row tiles: 118 -> 131 us (16 nodes, 24 x 8192); tiles of
// 16 keys and three workgroups per CU: 142 -> 172 us (64 sequences of one token).
#include "attention.hpp"

namespace llima {

struct At8Params : AttnParams {
    const float *ksc, *vsc;
    int64_t kss[3], vss[3];                                  // scales: page, token and head strides (elements)
    uint32_t g_mul, g_shift;                                 // row / G
};

// The arguments, loaded anew where they are used (at_args).
typedef const __attribute__((address_space(4))) At8Params* At8Args;
__device__ __forceinline__ At8Args a8_args() { return (At8Args)at_args(); }

template <int D> struct A8 {
    static constexpr int NW = 4;                             // waves
    static constexpr int KT = D == 256 ? 16 : 32;            // cached keys of a wave's tile
    static constexpr int DK = KT / 2;                        // drafted keys of one (16-bit values: the same bytes)
    static constexpr int S = D == 64 ? 3 : 2;                // stages of a wave's ring
    static constexpr int ST = 2 * KT * D + 256;              // bytes of a stage: K, V, their scales
    static constexpr int T = NW * KT, TD = NW * DK;          // keys of a tile of the workgroup
    static constexpr int MAXM = D == 256 ? 2 : 4;            // row tiles of 16 of a workgroup at most
    static constexpr int QL = D == 256 ? 1 : D == 128 ? 3 : 4;   // of them in LDS at most (two workgroups per CU), the rest in registers
};

#define A8_MOST 15.0f                                        // the logarithm of a row's greatest weight times scale, base 2
#define A8_HEAD 8.0f                                         // where it is passed, the row's maximum comes this much below it
#define A8_UNIT 8                                            // scales enter times 2^8 (that of the greatest bf16 value is 2^119)
#define A8_LEAST -85.0f                                      // and count as 2^-93 at least, so that weights without them stay below 2^100

// The partition's unit: tiles of T cached keys, then tiles of TD drafted ones.
template <int D>
struct Fp8Tiles {
    static constexpr int EXTRA = 4;                          // tiles that a sequence's start and end take the time of (6: 2 to 8 % longer; 2 and 9: longer)
    static __device__ __forceinline__ int cached(int len) { return (int)((uint32_t)(len + A8<D>::T - 1) / (uint32_t)A8<D>::T); }
    static __device__ __forceinline__ int drafted(int N) { return (int)((uint32_t)(N + A8<D>::TD - 1) / (uint32_t)A8<D>::TD); }
    static __device__ __forceinline__ int count(const AttnParams& P, int len) { return cached(len) + drafted(P.N) + EXTRA; }
};

typedef float a8_acc __attribute__((ext_vector_type(4)));
typedef int a8_i2 __attribute__((ext_vector_type(2)));

// 16 x 16 += 16 x 32 * 32 x 16, and 16 x 16 * 16 x 16.
template <int DT> __device__ __forceinline__ a8_acc a8_mfma(at_s8 a, at_s8 b, a8_acc c) {
    if constexpr (DT == LLIMA_BF16) {
        typedef __bf16 t8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(t8, a), __builtin_bit_cast(t8, b), c, 0, 0, 0);
    } else {
        typedef _Float16 t8 __attribute__((ext_vector_type(8)));
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(t8, a), __builtin_bit_cast(t8, b), c, 0, 0, 0);
    }
}
template <int DT> __device__ __forceinline__ a8_acc a8_mfma(at_s4 a, at_s4 b, a8_acc c) {
    if constexpr (DT == LLIMA_BF16) return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, b, c, 0, 0, 0);
    else {
        typedef _Float16 t4 __attribute__((ext_vector_type(4)));
        return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(t4, a), __builtin_bit_cast(t4, b), c, 0, 0, 0);
    }
}

// 8 e4m3 values as 16-bit ones, exactly.
template <int DT> __device__ __forceinline__ at_s8 a8_wide(uint32_t lo, uint32_t hi) {
    llima_u32x4 w;
    if constexpr (DT == LLIMA_BF16) {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true));
    } else {
        w[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, false));
        w[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(lo, 1.0f, true));
        w[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, false));
        w[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(hi, 1.0f, true));
    }
    return __builtin_bit_cast(at_s8, w);
}

// The greatest of three; NaN is left out.  (As builtins, every operand is
// canonicalised first.)  Its operands are results of ordinary operations, never a matrix
// instruction's own, and a swap of lanes takes its result only after a copy of it.
__device__ __forceinline__ float a8_max(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

__device__ __forceinline__ float a8_max_abs(float a, float b, float c) {
    float d;
    asm("v_max3_f32 %0, |%1|, |%2|, |%3|" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

// The maximum, or the sum, over the four lanes of a query row (l, l ^ 16, l ^ 32, l ^ 48).
__device__ __forceinline__ float a8_max4(float x) {
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = a8_max(__uint_as_float(s[0]), __uint_as_float(s[1]), __uint_as_float(s[1]));
    s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return a8_max(__uint_as_float(s[0]), __uint_as_float(s[1]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float a8_sum4(float x) {
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(s[0]) + __uint_as_float(s[1]);
    s = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// 4 or 8 pieces of V by the transposing loads, from a[i] on, in one piece with their wait (as builtins, the
// compiler waits for all the requests into LDS before them).
__device__ __forceinline__ void a8_tr8(const uint32_t (&a)[4], a8_i2 (&v)[4]) {
    asm volatile("ds_read_b64_tr_b8 %0, %4\n\tds_read_b64_tr_b8 %1, %5\n\tds_read_b64_tr_b8 %2, %6\n\tds_read_b64_tr_b8 %3, %7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]) : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]) : "memory");
}
__device__ __forceinline__ void a8_tr8(const uint32_t (&a)[8], a8_i2 (&v)[8]) {
    asm volatile("ds_read_b64_tr_b8 %0, %8\n\tds_read_b64_tr_b8 %1, %9\n\tds_read_b64_tr_b8 %2, %10\n\tds_read_b64_tr_b8 %3, %11\n\t"
                 "ds_read_b64_tr_b8 %4, %12\n\tds_read_b64_tr_b8 %5, %13\n\tds_read_b64_tr_b8 %6, %14\n\tds_read_b64_tr_b8 %7, %15\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]), "=&v"(v[4]), "=&v"(v[5]), "=&v"(v[6]), "=&v"(v[7])
                 : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "v"(a[4]), "v"(a[5]), "v"(a[6]), "v"(a[7]) : "memory");
}
__device__ __forceinline__ void a8_tr16(const uint32_t (&a)[4], at_s4 (&v)[4]) {
    asm volatile("ds_read_b64_tr_b16 %0, %4\n\tds_read_b64_tr_b16 %1, %5\n\tds_read_b64_tr_b16 %2, %6\n\tds_read_b64_tr_b16 %3, %7\n\t"
                 "s_waitcnt lgkmcnt(0)"
                 : "=&v"(v[0]), "=&v"(v[1]), "=&v"(v[2]), "=&v"(v[3]) : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]) : "memory");
}

template <int N> __device__ __forceinline__ void a8_wait() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// Rows of D bytes (cached) or 2 D bytes (drafted) in LDS: 16-byte unit u of key k stands at unit
// u ^ swz(k), so that 16 or 32 keys' same unit lie in different banks (256 bytes).
template <int ROW> __device__ __forceinline__ uint32_t a8_swz(uint32_t key) {
    return (ROW < 256 ? key / (256 / ROW) : key) & (ROW / 16 - 1) & 15;
}

// One workgroup: four waves over one share of the keys, one key head and M row tiles of 16.
// A wave's cached tile lies in one page (contiguous caches, pages of a multiple of its keys):
// its address comes from the scalar unit; or each 1 KB request of it does (AT_REQUEST), or
// every lane computes its own (AT_LANE).  KIND: A8_ONE and A8_MANY for the first mode and one or
// several row groups, A8_GEN for the last two.
#define A8_ONE 0
#define A8_MANY 1
#define A8_GEN 2
template <int DT, int D, int M, int KIND>
__global__ __launch_bounds__((64 * A8<D>::NW), 2) void tree_attn8(At8Params P) {
#ifdef __HIP_DEVICE_COMPILE__                               // (the host pass drops the launch stub over the descriptors)
    using C = A8<D>;
    constexpr bool GEN = KIND == A8_GEN;
    constexpr int NW = C::NW, KT = C::KT, DK = C::DK, S = C::S, ST = C::ST, T = C::T, TD = C::TD;
    constexpr int NB = KT / 16;                              // blocks of 16 keys
    constexpr int U = D / 16, U2 = D / 8;                    // 16-byte units of a cached and of a drafted row
    constexpr int KQ = 64 / U, NQ = KT / KQ;                 // keys of a 1 KB request, requests of K or V
    constexpr int KQ2 = U2 < 64 ? 64 / U2 : 1;
    constexpr int QL = M < C::QL ? M : C::QL, QR = M - QL;
    constexpr int NR = 2 * NQ + 2;                           // requests of a cached tile
    constexpr int DB = D / 16;                               // column blocks
    constexpr int VG = DB < 8 ? DB : 8;                      // of them read from LDS at a time
    constexpr bool AHEAD = M * D <= 384;                     // Q's pieces are read a step before their products (registers: else with it)
    constexpr int QT = 16 * 2 * D;                           // bytes of a row tile of Q
    constexpr int RING = NW * S * ST, XB = NW * DB * 1024;   // a row tile's sums of all waves
    constexpr int XN = 2 * XB + NW * M * 128 <= RING ? 2 : 1;
    static_assert(XB + NW * M * 128 <= RING, "room for the waves' sums");
    static_assert(DK * 2 * D == KT * D && NQ * 1024 == KT * D, "tiles are whole requests");
    __shared__ __align__(1024) uint8_t sm[RING + QL * QT + 16];
    uint8_t* const sq = sm + RING;
    uint32_t* const flag = (uint32_t*)(sq + QL * QT);        // a bad page or length; special values
    const int t = (int)threadIdx.x, lane = t & 63, r = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    // workgroups go to the 8 XCDs in turn: the row groups of a share and head on one of them, side by side, so
    // that its keys come from memory once and from that XCD's L2 for the other groups (requests of three row
    // groups alone over 4 x 131072 tokens: 513 -> 287 us)
    const uint32_t turn = blockIdx.x / 8u, pair = turn / (uint32_t)P.RG * 8u + blockIdx.x % 8u;
    const int rg = (int)(turn % (uint32_t)P.RG), part = (int)(pair / (uint32_t)P.Hkv), h = (int)(pair % (uint32_t)P.Hkv);
    if (part >= P.parts) return;                             // (the grid is a multiple of 8)
    uint8_t* const ring = sm + wave * (S * ST);
    bool bad = false;
    const int len0 = lane < P.B ? at_len(P, lane, bad) : 0;
    const int64_t share = (int64_t)readfirstlane64((uint64_t)at_share<Fp8Tiles<D>>(P, len0));
    const int64_t end = (part + 1) * share;
    const int nd = Fp8Tiles<D>::drafted(P.N);
    for (int64_t from = part * share; from < end;) {         // the share's sequences
    int b, len;
    int64_t first;
    if (!at_find<Fp8Tiles<D>>(P, from, len0, b, len, first)) return;   // uniform: past the last tile
    b = __builtin_amdgcn_readfirstlane(b);
    len = __builtin_amdgcn_readfirstlane(len);
    first = (int64_t)readfirstlane64((uint64_t)first);
    const int nc = Fp8Tiles<D>::cached(len), nt = nc + nd;
    const int64_t last = first + nt + Fp8Tiles<D>::EXTRA, upto = last < end ? last : end;
    const int c0 = __builtin_amdgcn_readfirstlane((int)(from - first));
    const int c1 = __builtin_amdgcn_readfirstlane(upto - first < nt ? (int)(upto - first) : nt);
    const bool whole = from == first && upto >= last - Fp8Tiles<D>::EXTRA;   // the sequence has no other part
    from = upto;
    if (c0 >= nt) continue;                                  // uniform: nothing of it but the extra tiles
    // the wave's tiles: cached ones c0 .., then drafted ones d0 ..
    const int cend = c1 < nc ? c1 : nc;
    int nC = cend > c0 ? cend - c0 : 0;
    if (nC > 0 && (cend - 1) * T + wave * KT >= len) --nC;
    const int d0 = (c0 > nc ? c0 : nc) - nc, dend = c1 - nc;
    int nD = dend > d0 ? dend - d0 : 0;
    if (nD > 0 && (dend - 1) * TD + wave * DK >= P.N) --nD;
    nC = __builtin_amdgcn_readfirstlane(nC);
    const int ntile = nC + __builtin_amdgcn_readfirstlane(nD);
    __syncthreads();                                         // (the sequence before is done with LDS)
    if (t == 0) {
        bool wrong;
        at_len(P, b, wrong);
        flag[0] = wrong ? 1u : 0u;
        flag[1] = 0u;
    }
    auto key_of = [&](int tile) { return (c0 + tile) * T + wave * KT; };         // a cached tile's first key
    auto draft_of = [&](int tile) { return (d0 + tile - nC) * TD + wave * DK; };   // a drafted tile's first token
    // ---------------------------------------------------------------- requests
    bool miss = false;                                       // a page of this sequence that does not exist
    auto page_of = [&](int j) {                              // the page of key j (uniform), by the scalar unit
        const __attribute__((address_space(4))) int32_t* tab = (const __attribute__((address_space(4))) int32_t*)(P.table + b * P.ts);
        return tab[at_page(P.page_mul, P.page_shift, j)];
    };
    auto pages_of = [&](int j, int n) {                      // the page of key j + lane % KT, the last of n for those behind
        const int e = (lane & (KT - 1)) < n ? (lane & (KT - 1)) : n - 1;
        return P.table ? P.table[b * P.ts + at_page(P.page_mul, P.page_shift, j + e)] : 0;
    };
    auto known = [&](int p) {                                // a page that exists; others are noted
        if (!P.table) return 0;                              // uniform
        const bool out = p < 0 || p >= P.pages;
        miss |= out;
        return out ? 0 : p;
    };
    auto inside = [&](int j) { return P.table ? j - (int)at_page(P.page_mul, P.page_shift, j) * P.page : j; };
    // the head's rows: of every page, or of the sequence where there are no pages (its page is 0 then)
    const int64_t own = P.table ? 0 : b;
    const uint8_t* kh = (const uint8_t*)P.kc + own * P.kcs[0] + h * P.kcs[2];
    const uint8_t* vh = (const uint8_t*)P.vc + own * P.vcs[0] + h * P.vcs[2];
    const float *ksh = P.ksc + own * P.kss[0] + h * P.kss[2], *vsh = P.vsc + own * P.vss[0] + h * P.vss[2];
    // What every tile's addresses are made from; hidden from the compiler, which else loads it anew for each tile, one
    // wait after the other: a fifth of a tile's time with three row tiles (with `aim`, 33 nodes over 4 x 131072 tokens 498
    // -> 470 us).  One row tile waits for memory in any case, and starts sequences more often (64 of one token: hidden
    // 143 us in a graph, not hidden 141).
    constexpr bool HIDE = !GEN && M > 1;
    uint32_t kst[2] = {(uint32_t)P.kcs[0], (uint32_t)P.kcs[1]}, vst[2] = {(uint32_t)P.vcs[0], (uint32_t)P.vcs[1]};
    uint32_t sst[4] = {(uint32_t)P.kss[0], (uint32_t)P.kss[1], (uint32_t)P.vss[0], (uint32_t)P.vss[1]};
    if constexpr (HIDE) {
        asm volatile("" : "+s"(kh), "+s"(vh), "+s"(ksh), "+s"(vsh));
        asm volatile("" : "+s"(kst[0]), "+s"(kst[1]), "+s"(vst[0]), "+s"(vst[1]), "+s"(sst[0]), "+s"(sst[1]), "+s"(sst[2]), "+s"(sst[3]));
    }
    // page p, place o of it, by strides below 2^32 (AT_TILE, AT_REQUEST)
    auto at32 = [&](auto* base, int p, int o, uint32_t s0, uint32_t s1) {
        return base + ((uint64_t)(uint32_t)p * s0 + (uint64_t)(uint32_t)o * s1);
    };
    auto lds = [](uint8_t* p) { return (__attribute__((address_space(3))) void*)p; };
    auto rsrc = [](const void* p) { return __builtin_amdgcn_make_buffer_rsrc((void*)p, 0, 0x7FFFFFFF, 0x00027000); };
    int pg = 0;                                              // the page of the next tile to request; GEN: of the lane's key
    // the next tile to request (AT_TILE): its addresses are made while the matrix cores are busy
    const uint8_t *ak = nullptr, *av = nullptr;
    const float *aks = nullptr, *avs = nullptr;
    auto aim = [&](int tile) __attribute__((always_inline)) {
        if constexpr (!GEN) {
            const int j = key_of(tile);
            if (tile >= nC || len - j < KT) return;          // uniform
            const int p = known(pg), o = inside(j);
            ak = at32(kh, p, o, kst[0], kst[1]);
            av = at32(vh, p, o, vst[0], vst[1]);
            aks = at32(ksh, p, o, sst[0], sst[1]);
            avs = at32(vsh, p, o, sst[2], sst[3]);
        }
    };
    auto lookup = [&](int tile) {
        if (tile >= nC) return;                              // uniform
        const int j = key_of(tile);
        if constexpr (GEN) pg = pages_of(j, len - j);
        else if (P.table) pg = page_of(j);                   // uniform
    };
    // lane numbers that the compiler does not know to be the same in every tile: what is made from them is not
    // kept in registers, nor spilled
    auto fresh = [&](int x) {
        if constexpr (M * D >= 384) asm volatile("" : "+v"(x));
        return (uint32_t)x;
    };
    // a cached tile, the lane's own addresses; its n keys, the last of them again behind it
    auto issue_lanes = [&](int j, int n, int pgl, uint8_t* st) {
        const At8Args A = a8_args();
        const int ln = (int)fresh(lane), kq = ln / U, unit = ln % U;
#pragma unroll 1
        for (int i = 0; i < 2 * NQ; ++i) {
            const int ki = (i % NQ) * KQ + kq, k = ki < n ? ki : n - 1;
            const int p = known(__shfl(pgl, k, 64)), o = inside(j + k);
            const uint32_t u = (uint32_t)(unit ^ a8_swz<D>((uint32_t)ki)) * 16;
            const uint8_t* src = i < NQ ? kh + p * A->kcs[0] + o * A->kcs[1] : vh + p * A->vcs[0] + o * A->vcs[1];
            const auto from = (const __attribute__((address_space(1))) void*)(src + u);
            const auto to = (__attribute__((address_space(3))) void*)(st + i * 1024);
            if (A->RG == 1) __builtin_amdgcn_global_load_lds(from, to, 16, 0, 2);   // uniform
            else __builtin_amdgcn_global_load_lds(from, to, 16, 0, 0);
            if (i % NQ == NQ - 1) {                          // uniform: K's or V's scales
                const int ks = (lane & (KT - 1)) < n ? (lane & (KT - 1)) : n - 1, ps = known(pgl), os = inside(j + ks);
                const float* sc = i < NQ ? ksh + ps * A->kss[0] + os * A->kss[1] : vsh + ps * A->vss[0] + os * A->vss[1];
                if (lane < KT)
                    __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)sc,
                                                     (__attribute__((address_space(3))) void*)(st + 2 * KT * D + i / NQ * (KT * 4)), 4, 0, 0);
            }
        }
    };
    auto issue = [&](int tile, uint8_t* st) __attribute__((always_inline)) {
        if (tile < nC) {                                     // uniform
            const int j = key_of(tile), n = len - j < KT ? len - j : KT;
            const int pgl = pg;
            if constexpr (GEN) lookup(tile + 1);
            const uint32_t ln = fresh(lane), kq = ln / U;
            auto unit_at = [&](int i) { return ((ln % U) ^ a8_swz<D>((uint32_t)(i * KQ) + kq)) * 16; };   // of request i
            if (!GEN && n == KT) {                           // uniform
                const auto rk = rsrc(ak), rv = rsrc(av), sk = rsrc(aks), sv = rsrc(avs);
                uint32_t k1 = kst[1], v1 = vst[1];           // (not kept multiplied: a value spilled costs more)
                if constexpr (HIDE) asm volatile("" : "+s"(k1), "+s"(v1));
                auto requests = [&](auto nt) {
                    constexpr int AUX = decltype(nt)::value;
#pragma unroll
                    for (int i = 0; i < NQ; ++i)
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, lds(st + i * 1024), 16, (int)(kq * k1 + unit_at(i)), i * KQ * (int)k1, 0, AUX);
                    if (lane < KT) __builtin_amdgcn_raw_ptr_buffer_load_lds(sk, lds(st + 2 * KT * D), 4, lane * (int)(4 * sst[1]), 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < NQ; ++i)
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, lds(st + KT * D + i * 1024), 16, (int)(kq * v1 + unit_at(i)), i * KQ * (int)v1, 0, AUX);
                    if (lane < KT) __builtin_amdgcn_raw_ptr_buffer_load_lds(sv, lds(st + 2 * KT * D + KT * 4), 4, lane * (int)(4 * sst[3]), 0, 0, 0);
                };
                // values that one workgroup reads pass by L2 (16 nodes, 24 x 8192 tokens: 114 -> 103 us), those of several
                // row groups stay in it; as a branch here, its spilled descriptors cost 465 instead of 430 us (33 nodes
                // over 4 x 131072)
                requests(std::integral_constant<int, KIND == A8_ONE ? 2 : 0>{});
            } else if (GEN && P.mode == AT_REQUEST && n == KT) {   // uniform
                int p[NQ], o[NQ];
#pragma unroll
                for (int i = 0; i < NQ; ++i) {
                    p[i] = known((int)readlane((uint32_t)pgl, (uint32_t)(i * KQ)));
                    o[i] = inside(j + i * KQ);
                }
                int pl = p[0], ol = o[0];                    // the lane's key of the scales
#pragma unroll
                for (int i = 1; i < NQ; ++i)
                    if ((lane & (KT - 1)) >= i * KQ) { pl = p[i]; ol = o[i]; }
                ol += lane & (KQ - 1);
                auto requests = [&](auto nt) {
                    constexpr int AUX = decltype(nt)::value;
#pragma unroll
                    for (int i = 0; i < NQ; ++i)
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(at32(kh, p[i], o[i], kst[0], kst[1])), lds(st + i * 1024), 16,
                            (int)(kq * (uint32_t)P.kcs[1] + unit_at(i)), 0, 0, AUX);
                    if (lane < KT) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(ksh), lds(st + 2 * KT * D), 4,
                            (pl * (int)P.kss[0] + ol * (int)P.kss[1]) * 4, 0, 0, 0);
#pragma unroll
                    for (int i = 0; i < NQ; ++i)
                        __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(at32(vh, p[i], o[i], vst[0], vst[1])), lds(st + KT * D + i * 1024), 16,
                            (int)(kq * (uint32_t)P.vcs[1] + unit_at(i)), 0, 0, AUX);
                    if (lane < KT) __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc(vsh), lds(st + 2 * KT * D + KT * 4), 4,
                            (pl * (int)P.vss[0] + ol * (int)P.vss[1]) * 4, 0, 0, 0);
                };
                if (P.RG == 1) requests(std::integral_constant<int, 2>{});   // uniform
                else requests(std::integral_constant<int, 0>{});
            } else {
                issue_lanes(j, n, GEN ? pgl : pages_of(j, n), st);
            }
        } else {
            const At8Args A = a8_args();
            const int m0 = draft_of(tile), n = A->N - m0 < DK ? A->N - m0 : DK;
            const int ln = (int)fresh(lane), kq2 = ln / U2, unit2 = ln % U2;
#pragma unroll 1
            for (int i = 0; i < 2 * NQ; ++i) {
                const int ki = (i % NQ) * KQ2 + kq2, k = ki < n ? ki : n - 1;
                const uint32_t u = (uint32_t)(unit2 ^ a8_swz<2 * D>((uint32_t)ki)) * 16;
                const uint16_t* src = i < NQ ? (const uint16_t*)A->k + b * A->ks[0] + (int64_t)(m0 + k) * A->ks[1] + h * A->ks[2]
                                             : (const uint16_t*)A->v + b * A->vs[0] + (int64_t)(m0 + k) * A->vs[1] + h * A->vs[2];
                at_dma((const uint8_t*)src + u, st + i * 1024);
            }
        }
    };
    // ---------------------------------------------------------------- Q, loaded before the first requests
    const int row0 = rg * M * 16;
    auto last_row = [&](int row) { return row < P.R ? row : P.R - 1; };
    auto node_of = [&](At8Args A, int row) { return (int)at_page(A->g_mul, A->g_shift, row); };   // row's node; its query head
    auto head_of = [&](At8Args A, int row, int n) { return h * A->G + row - n * A->G; };
    auto q_at = [&](At8Args A, int row, int col) {
        row = last_row(row);
        const int n = node_of(A, row);
        return (const uint16_t*)A->q + b * A->qs[0] + (int64_t)n * A->qs[1] + (int64_t)head_of(A, row, n) * A->qs[2] + col;
    };
    const At8Args AQ = a8_args();
    const int tq = (int)fresh(t);
    constexpr int QI = (QL * 16 * U2 + 64 * NW - 1) / (64 * NW);
    llima_u32x4 ql[QI];
#pragma unroll
    for (int e = 0; e < QI; ++e) {
        const int i = tq + e * 64 * NW;
        ql[e] = *(const llima_u32x4*)q_at(AQ, row0 + i / U2, i % U2 * 8);
    }
    at_s8 qr[QR > 0 ? QR : 1][D / 32];
#pragma unroll
    for (int m = 0; m < QR; ++m)
#pragma unroll
        for (int s = 0; s < D / 32; ++s) qr[m][s] = *(const at_s8*)q_at(AQ, row0 + (QL + m) * 16 + (tq & 15), (s >> 1) * 64 + (tq >> 4 & 3) * 16 + (s & 1) * 8);
    asm volatile("" ::: "memory");
    lookup(0);
    for (int e = 0; e < S - 1 && e < ntile; ++e) {
        aim(e);
        if constexpr (!GEN) lookup(e + 1);
        issue(e, ring + e * ST);
    }
    aim(S - 1);
#pragma unroll
    for (int e = 0; e < QI; ++e) {
        const int i = tq + e * 64 * NW, rw = i / U2;
        if (P.flip) ql[e] ^= 0x80008000u;                    // uniform: a negative scale's sign goes to q
        if (QL * 16 * U2 % (64 * NW) == 0 || rw < QL * 16)
            *(llima_u32x4*)(sq + rw * 2 * D + ((uint32_t)(i % U2) ^ a8_swz<2 * D>((uint32_t)(rw & 15))) * 16) = ql[e];
    }
#pragma unroll
    for (int m = 0; m < QR; ++m)
#pragma unroll
        for (int s = 0; s < D / 32; ++s)
            if (P.flip) qr[m][s] ^= (short)0x8000;
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    // step s of a product takes columns 64 (s / 2) + 16 g + 8 (s % 2) + 0 .. 7 of the lane
    auto qread = [&](int m, int s, uint32_t base) {
        if (m < QL) return *(const at_s8*)(sq + m * QT + (base ^ (uint32_t)((s >> 1) * 128 + (s & 1) * 16)));
        return qr[m < QL ? 0 : m - QL][s];
    };
    // the lane's place of step 0 in a row tile of Q
    auto qplace = [&](uint32_t rr, uint32_t gg) { return rr * 2 * D + ((2 * gg) ^ a8_swz<2 * D>(rr)) * 16; };
    // ---------------------------------------------------------------- products
    a8_acc o[M][DB];
    // mu: what a row's scores (base 2) are taken less; a score less mu is its weight's logarithm, which with the logarithm of
    // the value's scale is at most `most`: -inf for a row that has seen nothing yet
    float mu[M], most[M], l[M];
#pragma unroll
    for (int m = 0; m < M; ++m) {
        mu[m] = l[m] = 0.0f;
        most[m] = -__builtin_inff();
#pragma unroll
        for (int d = 0; d < DB; ++d) o[m][d] = (a8_acc){0.0f, 0.0f, 0.0f, 0.0f};
    }
    // The softmax of blocks of scores less mu, in place: x becomes the weights.  logs(k, i): the logarithm of what a key's
    // weight is multiplied by; bound: no less than that of any of the lane's keys.
    auto softmax = [&](auto& x, auto blocks, float bound, auto logs) {
        constexpr int BL = decltype(blocks)::value;
        bool up = false;
#pragma unroll
        for (int m = 0; m < M; ++m) {
            float a = a8_max(x[m][0][0], x[m][0][1], a8_max(x[m][0][2], x[m][0][3], x[m][0][3]));
#pragma unroll
            for (int k = 1; k < BL; ++k) a = a8_max(x[m][k][0], x[m][k][1], a8_max(x[m][k][2], x[m][k][3], a));
            up |= a > most[m] - bound;
        }
        if (__any(up)) {
#pragma unroll
            for (int m = 0; m < M; ++m) {
                float a0 = -__builtin_inff();
#pragma unroll
                for (int k = 0; k < BL; ++k)
                    a0 = a8_max(x[m][k][0] + logs(k, 0), x[m][k][1] + logs(k, 1), a8_max(x[m][k][2] + logs(k, 2), x[m][k][3] + logs(k, 3), a0));
                const float top = a8_max4(a0);               // of the row's
                const bool raise = top > most[m];
                // (more often than not the bound alone was passed: 455 -> 447 us, 33 nodes over 4 x 131072 tokens; with one row
                // tile, pages of 16: 85 -> 94, 24 x 8192)
                if (M > 1 && !__any(raise)) continue;
                const float to = raise ? mu[m] + (top - (A8_MOST - A8_HEAD)) : mu[m], by = to - mu[m];
                // (half of it, twice: a sum of weights without their scales may be 2^230 above what is added to it next)
                const float a = !raise ? 1.0f : most[m] > 0.0f ? __builtin_amdgcn_exp2f(-0.5f * by) : 0.0f;
                mu[m] = to;
                most[m] = raise ? A8_MOST : most[m];
                l[m] = l[m] * a * a;
#pragma unroll
                for (int d = 0; d < DB; ++d) o[m][d] *= a * a;
#pragma unroll
                for (int k = 0; k < BL; ++k) x[m][k] -= by;
            }
        }
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < BL; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[m][k][i] = __builtin_amdgcn_exp2f(x[m][k][i]);
                    l[m] += x[m][k][i];
                }
    };
    auto lds_at = [](const uint8_t* p) { return (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)p; };
    // A staged tile of n cached keys; K has landed, and V too unless there are requests of more tiles.
    auto math8 = [&](const uint8_t* st, int n, bool more, int next) __attribute__((always_inline)) {
        const uint32_t rr = fresh(r), gg = fresh(g), qb = qplace(rr, gg);
        a8_acc x[M][NB], ks[NB];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < NB; ++k) x[m][k] = (a8_acc){0.0f, 0.0f, 0.0f, 0.0f};
        // K's pieces of 64 columns, and Q's of 32, are read a step before their products (each waited for where it was
        // read before: 16 nodes, 24 x 8192 tokens, 118 -> 113 us)
        llima_u32x4 kr[2][NB];
        at_s8 q[2][M];
        auto kread = [&](int c) {
#pragma unroll
            for (int k = 0; k < NB; ++k)
                kr[c & 1][k] = *(const llima_u32x4*)(st + k * 16 * D + ((rr * D + (gg ^ a8_swz<D>(rr)) * 16) ^ (uint32_t)(c * 64)));
        };
        auto qreads = [&](int s) {
#pragma unroll
            for (int m = 0; m < M; ++m) q[s & 1][m] = qread(m, s, qb);
        };
        kread(0);
        if (AHEAD) qreads(0);
#pragma unroll
        for (int k = 0; k < NB; ++k) ks[k] = *(const a8_acc*)(st + 2 * KT * D + k * 64 + g * 16);
        __builtin_amdgcn_s_setprio(1);                       // the wave with products to issue goes before the one in the softmax
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            if (!AHEAD) qreads(s);
            if (s % 2 == 0 && s + 2 < D / 32) kread(s / 2 + 1);
            if (AHEAD && s + 1 < D / 32) qreads(s + 1);
            __builtin_amdgcn_sched_barrier(0);
            at_s8 kf[NB];
#pragma unroll
            for (int k = 0; k < NB; ++k) kf[k] = a8_wide<DT>(kr[s >> 1 & 1][k][2 * (s & 1)], kr[s >> 1 & 1][k][2 * (s & 1) + 1]);
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int k = 0; k < NB; ++k) x[m][k] = a8_mfma<DT>(kf[k], q[s & 1][m], x[m][k]);
            if (s == 0) aim(next);
            __builtin_amdgcn_sched_barrier(0);               // (else the reads of Q come all at once)
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int k = 0; k < NB; ++k) ks[k] *= P.scale2;
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) x[m][k][i] = __builtin_fmaf(x[m][k][i], ks[k][i], -mu[m]);
        if (n < KT) {                                        // uniform: the sequence's last cached keys
#pragma unroll
            for (int k = 0; k < NB; ++k)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const bool in = k * 16 + 4 * (int)gg + i < n;
#pragma unroll
                    for (int m = 0; m < M; ++m) x[m][k][i] = in ? x[m][k][i] : -__builtin_inff();
                }
        }
        if (more) a8_wait<(S - 1) * NR>();                   // uniform
        a8_acc vs[NB];
#pragma unroll
        for (int k = 0; k < NB; ++k) vs[k] = *(const a8_acc*)(st + 2 * KT * D + KT * 4 + k * 64 + g * 16);
        float top = 0.0f;
#pragma unroll
        for (int k = 0; k < NB; ++k) {
            vs[k] *= (float)(1 << A8_UNIT);
            top = a8_max_abs(vs[k][0], vs[k][1], a8_max_abs(vs[k][2], vs[k][3], top));
        }
        // (an infinite scale's logarithm is 127, its bound 129)
        softmax(x, std::integral_constant<int, NB>{}, __builtin_fminf(__builtin_fmaxf(__builtin_amdgcn_logf(top) + 0.001f, A8_LEAST), 129.0f),
                [&](int k, int i) { return __builtin_fminf(__builtin_fmaxf(__builtin_amdgcn_logf(__builtin_fabsf(vs[k][i])), A8_LEAST), 127.0f); });
        uint32_t pw[M][2 * NB];
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int k = 0; k < NB; ++k) {
                const a8_acc y = x[m][k] * vs[k];
                pw[m][2 * k] = at_pack<LLIMA_F16>(y[0], y[1]);
                pw[m][2 * k + 1] = at_pack<LLIMA_F16>(y[2], y[3]);
            }
        __builtin_amdgcn_s_setprio(1);
        // V: a transposing load takes 8 rows of 16 bytes from 16 lanes (row i / 2 of lane i, half i % 2)
        const uint32_t e = rr >> 1;
        if constexpr (NB == 2) {                             // keys 4 g + 0 .. 3 and 16 more of a column block
            const uint32_t key = 4 * gg + (e & 3) + (e >> 2) * 16;
            const uint32_t base = KT * D + ((key * D + (rr & 1) * 8) | (a8_swz<D>(key) << 4)), at = lds_at(st);
#pragma unroll
            for (int d = 0; d < DB; d += VG) {
                uint32_t a[VG];
                a8_i2 v[VG];
#pragma unroll
                for (int i = 0; i < VG; ++i) a[i] = at + (base ^ (uint32_t)((d + i) << 4));
                a8_tr8(a, v);
#pragma unroll
                for (int i = 0; i < VG; ++i) {
                    const at_s8 vf = a8_wide<LLIMA_F16>((uint32_t)v[i][0], (uint32_t)v[i][1]);
#pragma unroll
                    for (int m = 0; m < M; ++m)
                        o[m][d + i] = a8_mfma<LLIMA_F16>(vf, __builtin_bit_cast(at_s8, (llima_u32x4){pw[m][0], pw[m][1], pw[m][2 * NB - 2], pw[m][2 * NB - 1]}), o[m][d + i]);
                }
            }
        } else {                                             // keys 4 g + 0 .. 3 of two column blocks
            const uint32_t key = 4 * gg + (e & 3);
            const uint32_t base = KT * D + ((key * D + (rr & 1) * 8) | (a8_swz<D>(key) ^ (e >> 2)) << 4), at = lds_at(st);
#pragma unroll
            for (int d = 0; d < DB; d += 8) {
                uint32_t a[4];
                a8_i2 v[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) a[i] = at + (base ^ (uint32_t)((d + 2 * i) << 4));
                a8_tr8(a, v);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const at_s8 vf = a8_wide<LLIMA_F16>((uint32_t)v[i][0], (uint32_t)v[i][1]);
#pragma unroll
                    for (int m = 0; m < M; ++m) {
                        const at_s4 pf = __builtin_bit_cast(at_s4, (a8_i2){(int)pw[m][0], (int)pw[m][1]});
                        o[m][d + 2 * i] = a8_mfma<LLIMA_F16>(__builtin_shufflevector(vf, vf, 0, 1, 2, 3), pf, o[m][d + 2 * i]);
                        o[m][d + 2 * i + 1] = a8_mfma<LLIMA_F16>(__builtin_shufflevector(vf, vf, 4, 5, 6, 7), pf, o[m][d + 2 * i + 1]);
                    }
                }
            }
        }
        __builtin_amdgcn_s_setprio(0);
    };
    auto seen = [&](At8Args A, int n, int mm) {              // node n sees drafted token mm
        if (!A->mask) return mm <= n;
        if (A->mask_f32) return ((const float*)A->mask)[b * A->ms[0] + n * A->ms[1] + mm] > 0.0f;
        return ((const uint8_t*)A->mask)[b * A->ms[0] + n * A->ms[1] + mm] != 0;
    };
    // A staged tile of n drafted tokens from m0 on.
    auto math16 = [&](uint8_t* st, int m0, int n) __attribute__((always_inline)) {
        const At8Args A = a8_args();
        const int r = (int)fresh(t) & 15, g = (int)fresh(t) >> 4 & 3;
        a8_acc x[M][1];
        uint32_t sees[M];                                    // bit i: the row sees token m0 + 4 g + i
        auto masks = [&](auto at) {                          // every load before the first use
            decltype(at(0)) v[M][4];
#pragma unroll
            for (int m = 0; m < M; ++m)
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[m][i] = at(b * A->ms[0] + node_of(A, last_row(row0 + m * 16 + r)) * A->ms[1] + m0 + (4 * g + i < n ? 4 * g + i : n - 1));
#pragma unroll
            for (int m = 0; m < M; ++m) {
                sees[m] = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) sees[m] |= v[m][i] > 0 ? 1u << i : 0u;
            }
        };
        if (!A->mask) {                                      // uniform
#pragma unroll
            for (int m = 0; m < M; ++m) {
                const int c = node_of(A, last_row(row0 + m * 16 + r)) - m0 - 4 * g + 1;
                sees[m] = c <= 0 ? 0u : c >= 4 ? 15u : (1u << c) - 1;
            }
        } else if (A->mask_f32) {                            // uniform
            masks([&](int64_t i) { return ((const float*)A->mask)[i]; });
        } else {
            masks([&](int64_t i) { return ((const uint8_t*)A->mask)[i]; });
        }
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const int c = n - 4 * g;                         // tokens behind the last are nobody's
            sees[m] &= c <= 0 ? 0u : c >= 4 ? 15u : (1u << c) - 1;
            x[m][0] = (a8_acc){0.0f, 0.0f, 0.0f, 0.0f};
        }
        a8_wait<0>();
        // Values that not every row sees: infinities and NaN become 0 (0 times them would be NaN
        // for the rows that do not see them; at the end they are added to the rows that do).
        for (int p = lane; p < DK * U2; p += 64) {
            llima_u32x4* const at = (llima_u32x4*)(st + KT * D + p * 16);
            llima_u32x4 y = *at;
            bool put = false;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                uint32_t w = y[e];
                if (at_special<DT>((uint16_t)w)) { w &= 0xFFFF0000u; put = true; }
                if (at_special<DT>((uint16_t)(w >> 16))) { w &= 0xFFFFu; put = true; }
                y[e] = w;
            }
            if (put) { *at = y; flag[1] = 1u; }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        const uint32_t kr = (uint32_t)r & (DK - 1);
#pragma unroll
        for (int s = 0; s < D / 32; ++s) {
            const at_s8 kf = *(const at_s8*)(st + kr * 2 * D + ((uint32_t)((s >> 1) * 8 + 2 * g + (s & 1)) ^ a8_swz<2 * D>(kr)) * 16);
#pragma unroll
            for (int m = 0; m < M; ++m) x[m][0] = a8_mfma<DT>(kf, qread(m, s, qplace((uint32_t)r, (uint32_t)g)), x[m][0]);
        }
#pragma unroll
        for (int m = 0; m < M; ++m)
#pragma unroll
            for (int i = 0; i < 4; ++i) x[m][0][i] = sees[m] >> i & 1 ? __builtin_fmaf(x[m][0][i], P.scale2, -mu[m]) : -__builtin_inff();
        // bf16: weights of at most 2^-11, which keep the sum of 1024 products with any values of the type finite
        constexpr float LG = DT == LLIMA_BF16 ? A8_UNIT + A8_MOST + 11.0f : A8_UNIT;
        softmax(x, std::integral_constant<int, 1>{}, LG, [](int, int) { return LG; });
        at_s4 pf[M];
#pragma unroll
        for (int m = 0; m < M; ++m) {
            const a8_acc y = x[m][0] * (float)(1 << A8_UNIT);
            pf[m] = __builtin_bit_cast(at_s4, (a8_i2){(int)at_pack<DT>(y[0], y[1]), (int)at_pack<DT>(y[2], y[3])});
        }
        // a transposing load takes 4 rows of 32 bytes from 16 lanes (row i / 4 of lane i, 8 bytes i % 4)
        const uint32_t key = (uint32_t)(4 * g + (r >> 2)) & (DK - 1);
        const uint32_t base = lds_at(st) + KT * D + key * 2 * D + (uint32_t)(r & 1) * 8, z = a8_swz<2 * D>(key), half = (uint32_t)(r >> 1 & 1);
#pragma unroll
        for (int d = 0; d < DB; d += 4) {
            uint32_t a[4];
            at_s4 v[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = base + (((uint32_t)(2 * (d + i)) + half ^ z) << 4);
            a8_tr16(a, v);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int m = 0; m < M; ++m) o[m][d + i] = a8_mfma<DT>(v[i], pf[m], o[m][d + i]);
        }
    };
    int slot = 0;
    for (int tile = 0; tile < nC; ++tile) {
        const int ahead = tile + S - 1;
        uint8_t* const st = ring + slot * ST;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");   // the slot's last tile has been read
        if (ahead < ntile) issue(ahead, ring + (slot == 0 ? S - 1 : slot - 1) * ST);   // uniform
        const int n = len - key_of(tile) < KT ? len - key_of(tile) : KT;
        // cached tiles behind this one have NR requests each, drafted ones fewer: then everything is waited for
        const bool more = ahead < nC;                        // uniform
        if constexpr (!GEN) lookup(ahead + 1);
        if (more) a8_wait<(S - 1) * NR + NQ + 1>();
        else a8_wait<0>();
        math8(st, n, more, ahead + 1);
        slot = slot + 1 < S ? slot + 1 : 0;
    }
    for (int tile = nC; tile < ntile; ++tile) {
        const int ahead = tile + S - 1;
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (ahead < ntile) issue(ahead, ring + (slot == 0 ? S - 1 : slot - 1) * ST);   // uniform
        const int m0 = draft_of(tile);
        math16(ring + slot * ST, m0, P.N - m0 < DK ? P.N - m0 : DK);
        slot = slot + 1 < S ? slot + 1 : 0;
    }
    // ---------------------------------------------------------------- the waves' sums
    if (miss) flag[0] = 1u;
    __syncthreads();                                         // no wave reads or fills its ring any more
    const int r = (int)fresh(t) & 15, g = (int)fresh(t) >> 4 & 3, lane = (int)fresh(t) & 63;
    float2* const ml = (float2*)(sm + XN * XB);              // [wave][row]
#pragma unroll
    for (int m = 0; m < M; ++m) {
        // the sum's exponent goes into mu: sums of other waves and parts may have had far smaller or larger scales; sums of
        // less than 2^-11, which keep those of four waves in 512 parts times any values finite
        const float sum = a8_sum4(l[m]);
        const int e = __builtin_amdgcn_frexp_expf(sum) + 11; // (of 0, infinities and NaN: 0)
        mu[m] += (float)e;
        l[m] = __int_as_float(-e - A8_UNIT);                 // the exponent of what o is multiplied by
        if (g == 0) ml[wave * M * 16 + m * 16 + r] = make_float2(most[m] > 0.0f ? mu[m] : -__builtin_inff(), __builtin_amdgcn_ldexpf(sum, -e));
    }
    __syncthreads();
    const At8Args A = a8_args();
    const bool nan = flag[0] != 0, special = flag[1] != 0;
    const int drow0 = (c0 > nc ? c0 - nc : 0) * TD, drow1 = c1 - nc <= 0 ? 0 : (c1 - nc) * TD < P.N ? (c1 - nc) * TD : P.N;   // the part's drafted tokens
#pragma unroll
    for (int m = 0; m < M; ++m) {
        float2 x[NW];
        float top = -__builtin_inff(), sum = 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) {
            x[w] = ml[w * M * 16 + m * 16 + r];
            top = __builtin_fmaxf(top, x[w].x);
        }
        const float zero = top > -__builtin_inff() ? top : 0.0f;
#pragma unroll
        for (int w = 0; w < NW; ++w) sum += x[w].y * __builtin_amdgcn_exp2f(x[w].x - zero);
        const float a = __builtin_amdgcn_ldexpf(most[m] > 0.0f ? __builtin_amdgcn_exp2f(mu[m] - zero) : 0.0f, __float_as_int(l[m]));
        uint8_t* const xb = sm + (XN == 2 ? (m & 1) * XB : 0);
        if (XN == 1 && m > 0) __syncthreads();
#pragma unroll
        for (int d = 0; d < DB; ++d) *(a8_acc*)(xb + (wave * DB + d) * 1024 + lane * 16) = o[m][d] * a;
        __syncthreads();
        const int row = row0 + m * 16 + r;
        if (nan) sum = __builtin_nanf("");
        if (row < P.R) {
            const int n = node_of(A, row), hq = head_of(A, row, n);
            const float inv = whole ? at_inverse(A, sum, b, n, len) : 1.0f;
            const size_t at = ((size_t)at_slot(A->pairs, part, b, c0 == 0) * A->Hkv + h) * P.R + row;
            if (!whole && wave == 0 && g == 0) A->part_ml[at] = make_float2(top, sum);
#pragma unroll
            for (int i = 0; i < DB / NW; ++i) {
                const int d = wave + NW * i;
                a8_acc y = *(const a8_acc*)(xb + d * 1024 + lane * 16);
#pragma unroll
                for (int w = 1; w < NW; ++w) y += *(const a8_acc*)(xb + (w * DB + d) * 1024 + lane * 16);
                if (special) {                               // uniform: infinities and NaN of drafted tokens in this part
                    for (int mm = drow0; mm < drow1; ++mm) {
                        if (!seen(A, n, mm)) continue;          // (of the loop over mm)
                        const uint2 v = *(const uint2*)((const uint16_t*)A->v + b * A->vs[0] + (int64_t)mm * A->vs[1] + h * A->vs[2] + d * 16 + 4 * g);
                        auto add = [&](int e, uint32_t u) { y[e] += at_special<DT>((uint16_t)u) ? at_f32<DT>((uint16_t)u) : 0.0f; };
                        add(0, v.x); add(1, v.x >> 16); add(2, v.y); add(3, v.y >> 16);
                    }
                }
                if (whole) {
                    y *= inv;
                    *(uint2*)((uint16_t*)A->out + b * A->os[0] + n * A->os[1] + hq * A->os[2] + d * 16 + 4 * g) =
                        make_uint2(at_pack<DT>(y[0], y[1]), at_pack<DT>(y[2], y[3]));
                } else {
                    *(a8_acc*)(A->part_o + at * D + d * 16 + 4 * g) = y;
                }
            }
        }
    }
    }
#endif
}

// f(M) with the number of row tiles as a constant.
template <int D, class F>
static void a8_tiles(int RT, F f) {
    if (RT == 1) f(std::integral_constant<int, 1>{});
    else if (RT == 2) f(std::integral_constant<int, 2>{});
    else if constexpr (A8<D>::MAXM > 2) {
        if (RT == 3) f(std::integral_constant<int, 3>{});
        else f(std::integral_constant<int, 4>{});
    }
}

template <int D>
static void a8_plan_at(AttnParams& P) {                      // RT: row tiles of 16 of a group
    P.R = P.N * P.G;
    const int tiles = (P.R + 15) / 16;
    P.RG = (tiles + A8<D>::MAXM - 1) / A8<D>::MAXM;
    P.RT = (tiles + P.RG - 1) / P.RG;
    P.parts = 512 / (P.Hkv * P.RG);                          // as many workgroups as the device holds at a time, two per CU
    if (P.parts < 1) P.parts = 1;
    at_slots(P);
}

static void a8_plan(AttnParams& P, int D) {
    if (D == 64) a8_plan_at<64>(P);
    else if (D == 128) a8_plan_at<128>(P);
    else a8_plan_at<256>(P);
}

template <int DT, int D, bool GEN>
static void a8_launch(const At8Params& P, hipStream_t st) {
    a8_tiles<D>(P.RT, [&](auto m) {
        constexpr int M = decltype(m)::value;
        const int64_t rows = (int64_t)P.B * P.N * P.Hq;
        const AttnParams& J = P;
        auto go = [&](auto kind) {
            constexpr int KIND = decltype(kind)::value;
            hipLaunchKernelGGL((tree_attn8<DT, D, M, KIND>), dim3(((uint32_t)P.parts * P.Hkv + 7) / 8 * 8 * P.RG), dim3(64 * A8<D>::NW), 0, st, P);
        };
        if constexpr (GEN) go(std::integral_constant<int, A8_GEN>{});
        else if constexpr (2 * M <= A8<D>::MAXM) go(std::integral_constant<int, A8_ONE>{});   // (several groups have more tiles each)
        else if (P.RG == 1) go(std::integral_constant<int, A8_ONE>{});
        else go(std::integral_constant<int, A8_MANY>{});
        if (rows <= 1024) hipLaunchKernelGGL((tree_attn_join<DT, D, Fp8Tiles<D>, 4>), dim3((uint32_t)rows), dim3(LLIMA_WG), 0, st, J);
        else hipLaunchKernelGGL((tree_attn_join<DT, D, Fp8Tiles<D>, 1>), dim3((uint32_t)((rows + 3) / 4)), dim3(LLIMA_WG), 0, st, J);
    });
}

template <int DT>
static int a8_dispatch(const At8Params& P, int D, hipStream_t st) {
    const bool gen = P.mode != AT_TILE;
    if (D == 64) gen ? a8_launch<DT, 64, true>(P, st) : a8_launch<DT, 64, false>(P, st);
    else if (D == 128) gen ? a8_launch<DT, 128, true>(P, st) : a8_launch<DT, 128, false>(P, st);
    else gen ? a8_launch<DT, 256, true>(P, st) : a8_launch<DT, 256, false>(P, st);
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}

}  // namespace llima

using namespace llima;

extern "C" size_t llima_tree_attention_fp8_workspace_bytes(int32_t B, int32_t N, int32_t Hq, int32_t Hkv, int32_t D) {
    if (B <= 0 || !at_sizes_ok(B, N, Hq, Hkv, D)) return 0;
    AttnParams P = {};
    P.B = B; P.N = N; P.Hkv = Hkv; P.G = Hq / Hkv;
    a8_plan(P, D);
    return at_parts_bytes(P, D);
}

extern "C" int llima_tree_attention_fp8(const llima_tree_attention_fp8_args* x, void* workspace, size_t workspace_bytes,
                                        void* stream) {
    if (!x) return LLIMA_E_INVAL;
    const llima_tree_attention_args* a = &x->a;
    At8Params P = {};
    const int ok = at_fill(a, 16, P);
    if (ok != LLIMA_OK) return ok;
    if (!at_strides_ok(x->k_scale_strides, 3, 1) || !at_strides_ok(x->v_scale_strides, 3, 1)) return LLIMA_E_INVAL;
    if (a->B == 0) return LLIMA_OK;
    if (P.cap > 0 && (!x->k_scales || !x->v_scales)) return LLIMA_E_INVAL;
    if ((uintptr_t)x->k_scales % 4 || (uintptr_t)x->v_scales % 4) return LLIMA_E_INVAL;
    if (!workspace || workspace_bytes < llima_tree_attention_fp8_workspace_bytes(a->B, a->N, a->Hq, a->Hkv, a->D))
        return LLIMA_E_WORKSPACE;
    if ((uintptr_t)workspace % 16) return LLIMA_E_INVAL;
    P.ksc = x->k_scales; P.vsc = x->v_scales;
    int64_t span = 0;                                        // of the scales from a head's first on, in elements
    for (int i = 0; i < 3; ++i) {
        P.kss[i] = x->k_scale_strides[i]; P.vss[i] = x->v_scale_strides[i];
    }
    for (const int64_t* s : {P.kss, P.vss}) {
        const int64_t e = (s[0] > (1 << 29) ? 1 << 29 : s[0]) * (int64_t)P.pages + (s[1] > (1 << 29) ? 1 << 29 : s[1]) * (int64_t)P.page;
        span = e > span ? e : span;
    }
    // offsets within a tile (32 keys) or a request, and of the scales, have 31 bits
    const int64_t ts = P.kcs[1] > P.vcs[1] ? P.kcs[1] : P.vcs[1], ss = P.kss[1] > P.vss[1] ? P.kss[1] : P.vss[1];
    const int kt = a->D == 256 ? A8<256>::KT : A8<128>::KT, kq = 1024 / a->D;
    int64_t far = 0;                                         // the longest stride of pages
    for (const int64_t* s : {P.kcs, P.vcs, P.kss, P.vss}) far = P.table && s[0] > far ? s[0] : far;
    P.mode = ts > (1 << 25) || far > (int64_t)UINT32_MAX ? AT_LANE
           : ss <= (1 << 23) && (!P.table || P.page % kt == 0) ? AT_TILE
           : span < (1 << 29) && P.page % kq == 0 ? AT_REQUEST : AT_LANE;
    at_divisor(P.G, P.g_mul, P.g_shift);
    a8_plan(P, a->D);
    at_parts_at(P, a->D, workspace);
    return a->dtype == LLIMA_BF16 ? a8_dispatch<LLIMA_BF16>(P, a->D, (hipStream_t)stream)
                                  : a8_dispatch<LLIMA_F16>(P, a->D, (hipStream_t)stream);
}
