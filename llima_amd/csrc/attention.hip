// attention.hip -- attention of drafted tokens over a KV cache under a tree mask,
// and the commit of an accepted path into the cache (gfx950).
//
//   out[b][n][h] = sum_j p_j v_j,  p = softmax over the visible j of scale q . k_j
//
// Keys 0 .. len_b - 1 of sequence b are its cached tokens (every drafted token
// sees them), keys len_b + m its N drafted tokens, of which node n sees those with
// mask[b][n][m].  A row that sees nothing is 0.
//
// One pass over the keys with the running maximum and sum of the softmax (fp32,
// base 2).  The products are taken transposed: S^T = K Q^T has a query row in
// each lane's column, so that a row's maximum and sum are one lane's (and its
// partner's, lane ^ 32) and the rescaling is a scalar per lane; the lane's 16
// sums of a block of 32 keys are at once the operand of O^T = V^T P^T, whose key
// order is the one the lane holds (16 s + e % 4 + 8 (e / 4) + 4 g for element e of
// half g), and V is read from LDS through the transposing loads in that order.
// P is rounded to the cache's type for that product (by 2^-8 of a weight at most
// in bf16, 2^-11 in fp16: the precision of the values it multiplies; the outputs' error
// grows by 4 to 10 % by it, and each weight in two parts, which avoids that, takes 532 ->
// 665 us for 33 nodes over 4 x 131072 tokens); the row's sum takes the weights before the
// rounding.  In fp16 the weights carry a factor
// of 2^10, so that they become subnormal below 2^-24 of the row's largest.
//
// Bound: reading K and V once for all N Hq / Hkv rows of a key head.  Up to 128 such
// rows the loop over the tiles runs at the memory's rate (16 nodes, 4 query heads per key
// head: 8 x 16384 tokens 537 MB in 125 us, twice as many sequences 215: 5.9 TB/s for what
// is added, and as long with the products left out); some 25 us are the call's start, the
// masked tile, the partial sums and the join.  From five row tiles on the waves' chain
// of LDS reads, product, softmax and product bounds (4 x 131072 tokens, 33 nodes: 2.15 GB in
// 528-552 us, requests alone 408).  Heads of 256 with five row tiles and more spill 64 to 69
// registers.
#include "attention.hpp"

namespace llima {

// Keys KEY + (0 .. 3, 8 .. 11) + 4 g of every block of 32 columns, by the transposing
// loads from the lane's places.  In one piece with their wait: as builtins, the
// compiler waits for all the requests into LDS before them.
template <int D, int KEY>
__device__ __forceinline__ void at_vread(const uint32_t (&a)[4], at_s4 (&v)[D / 32][2]) {
    constexpr int K0 = KEY * D * 2, K1 = (KEY + 8) * D * 2;
    if constexpr (D == 64) {
        asm volatile("ds_read_b64_tr_b16 %0, %4 offset:%6\n\tds_read_b64_tr_b16 %1, %4 offset:%7\n\t"
                     "ds_read_b64_tr_b16 %2, %5 offset:%6\n\tds_read_b64_tr_b16 %3, %5 offset:%7\n\t"
                     "s_waitcnt lgkmcnt(0)"
                     : "=&v"(v[0][0]), "=&v"(v[0][1]), "=&v"(v[1][0]), "=&v"(v[1][1])
                     : "v"(a[0]), "v"(a[1]), "n"(K0), "n"(K1));
    } else {
#pragma unroll
        for (int d = 0; d < D / 32; d += 4)
            asm volatile("ds_read_b64_tr_b16 %0, %8 offset:%12\n\tds_read_b64_tr_b16 %1, %8 offset:%13\n\t"
                         "ds_read_b64_tr_b16 %2, %9 offset:%12\n\tds_read_b64_tr_b16 %3, %9 offset:%13\n\t"
                         "ds_read_b64_tr_b16 %4, %10 offset:%12\n\tds_read_b64_tr_b16 %5, %10 offset:%13\n\t"
                         "ds_read_b64_tr_b16 %6, %11 offset:%12\n\tds_read_b64_tr_b16 %7, %11 offset:%13\n\t"
                         "s_waitcnt lgkmcnt(0)"
                         : "=&v"(v[d][0]), "=&v"(v[d][1]), "=&v"(v[d + 1][0]), "=&v"(v[d + 1][1]),
                           "=&v"(v[d + 2][0]), "=&v"(v[d + 2][1]), "=&v"(v[d + 3][0]), "=&v"(v[d + 3][1])
                         : "v"(a[0]), "v"(a[1]), "v"(a[2]), "v"(a[3]), "n"(K0 + d * 64), "n"(K1 + d * 64));
    }
}

template <int N>
__device__ __forceinline__ void at_wait_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(N) : "memory");
}

// One workgroup: NW waves over one share of the keys, one key head and a group of
// up to NW / KW row tiles (32 rows each).  Keys come in tiles of T, requested straight
// into a ring of S stages; KW waves share a row tile and take half of a tile's keys each
// (KW = 2), or one takes all.  Two workgroups per CU with two stages of 64 keys each: one
// with four stages leaves the products alone on a SIMD (16 nodes over 8 x 16384 tokens 127
// -> 148 us), a third stage for K alone has nothing more to hide (127 -> 129).  Five and
// six row tiles take the eight waves too: twelve with halves of the keys need more
// registers than they have (33 nodes 590 -> 700 us).
//
// Tiles of cached keys alone are requested by mode: a tile lies in one page
// (contiguous caches and pages of a multiple of 64), its address is the wave's
// and comes from the scalar unit; or each request does (its 8 keys at most: pages of
// a multiple of 8); or every lane computes its own.  The tiles after them, which hold drafted keys
// or end a part, are requested by key and have the mask.  GEN: the last two modes.
template <int DT, int D, int NW, int KW, int T, int S, bool GEN>
__global__ __launch_bounds__(64 * NW, (D == 256 || NW == 2) ? 1 : 2) void tree_attn(AttnParams P) {
#ifdef __HIP_DEVICE_COMPILE__                               // (the host pass drops the launch stub over the descriptors)
    constexpr int U = D / 8;                                 // 16-byte units of a key row
    constexpr int KQ = 64 / U;                               // keys per 1 KB request
    constexpr int NQ = (T / KQ + NW - 1) / NW;               // requests per wave and tile, K and V each
    constexpr int TB = T * D * 2;                            // bytes of a tile of K or V
    constexpr int KPW = T / 32 / KW;                         // 32-key blocks per wave
    static_assert(T / KQ % NW == 0, "requests split evenly");
    static_assert(KPW >= 1, "a block per wave");
    __shared__ __align__(1024) uint8_t sm[S * 2 * TB + 16];
    uint32_t* const flag = (uint32_t*)(sm + S * 2 * TB);     // a bad page or length; special values
    const int t = (int)threadIdx.x, lane = t & 63, g = lane >> 5, r = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int rw = wave / KW, kw = wave % KW;
    const int h = (int)(blockIdx.x % (uint32_t)P.Hkv), rg = (int)(blockIdx.x / (uint32_t)P.Hkv % (uint32_t)P.RG);
    const int part = (int)(blockIdx.x / (uint32_t)(P.Hkv * P.RG));
    bool bad = false;
    const int len0 = lane < P.B ? at_len(P, lane, bad) : 0;
    const int64_t share = (int64_t)readfirstlane64((uint64_t)at_share<KeyTiles<T>>(P, len0));
    const int64_t end = (part + 1) * share;
    for (int64_t from = part * share; from < end;) {         // the share's sequences
    int b, len;
    int64_t first;
    if (!at_find<KeyTiles<T>>(P, from, len0, b, len, first)) return;   // uniform: past the last tile
    b = __builtin_amdgcn_readfirstlane(b);
    len = __builtin_amdgcn_readfirstlane(len);
    first = (int64_t)readfirstlane64((uint64_t)first);
    const int nkeys = len + P.N;
    const int64_t last = first + KeyTiles<T>::count(P, len), upto = last < end ? last : end;
    const int64_t je = (upto - first) * T;
    const int j0 = (int)(from - first) * T, j1 = je < nkeys ? (int)je : nkeys;
    const bool whole = from == first && upto >= last - AT_EXTRA;   // the sequence has no other part
    from = upto;
    if (j0 >= nkeys) continue;                               // uniform: nothing of it but the extra tiles
    const int jc = j1 < len ? j1 : len;                      // the part's cached keys end here
    const int nfull = jc > j0 ? (jc - j0) / T : 0;           // tiles of cached keys alone
    __syncthreads();                                         // (the sequence before is done with LDS)
    if (t == 0) {
        bool wrong;
        at_len(P, b, wrong);
        flag[0] = wrong ? 1u : 0u;
        flag[1] = 0u;
    }
    // the wave's rows: node n and query head of row tile rw
    const int row = (rg * P.RT + rw) * 32 + r;
    const bool active = rw < P.RT && (rg * P.RT + rw) * 32 < P.R;   // uniform: the wave has rows
    const int rc = row < P.R ? row : P.R - 1;
    const int n = rc / P.G, hq = h * P.G + rc % P.G;
    // requests: the lane's key of a request and its 16-byte unit of K and V
    const int kq = lane / U, unit = lane % U;
    bool miss = false;
    auto at_k = [&](int i) { return (uint32_t)((unit ^ (((wave + NW * i) * KQ + kq) & (U - 1) & 15)) * 16); };
    auto at_v = [&](int i) { return (uint32_t)((unit ^ ((((wave + NW * i) * KQ + kq) & 3) << 2 & (U - 1))) * 16); };
    // one key's rows, by lane: cached key or drafted token j
    auto issue_key = [&](int i, int j, uint8_t* sk) {
        const uint16_t *kp, *vp;
        if (j < len) {
            int64_t p = b, o = j;
            if (P.table) {                                   // uniform
                const uint32_t e = at_page(P.page_mul, P.page_shift, j);
                o = j - (int)e * P.page;
                int pi = P.table[b * P.ts + e];
                if (pi < 0 || pi >= P.pages) { pi = 0; miss = true; }
                p = pi;
            }
            kp = (const uint16_t*)P.kc + p * P.kcs[0] + o * P.kcs[1] + h * P.kcs[2];
            vp = (const uint16_t*)P.vc + p * P.vcs[0] + o * P.vcs[1] + h * P.vcs[2];
        } else {
            kp = (const uint16_t*)P.k + b * P.ks[0] + (j - len) * P.ks[1] + h * P.ks[2];
            vp = (const uint16_t*)P.v + b * P.vs[0] + (j - len) * P.vs[1] + h * P.vs[2];
        }
        at_dma((const uint8_t*)kp + at_k(i), sk + (wave + NW * i) * 1024);
        at_dma((const uint8_t*)vp + at_v(i), sk + TB + (wave + NW * i) * 1024);
    };
    // the page of key j (uniform), by the scalar unit
    auto page_of = [&](int j) {
        const __attribute__((address_space(4))) int32_t* tab = (const __attribute__((address_space(4))) int32_t*)(P.table + b * P.ts);
        return tab[at_page(P.page_mul, P.page_shift, j)];
    };
    auto base_of = [&](const void* c, const int64_t (&cs)[3], int p, int o) {
        return (void*)((const uint16_t*)c + p * cs[0] + o * cs[1] + h * cs[2]);
    };
    uint32_t ok[NQ], ov[NQ];                                 // the lane's offsets within a tile
#pragma unroll
    for (int i = 0; i < NQ; ++i) {
        const uint32_t key = (uint32_t)((wave + NW * i) * KQ + kq);
        ok[i] = key * (uint32_t)(2 * P.kcs[1]) + at_k(i);
        ov[i] = key * (uint32_t)(2 * P.vcs[1]) + at_v(i);
    }
    auto place = [&](int j, int pi, int& p, int& o) {        // cached key j's page and place in it
        p = b;
        o = j;
        if (P.table) {                                       // uniform
            o = j - (int)at_page(P.page_mul, P.page_shift, j) * P.page;
            const bool out = pi < 0 || pi >= P.pages;
            miss |= out;
            p = out ? 0 : pi;
        }
    };
    int pg = 0;                                              // the page of the next tile to request
    auto lookup = [&](int tile) {
        if (!GEN && P.table && tile < nfull) pg = page_of(j0 + tile * T);   // uniform
    };
    auto issue = [&](int tile, int st) {                     // a tile of cached keys
        uint8_t* const sk = sm + st * 2 * TB;
        const int jt = j0 + tile * T;
        if constexpr (!GEN) {
            int p, o;
            place(jt, pg, p, o);
            const __amdgpu_buffer_rsrc_t rk = __builtin_amdgcn_make_buffer_rsrc(base_of(P.kc, P.kcs, p, o), 0, 0x7FFFFFFF, 0x00027000);
            const __amdgpu_buffer_rsrc_t rv = __builtin_amdgcn_make_buffer_rsrc(base_of(P.vc, P.vcs, p, o), 0, 0x7FFFFFFF, 0x00027000);
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (__attribute__((address_space(3))) void*)(sk + (wave + NW * i) * 1024), 16, (int)ok[i], 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (__attribute__((address_space(3))) void*)(sk + TB + (wave + NW * i) * 1024), 16, (int)ov[i], 0, 0, 0);
            }
        } else if (P.mode == AT_REQUEST) {                   // uniform
#pragma unroll 1
            for (int i = 0; i < NQ; ++i) {
                const int j = jt + (wave + NW * i) * KQ;
                int p, o;
                place(j, P.table ? page_of(j) : 0, p, o);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(base_of(P.kc, P.kcs, p, o), 0, 0x7FFFFFFF, 0x00027000),
                    (__attribute__((address_space(3))) void*)(sk + (wave + NW * i) * 1024), 16, (int)((uint32_t)kq * (uint32_t)(2 * P.kcs[1]) + at_k(i)), 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(__builtin_amdgcn_make_buffer_rsrc(base_of(P.vc, P.vcs, p, o), 0, 0x7FFFFFFF, 0x00027000),
                    (__attribute__((address_space(3))) void*)(sk + TB + (wave + NW * i) * 1024), 16, (int)((uint32_t)kq * (uint32_t)(2 * P.vcs[1]) + at_v(i)), 0, 0, 0);
            }
        } else {
#pragma unroll 1
            for (int i = 0; i < NQ; ++i) issue_key(i, jt + (wave + NW * i) * KQ + kq, sk);
        }
    };
    at_s8 qf[D / 16];
    {
        const uint16_t* qp = (const uint16_t*)P.q + b * P.qs[0] + n * P.qs[1] + hq * P.qs[2] + g * 8;
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {                   // a negative scale's sign goes to q
            qf[s] = *(const at_s8*)(qp + s * 16);
            if (P.flip) qf[s] ^= (short)0x8000;              // uniform
        }
    }
    at_acc o[D / 32];
#pragma unroll
    for (int d = 0; d < D / 32; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.0f;
    float m = -__builtin_inff(), l = 0.0f;
    // The products and the softmax of a staged tile.  Bit j of bits: the lane's
    // row sees the tile's key j; ALL: it sees every one.
    auto math = [&](const uint8_t* sk, auto all, uint64_t bits) __attribute__((always_inline)) {
        constexpr bool ALL = decltype(all)::value;
        at_acc s[KPW];
#pragma unroll
        for (int kb = 0; kb < KPW; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[kb][i] = 0.0f;
        // four pieces of K at a time, read while the four before are multiplied
        constexpr int NG = KPW * D / 64;
        at_s8 kf[2][4];
        auto kread = [&](int e) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int kt = (kw * KPW + e * 4 / (D / 16)) * 32 + r, d = e * 4 % (D / 16) + i;   // the lane's key row
                kf[e & 1][i] = *(const at_s8*)(sk + kt * (D * 2) + (((2 * d + g) ^ (r & (U - 1) & 15)) << 4));
            }
        };
        kread(0);
#pragma unroll
        for (int e = 0; e < NG; ++e) {
            if (e + 1 < NG) kread(e + 1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int i = 0; i < 4; ++i) s[e * 4 / (D / 16)] = at_mfma<DT>(kf[e & 1][i], qf[e * 4 % (D / 16) + i], s[e * 4 / (D / 16)]);
            __builtin_amdgcn_sched_barrier(0);
        }
        uint32_t va[4];                                      // V: the lane's places of four column blocks
        {
            const uint32_t base = (uint32_t)(uintptr_t)(const __attribute__((address_space(3))) uint8_t*)sk + TB +
                                  (uint32_t)((kw * KPW * 32 + 4 * g + (lane >> 2 & 3)) * (D * 2) + (lane >> 4 & 1) * 32 + (lane & 3) * 8);
#pragma unroll
            for (int d = 0; d < 4; ++d) va[d] = base + (uint32_t)(((d * 4) ^ ((lane >> 2 & 3) << 2 & (U - 1))) * 16);
        }
        float mt = -__builtin_inff();
#pragma unroll
        for (int kb = 0; kb < KPW; ++kb)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                if constexpr (!ALL) {
                    const float x = s[kb][i] * P.scale2;
                    const uint32_t w = (uint32_t)(bits >> ((kw * KPW + kb) * 32)) >> (4 * g);
                    s[kb][i] = w >> ((i & 3) + 8 * (i >> 2)) & 1u ? x : -__builtin_inff();
                }
                mt = __builtin_fmaxf(mt, s[kb][i]);
            }
        mt = __builtin_fmaxf(mt, __shfl_xor(mt, 32, 64));
        if constexpr (ALL) mt *= P.scale2;                   // scale2 >= 0
        const float mn = __builtin_fmaxf(m, mt);
        const float mu = mn > -__builtin_inff() ? mn : 0.0f;
        const float mup = DT == LLIMA_F16 ? mu - 10.0f : mu;
        if (__any(mn > m)) {                                 // else the factor is 1 for every row
            const float a = __builtin_amdgcn_exp2f(m - mu);
            l *= a;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= a;
            m = mn;
        }
#pragma unroll
        for (int kb = 0; kb < KPW; ++kb) {
            float ls = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[kb][i] = __builtin_amdgcn_exp2f(ALL ? __builtin_fmaf(s[kb][i], P.scale2, -mup) : s[kb][i] - mup);
                ls += s[kb][i];
            }
            l += ls;
#pragma unroll
            for (int st = 0; st < 2; ++st) {                 // 16 keys of the block
                uint32_t pw[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) pw[e] = at_pack<DT>(s[kb][8 * st + 2 * e], s[kb][8 * st + 2 * e + 1]);
                const at_s8 pf = __builtin_bit_cast(at_s8, (llima_u32x4){pw[0], pw[1], pw[2], pw[3]});
                // element e of half g is key 16 st + e % 4 + 8 (e / 4) + 4 g: a
                // transposing load takes 4 keys by 16 columns from 16 lanes
                at_s4 v[D / 32][2];
                if (kb == 0 && st == 0) at_vread<D, 0>(va, v);
                else if (kb == 0) at_vread<D, 16>(va, v);
                else if (st == 0) at_vread<D, 32>(va, v);
                else at_vread<D, 48>(va, v);
#pragma unroll
                for (int d = 0; d < D / 32; ++d)
                    o[d] = at_mfma<DT>(__builtin_shufflevector(v[d][0], v[d][1], 0, 1, 2, 3, 4, 5, 6, 7), pf, o[d]);
            }
        }
    };
    auto seen = [&](int mm) {                                // the lane's row sees drafted token mm
        if (!P.mask) return mm <= n;
        if (P.mask_f32) return ((const float*)P.mask)[b * P.ms[0] + n * P.ms[1] + mm] > 0.0f;
        return ((const uint8_t*)P.mask)[b * P.ms[0] + n * P.ms[1] + mm] != 0;
    };
    const int ntile = (j1 - j0 + T - 1) / T;
    // a tile of the part; past the last one that again, which nobody reads
    auto request = [&](int tile, int st) {
        const int tl = tile < ntile ? tile : ntile - 1;
        if (tl < nfull) {                                    // uniform
            issue(tl, st);
        } else {
            uint8_t* const sk = sm + st * 2 * TB;
#pragma unroll 1
            for (int i = 0; i < NQ; ++i) {
                const int j = j0 + tl * T + (wave + NW * i) * KQ + kq;   // past the part's end: its last key
                issue_key(i, j < j1 ? j : j1 - 1, sk);
            }
        }
        if (tile + 1 < nfull) lookup(tile + 1);
    };
    lookup(0);
#pragma unroll 1
    for (int e = 0; e < S - 1; ++e) request(e, e);
    int tile = 0;
    for (; tile < nfull; ++tile) {
        at_wait_barrier<(S - 2) * 2 * NQ>();                 // the tile has landed, and the last one is read
        request(tile + S - 1, (tile + S - 1) % S);
        if (active) math(sm + (tile % S) * 2 * TB, std::integral_constant<bool, true>{}, 0ull);
    }
    for (; tile < ntile; ++tile) {                           // the tiles with a mask
        const int jt = j0 + tile * T, je = jt + T < j1 ? jt + T : j1;
        uint8_t* const sk = sm + (tile % S) * 2 * TB;
        uint64_t bits = 0;
        if (active) {                                        // uniform
            // the cached keys, and with no mask the drafted ones up to n
            auto below = [&](int j) {                        // the tile's keys below j
                const int c = j - jt;
                return c <= 0 ? 0ull : c >= 64 ? ~0ull : (1ull << c) - 1;
            };
            bits = below(P.mask ? (len < je ? len : je) : (len + n + 1 < je ? len + n + 1 : je));
            if (P.mask)                                      // uniform
                for (int j = jt > len ? jt : len; j < je; j += 8) {
                    bool v[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = seen((j + e < je ? j + e : je - 1) - len);
#pragma unroll
                    for (int e = 0; e < 8; ++e) bits |= j + e < je && v[e] ? 1ull << (j + e - jt) : 0ull;
                }
        }
        at_wait_barrier<(S - 2) * 2 * NQ>();
        request(tile + S - 1, (tile + S - 1) % S);
        // Values that not every row sees: rows past the end become 0, and so do
        // infinities and NaN of drafted tokens (0 times them would be NaN for the
        // rows that do not see them; at the end they are added to the rows that do).
        const int clean = jc - jt > 0 ? jc - jt : 0;         // the tile's cached keys
        for (int p = clean * U + t; p < T * U; p += 64 * NW) {
            const int j = jt + p / U;
            llima_u32x4* const at = (llima_u32x4*)(sk + TB + p * 16);
            llima_u32x4 x = *at;
            bool put = j >= j1;
            if (put) x = (llima_u32x4){0u, 0u, 0u, 0u};
            if (!put && j >= len) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    uint32_t w = x[e];
                    if (at_special<DT>((uint16_t)w)) { w &= 0xFFFF0000u; put = true; flag[1] = 1u; }
                    if (at_special<DT>((uint16_t)(w >> 16))) { w &= 0xFFFFu; put = true; flag[1] = 1u; }
                    x[e] = w;
                }
            }
            if (put) *at = x;
        }
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        if (active) math(sk, std::integral_constant<bool, false>{}, bits);
    }
    if (miss) flag[0] = 1u;
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // no request outlives this
    __syncthreads();
    l += __shfl_xor(l, 32, 64);
    if constexpr (KW > 1) {                                  // the second half of the keys joins the first
        float* const red = (float*)sm + (size_t)rw * 64 * (D / 2 + 2);
        static_assert(NW / KW * 64 * (D / 2 + 2) * 4 <= S * 2 * TB, "room for the second halves");
        if (active && kw == 1) {
            red[lane] = m;
            red[64 + lane] = l;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) red[(2 + d * 16 + i) * 64 + lane] = o[d][i];
        }
        __syncthreads();
        if (active && kw == 0) {
            const float m2 = red[lane], mn = __builtin_fmaxf(m, m2), mu = mn > -__builtin_inff() ? mn : 0.0f;
            const float a = __builtin_amdgcn_exp2f(m - mu), a2 = __builtin_amdgcn_exp2f(m2 - mu);
            m = mn;
            l = l * a + red[64 + lane] * a2;
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] = o[d][i] * a + red[(2 + d * 16 + i) * 64 + lane] * a2;
        }
    }
    if (!active || row >= P.R || kw != 0) continue;
    const AttnArgs A = at_args();
    if (flag[1]) {                                           // infinities and NaN of drafted tokens in this part
        for (int mm = (j0 > len ? j0 : len) - len; mm < j1 - len; ++mm) {
            if (!seen(mm)) continue;                         // (of the loop over mm)
            const uint16_t* vp = (const uint16_t*)A->v + b * A->vs[0] + mm * A->vs[1] + h * A->vs[2];
#pragma unroll
            for (int d = 0; d < D / 32; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4) {
                    const uint2 w = *(const uint2*)(vp + d * 32 + 2 * i + 4 * g);
                    auto add = [&](int e, uint32_t x) { o[d][e] += at_special<DT>((uint16_t)x) ? at_f32<DT>((uint16_t)x) : 0.0f; };
                    add(i, w.x); add(i + 1, w.x >> 16); add(i + 2, w.y); add(i + 3, w.y >> 16);
                }
        }
    }
    if (flag[0]) l = __builtin_nanf("");
    if (whole) {
        const float inv = at_inverse(A, l, b, n, len);
        uint16_t* op = (uint16_t*)A->out + b * A->os[0] + n * A->os[1] + hq * A->os[2] + 4 * g;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(uint2*)(op + d * 32 + 2 * i) = make_uint2(at_pack<DT>(o[d][i] * inv, o[d][i + 1] * inv),
                                                            at_pack<DT>(o[d][i + 2] * inv, o[d][i + 3] * inv));
    } else {
        const size_t at = ((size_t)at_slot(A->pairs, part, b, j0 == 0) * A->Hkv + h) * A->R + row;
        if (g == 0) A->part_ml[at] = make_float2(m, l);
        float* op = A->part_o + at * D + 4 * g;
#pragma unroll
        for (int d = 0; d < D / 32; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *(float4*)(op + d * 32 + 2 * i) = make_float4(o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
    }
    }
#endif
}

struct CommitParams {
    const uint8_t *k, *v;
    uint8_t *kc, *vc;
    const int32_t *nodes, *counts, *lens, *table;
    int32_t* new_lens;
    int64_t ks[4], vs[4];                                    // layer, batch, node and head strides (bytes)
    int64_t kcs[4], vcs[4];                                  // layer, page, token and head strides
    int64_t ns, ts, cap;
    int32_t B, N, L, Hkv, U;                                 // U: 16-byte units of a head's row
    int32_t page, pages;
};

// One workgroup per path place, sequence and `per` layers (8 at most): checks
// the sequence's path and room (every workgroup of a sequence comes to the same
// answer), then copies one token's K and V rows, all layers' loads in flight together.
__global__ __launch_bounds__(LLIMA_WG) void tree_commit(CommitParams P, int layers, int per) {
    const int j = (int)(blockIdx.x % (uint32_t)P.L), b = (int)(blockIdx.x / (uint32_t)P.L), t = (int)threadIdx.x;
    const int l0 = (int)blockIdx.y * per, nl = layers - l0 < per ? layers - l0 : per;
    const int len = P.lens[b], cnt = P.counts[b];
    bool ok = len >= 0 && cnt >= 0 && cnt <= P.L && len <= P.cap && (int64_t)len + cnt <= P.cap;
    if (ok) {
        bool all = true;
        for (int i = t & 63; i < cnt; i += 64) {
            const int node = P.nodes[b * P.ns + i];
            all = all && node >= 0 && node < P.N;
            if (P.table) {
                const int p = P.table[b * P.ts + (uint32_t)(len + i) / (uint32_t)P.page];
                all = all && p >= 0 && p < P.pages;
            }
        }
        ok = __all(all);
    }
    if (j == 0 && l0 == 0 && t == 0) P.new_lens[b] = ok ? len + cnt : LLIMA_E_RANGE;
    if (!ok || j >= cnt) return;                             // uniform
    const int64_t node = P.nodes[b * P.ns + j];
    int64_t p = b, o = len + j;
    if (P.table) {
        p = P.table[b * P.ts + (uint32_t)(len + j) / (uint32_t)P.page];
        o = (uint32_t)(len + j) % (uint32_t)P.page;
    }
    const int n = P.Hkv * P.U;
    for (int i = t; i < 2 * n; i += LLIMA_WG) {
        const bool isv = i >= n;
        const int e = isv ? i - n : i, h = e / P.U, u = e % P.U;
        const int64_t* fs = isv ? P.vs : P.ks;
        const int64_t* ts = isv ? P.vcs : P.kcs;
        const uint8_t* src = (isv ? P.v : P.k) + l0 * fs[0] + b * fs[1] + node * fs[2] + h * fs[3] + u * 16;
        uint8_t* dst = (isv ? P.vc : P.kc) + l0 * ts[0] + p * ts[1] + o * ts[2] + h * ts[3] + u * 16;
        llima_u32x4 x[8];
#pragma unroll
        for (int l = 0; l < 8; ++l)
            if (l < nl) x[l] = *(const llima_u32x4*)(src + l * fs[0]);   // uniform
#pragma unroll
        for (int l = 0; l < 8; ++l)
            if (l < nl) *(llima_u32x4*)(dst + l * ts[0]) = x[l];
    }
}

// Shares of the keys: as many workgroups as the device holds at a time, two per
// CU, or one of those that take more than half of its LDS.
static int at_parts(int Hkv, int RG, int RT, int D) {
    const int n = (RT > 4 || (D == 256 && RT > 2) ? 256 : 512) / (Hkv * RG);
    return n < 1 ? 1 : n;
}

static int at_row_tiles(int R, int& RG) {                    // row tiles of a group, groups
    const int rt = (R + 31) / 32;
    RG = (rt + 7) / 8;
    return (rt + RG - 1) / RG;
}

template <int DT, int D, bool GEN>
static void at_launch(const AttnParams& P, hipStream_t st) {
    const dim3 g((uint32_t)P.parts * P.RG * P.Hkv);
    constexpr int T = D == 256 ? 32 : 64, K2 = D == 256 ? 1 : 2;
    constexpr int S2 = D == 64 ? 4 : 2, S4 = D == 256 ? 4 : S2, S8 = 4;
    if (P.RT <= (K2 == 2 ? 1 : 2)) {
        hipLaunchKernelGGL((tree_attn<DT, D, 2, K2, T, S2, GEN>), g, dim3(128), 0, st, P);
    } else if (P.RT <= 4) {
        if constexpr (K2 == 2) {
            if (P.RT <= 2) hipLaunchKernelGGL((tree_attn<DT, D, 4, 2, T, S4, GEN>), g, dim3(256), 0, st, P);
        }
        if (K2 == 1 || P.RT > 2) hipLaunchKernelGGL((tree_attn<DT, D, 4, 1, T, S4, GEN>), g, dim3(256), 0, st, P);
    } else {
        hipLaunchKernelGGL((tree_attn<DT, D, 8, 1, T, S8, GEN>), g, dim3(512), 0, st, P);
    }
    const int64_t rows = (int64_t)P.B * P.N * P.Hq;
    if (rows <= 1024) hipLaunchKernelGGL((tree_attn_join<DT, D, KeyTiles<T>, 4>), dim3((uint32_t)rows), dim3(LLIMA_WG), 0, st, P);
    else hipLaunchKernelGGL((tree_attn_join<DT, D, KeyTiles<T>, 1>), dim3((uint32_t)((rows + 3) / 4)), dim3(LLIMA_WG), 0, st, P);
}

template <int DT>
static int at_dispatch(const AttnParams& P, int D, hipStream_t st) {
    const bool gen = P.mode != AT_TILE;
    if (D == 64) gen ? at_launch<DT, 64, true>(P, st) : at_launch<DT, 64, false>(P, st);
    else if (D == 128) gen ? at_launch<DT, 128, true>(P, st) : at_launch<DT, 128, false>(P, st);
    else gen ? at_launch<DT, 256, true>(P, st) : at_launch<DT, 256, false>(P, st);
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}

}  // namespace llima

using namespace llima;


static void at_plan(AttnParams& P, int D) {
    P.R = P.N * P.G;
    P.RT = at_row_tiles(P.R, P.RG);
    P.parts = at_parts(P.Hkv, P.RG, P.RT, D);
    at_slots(P);
}

extern "C" size_t llima_tree_attention_workspace_bytes(int32_t B, int32_t N, int32_t Hq,
                                                       int32_t Hkv, int32_t D) {
    if (B <= 0 || !at_sizes_ok(B, N, Hq, Hkv, D)) return 0;
    AttnParams P = {};
    P.B = B; P.N = N; P.Hkv = Hkv; P.G = Hq / Hkv;
    at_plan(P, D);
    return at_parts_bytes(P, D);
}

extern "C" int llima_tree_attention(const llima_tree_attention_args* a, void* workspace,
                                    size_t workspace_bytes, void* stream) {
    AttnParams P = {};
    const int ok = at_fill(a, 8, P);
    if (ok != LLIMA_OK || a->B == 0) return ok;
    if (!workspace || workspace_bytes < llima_tree_attention_workspace_bytes(a->B, a->N, a->Hq, a->Hkv, a->D))
        return LLIMA_E_WORKSPACE;
    if ((uintptr_t)workspace % 16) return LLIMA_E_INVAL;
    // offsets within a tile (64 keys) or a request have 31 bits
    const int64_t ts = P.kcs[1] > P.vcs[1] ? P.kcs[1] : P.vcs[1];
    P.mode = ts <= (1 << 23) && (!P.table || P.page % 64 == 0) ? AT_TILE
           : ts <= (1 << 26) && (!P.table || P.page % 8 == 0) ? AT_REQUEST : AT_LANE;
    at_plan(P, a->D);
    at_parts_at(P, a->D, workspace);
    return a->dtype == LLIMA_BF16 ? at_dispatch<LLIMA_BF16>(P, a->D, (hipStream_t)stream)
                                  : at_dispatch<LLIMA_F16>(P, a->D, (hipStream_t)stream);
}

extern "C" int llima_tree_commit(const llima_tree_commit_args* a, void* stream) {
    if (!a || a->layers <= 0 || a->layers > 65535 || a->B < 0 || a->N <= 0 || a->L <= 0 || a->Hkv <= 0 || a->D <= 0)
        return LLIMA_E_INVAL;
    if (a->D % 8 != 0 || a->D > 65536 || a->Hkv > 65536 || (int64_t)a->Hkv * a->D > (1 << 24)) return LLIMA_E_INVAL;
    if (a->page_size <= 0 || a->pages < 0 || a->max_blocks < 0) return LLIMA_E_INVAL;
    if (!a->block_table && (a->pages < a->B || a->max_blocks != 1)) return LLIMA_E_INVAL;
    if ((int64_t)a->page_size * a->max_blocks > (int64_t)INT32_MAX) return LLIMA_E_INVAL;
    if ((int64_t)a->B * a->L >= (1 << 24)) return LLIMA_E_INVAL;   // (the launch: fewer than 2^32 threads)
    if (!at_strides_ok(a->k_strides, 4, 8) || !at_strides_ok(a->v_strides, 4, 8) || !at_strides_ok(a->k_cache_strides, 4, 8) ||
        !at_strides_ok(a->v_cache_strides, 4, 8) || a->nodes_stride < 0 || (a->block_table && a->table_stride < 0))
        return LLIMA_E_INVAL;
    if (a->B == 0) return LLIMA_OK;
    const bool cached = a->pages > 0 && a->max_blocks > 0;
    if (!a->nodes || !a->counts || !a->cache_lens || !a->new_lens) return LLIMA_E_INVAL;
    if (!a->k || !a->v || (cached && (!a->k_cache || !a->v_cache))) return LLIMA_E_INVAL;
    const void* ptrs[] = {a->k, a->v, a->k_cache, a->v_cache};
    for (const void* p : ptrs)
        if ((uintptr_t)p % 16) return LLIMA_E_INVAL;
    CommitParams P = {};
    P.k = (const uint8_t*)a->k; P.v = (const uint8_t*)a->v;
    P.kc = (uint8_t*)a->k_cache; P.vc = (uint8_t*)a->v_cache;
    P.nodes = a->nodes; P.counts = a->counts; P.lens = a->cache_lens; P.table = a->block_table;
    P.new_lens = a->new_lens;
    for (int i = 0; i < 4; ++i) {
        P.ks[i] = 2 * a->k_strides[i]; P.vs[i] = 2 * a->v_strides[i];
        P.kcs[i] = 2 * a->k_cache_strides[i]; P.vcs[i] = 2 * a->v_cache_strides[i];
    }
    P.ns = a->nodes_stride; P.ts = a->table_stride;
    P.cap = a->pages > 0 ? (int64_t)a->page_size * a->max_blocks : 0;
    P.B = a->B; P.N = a->N; P.L = a->L; P.Hkv = a->Hkv; P.U = a->D / 8;
    P.page = a->page_size; P.pages = a->pages;
    // a layer to a workgroup where there are few, 8 where they fill the device (one / 8
    // layers: 1280 and 4096 tokens' layers 17.1 / 17.0 us and 17.3 / 17.2, 8192 19.1 / 17.3,
    // 16384 33.1 / 19.7)
    const int per = (int64_t)a->B * a->L * a->layers <= 2048 ? 1 : 8;
    hipLaunchKernelGGL(tree_commit, dim3((uint32_t)(a->B * a->L), (uint32_t)((a->layers + per - 1) / per)),
                       dim3(LLIMA_WG), 0, (hipStream_t)stream, P, a->layers, per);
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}
