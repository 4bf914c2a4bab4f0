// lmhead_fp8.hpp -- the LM head over an 8-bit weight: e4m3 values with an fp32
// scale per block of 128 (included by lmhead.hip, whose epilogue and finish
// kernels it shares).
//
//   s[b][v] = sum over kb of (xs[b][kb] ws[v / 128][kb]) p,
//   p       = sum over the block's k of xq[b][k] wq[v][k]
//
// p is one block's sum in the matrix core, scaled and added in fp32; then
// softcap, rounding and argmax as the bf16 head (lmh_logit).  The values go into
// the matrix core as bf16, which holds every e4m3 value: its 8-bit instructions
// are twice as fast but drop low bits of the products when they add them (128
// products of values from N(0, 60^2): off by 2^-16 of the terms' magnitude at
// most, by 2^-12 where one product in 64 is 2^11 times the others; the bf16
// instructions 2^-25 and 2^-22), which is not a sum in 32 bits.  xq [B][H] and
// xs [B][NK] are a hidden row's values and scales, wq [V][H] and ws [ceil(V/128)][NK]
// the weight's, NK = ceil(H/128).
#pragma once

// Eight e4m3 values as bf16 (exact; NaN stays NaN).
__device__ __forceinline__ lmh_b8 lmh8_wide(uint32_t lo, uint32_t hi) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    const b2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, false);
    const b2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(lo, 1.0f, true);
    const b2 c = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, false);
    const b2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(hi, 1.0f, true);
    return (lmh_b8){a.x, a.y, b.x, b.y, c.x, c.y, d.x, d.y};
}

struct Lmh8Params {
    LmhParams P;
    const uint8_t* xq;
    const float* xs;
    const uint8_t* wq;
    const float* ws;
    int32_t NK;
};

// NX sums of one lane as the argmax sees them (lmh_logit), in place.
template <int NX>
__device__ __forceinline__ void lmh8_logits(const LmhParams& P, float (&x)[NX]) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    typedef __bf16 h2 __attribute__((ext_vector_type(2)));
    if (P.cap > 0.0f) {                                      // uniform
#pragma unroll
        for (int k = 0; k < NX; ++k) {
            x[k] = P.cap * tanhf(x[k] / P.cap);
            if (NX > 16) __builtin_amdgcn_sched_barrier(0);  // one at a time: interleaved, they spill
        }
    }
    if (P.round_bf16) {                                      // uniform
#pragma unroll
        for (int k = 0; k < NX; k += 2) {
            const f2 v = {x[k], x[k + 1]};
            const uint32_t u = __builtin_bit_cast(uint32_t, __builtin_convertvector(v, h2));
            x[k] = __uint_as_float(u << 16);
            x[k + 1] = __uint_as_float(u & 0xFFFF0000u);
        }
    }
}

// What a lane keeps of its hidden row over the tiles of its wave: the best key
// (both lanes of the pair the same), and with SC the sum of exp(logit - m), m
// its greatest non-NaN logit (each lane its own half of the rows).
struct Lmh8Best {
    uint64_t key;
    float m, s;
};

// 2 NX vocab rows from n of one hidden row per lane pair (r, 0), (r, 1): x[k]
// of lane half g is row n + (k / 16) 32 + (k / 4 % 4) 8 + 4 g + k % 4.  Writes the
// logits when asked, and with SC the target's logit.  b: the hidden row (row
// false: none); end: the first row that is not the tile's.
template <int NX, bool SC>
__device__ __forceinline__ void lmh8_slot_out(const LmhParams& P, float (&x)[NX], Lmh8Best& B, int b,
                                              bool row, int n, int end, int g) {
    const int left = end - n;                                // <= 0: nothing
    auto col = [&](int k) { return (k >> 4) * 32 + (k >> 2 & 3) * 8 + 4 * g + (k & 3); };
    lmh8_logits<NX>(P, x);
    if (P.out_logits) {                                      // uniform
        const bool wide = ((uintptr_t)P.out_logits & 15u) == 0 && P.V % 4 == 0;
        const size_t at = (size_t)(row ? b : 0) * P.V + n;
        if (P.logits_bf16) {
            auto h = [](float v) { return v == v ? __float_as_uint(v) >> 16 : 0x7FC0u; };
            uint16_t* o = (uint16_t*)P.out_logits + at;
#pragma unroll
            for (int k = 0; k < NX; k += 4) {
                if (row && wide && col(k) < left) {
                    *(uint2*)(o + col(k)) = make_uint2(h(x[k]) | h(x[k + 1]) << 16, h(x[k + 2]) | h(x[k + 3]) << 16);
                } else if (row && !wide) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col(k + e) < left) o[col(k + e)] = (uint16_t)h(x[k + e]);
                }
            }
        } else {
            float* o = P.out_logits + at;
#pragma unroll
            for (int k = 0; k < NX; k += 4) {
                if (row && wide && col(k) < left) {
                    *(float4*)(o + col(k)) = make_float4(x[k], x[k + 1], x[k + 2], x[k + 3]);
                } else if (row && !wide) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col(k + e) < left) o[col(k + e)] = x[k + e];
                }
            }
        }
    }
    if (left < 2 * NX) {                                     // uniform: rows past the tile
#pragma unroll
        for (int k = 0; k < NX; ++k) x[k] = col(k) < left ? x[k] : __builtin_nanf("");
    }
    // the greatest of the two lanes' logits (NaN only when all are), and its first row
    float best = lmh_max3(x[0], x[1], x[1]);
#pragma unroll
    for (int k = 2; k < NX; k += 2) best = lmh_max3(best, x[k], x[k + 1]);
    const float own = best;
    best = lmh_max3(best, __shfl_xor(best, 32, 64), best);
    int at = 255;
#pragma unroll
    for (int k = NX - 1; k >= 0; --k) at = x[k] == best ? (k >> 4) * 32 + (k >> 2 & 3) * 8 + (k & 3) : at;
    at = at == 255 ? 255 : at + 4 * g;
    const int other = __shfl_xor(at, 32, 64);
    at = at < other ? at : other;
    const uint64_t key = at < 255 ? ((uint64_t)f32_key(best) << 32) | (uint32_t)~(uint32_t)(n + at) : 0ull;
    B.key = key > B.key ? key : B.key;
    if constexpr (SC) {
        const int32_t tg = row ? P.targets[b] : -1;
        if (left < 2 * NX) {                                 // uniform
#pragma unroll
            for (int k = 0; k < NX; ++k) x[k] = col(k) < left ? x[k] : -__builtin_inff();
        }
        const float mn = own > B.m ? own : B.m;              // (own NaN: all of them, the sum becomes NaN)
        const float mw = mn > -__builtin_inff() ? mn : 0.0f;
        float e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < NX; ++k) e[k & 3] += __builtin_amdgcn_exp2f((x[k] - mw) * LMH_LOG2E);
        const float old = B.m > -__builtin_inff() ? B.s * __builtin_amdgcn_exp2f((B.m - mw) * LMH_LOG2E) : B.s;
        B.s = old + ((e[0] + e[1]) + (e[2] + e[3]));
        B.m = mn;
        const int ts = tg >= 0 ? tg - n : -1;                // the target's column of the slot
        const bool hit = ts >= 0 && ts < 2 * NX && ts < left && (ts >> 2 & 1) == g;
        if (__any(hit)) {
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < NX; ++k) v = ts == col(k) ? x[k] : v;
            if (hit) P.tval[b] = v;
        }
    }
}

// lmh8_tiles: up to 32 CWV MB hidden rows in a pass.  A workgroup of eight waves
// (two per SIMD: one alone issues a vector instruction every nine cycles, two
// together every 4.6), one workgroup per CU, takes tiles of 256 vocab rows (tile,
// tile + grid, ...), RWV waves along the vocab rows (VB blocks of 32 each) and CWV
// along the hidden rows (MB blocks of 32).  k goes in steps of one block of 128
// ids: 128 bytes of each weight row and of each hidden row are requested
// straight into a ring of S LDS slots.  LDS rows are 128 bytes with their 16-byte
// columns exchanged by row / 2 (the request's source address does it): fragment
// reads have no bank conflicts.  The scales are loaded a step ahead, before the
// requests, so that waiting for them leaves those in flight (with requests made by
// global loads the compiler takes them to return in any order and waits for all).  A
// step's values are read, converted and multiplied piece by piece (piece e of half g:
// ids 32 e + 16 g .. + 15, its halves two MFMAs), its sums scaled and added to the
// tile's.  The weight is the MFMA's row operand: lane (r, g) has, for hidden row r of a
// block, half of a wave's vocab rows (the lane with the other g the other half).
//
// The order of a sum may not depend on where its vocab row lies, or equal rows would get
// logits that differ in their last bits and the greater id could win.  But workgroups that
// all start their tiles at the first block of k read the same 128 bytes of every 4 KB, which
// is a part of the memory channels.  So the blocks stand in 2^K groups, each summed from its
// first block on, and the groups' sums are added in pairs, then the pairs': every order
// q ^ rot of the groups adds the same two values in one order or the other, and workgroups
// start at different groups.  K = 2 from H = 4096 on, up to 64 rows (V 128256, from block 0 /
// K = 2: 1 row of 4096 ids 114 / 94 us, 64 rows 123 / 112, 1 row of 8192 230 / 181).  Narrower
// rows lie apart by themselves (V 152064, 3584 ids, 1 row 105 / 107, 64 rows 125 / 129; V 32000,
// 512 ids 9.6 / 10.4), and above 64 rows the waiting sums' registers are not there (K = 1 at
// 128 rows: 154 -> 176 us) and reading bounds less: K = 0, from block 0 on, the last pass of
// such a batch too.
//
// Shapes <RWV, VB, CWV, MB, S>: <8, 1, 1, 1, 4> up to 32 rows, <4, 2, 2, 1, 4> up to 64,
// <4, 2, 2, 2, 3> up to 128, and larger batches in passes of 128.  The waves' split along the
// hidden rows halves what each converts of the weight; along the vocab rows alone
// (8 waves) the LDS reads bound (64 / 128 rows 130 / 199 us, this 101 / 151 in that build).
//
// Bound: reading the weight up to 64 rows (H 4096, V 128256, 0.53 GB: 1 row 94 us,
// 32 rows 96, 64 106-112; the requests alone 88), from 128 on (155-160, 500 rows 630) the issue
// of the vector instructions that widen, scale and add.  256 registers: 33 to 64 rows spill 3
// (10 with SC), 65 and more 4 (19).
#define LMH8_NV 256                    // vocab rows per tile
#define LMH8_CUS 256                   // workgroups: one per CU (its LDS)

template <int RWV, int VB, int CWV, int MB, int S, int K, bool SC>
__global__ __launch_bounds__(512) void lmh8_tiles(Lmh8Params Q, int b0, int nb) {
    constexpr int NM = 32 * CWV * MB;                        // hidden rows of the pass
    constexpr int LW = LMH8_NV / 64;                         // 1 KB requests per wave and step: weight,
    constexpr int LX = NM >= 64 ? NM / 64 : 1;               // hidden rows (NM = 32: half of the waves' again)
    constexpr int WB = LMH8_NV * 128, SB = WB + NM * 128;    // bytes of a slot
    static_assert(RWV * CWV == 8 && RWV * VB * 32 == LMH8_NV && S >= 2 && S * SB <= 163840, "shape");
    __shared__ __align__(1024) uint8_t sm[S * SB];
    const LmhParams& P = Q.P;
    const int t = (int)threadIdx.x, lane = t & 63, g = lane >> 5, r = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int wr = wave % RWV, wc = wave / RWV;
    const int H = P.H, V = P.V, NK = Q.NK, G = (int)gridDim.x;
    const int ntile = (V + LMH8_NV - 1) / LMH8_NV;           // grid <= ntile
    constexpr int NG = 1 << K;                               // groups of blocks; NK >= NG
    const int rot = (int)(blockIdx.x >> 3) & (NG - 1);       // they are taken in the order q ^ rot
    auto start = [&](int q) { return (q * NK) >> K; };       // group q's first block
    // The request stream: a tile and a block of it.  Through buffer descriptors:
    // rows past the vocabulary or the batch lie outside them and read as 0, as
    // does what the last row's last block has past H (other rows read the next
    // row's there; it is not used).
    uint32_t ow[LW], ox[LX];                                 // the lane's row and column of its requests
#pragma unroll
    for (int q = 0; q < LW; ++q) {
        const int row = 8 * (wave + 8 * q) + (lane >> 3);
        ow[q] = (uint32_t)row * (uint32_t)H + (uint32_t)(((lane & 7) ^ (row >> 1 & 7)) * 16);
    }
#pragma unroll
    for (int q = 0; q < LX; ++q) {
        const int row = 8 * ((wave + 8 * q) % (NM / 8)) + (lane >> 3);
        ox[q] = (uint32_t)row * (uint32_t)H + (uint32_t)(((lane & 7) ^ (row >> 1 & 7)) * 16);
    }
    const __amdgpu_buffer_rsrc_t rx = __builtin_amdgcn_make_buffer_rsrc((void*)(Q.xq + (size_t)b0 * H), 0, nb * H, 0x00027000);
    int tw = (int)blockIdx.x, qw = 0, cw = start(rot), ew = start(rot + 1), sw = 0;
    auto issue = [&]() {
        const int rows = V - tw * LMH8_NV < LMH8_NV ? V - tw * LMH8_NV : LMH8_NV;
        const __amdgpu_buffer_rsrc_t rw = __builtin_amdgcn_make_buffer_rsrc((void*)(Q.wq + (size_t)tw * LMH8_NV * H), 0, rows * H, 0x00027000);
        uint8_t* const at = sm + sw * SB;
#pragma unroll
        for (int q = 0; q < LX; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rx, (__attribute__((address_space(3))) void*)(at + WB + ((wave + 8 * q) % (NM / 8)) * 1024),
                                                     16, (int)ox[q], cw * 128, 0, 0);
#pragma unroll
        for (int q = 0; q < LW; ++q)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(rw, (__attribute__((address_space(3))) void*)(at + (wave + 8 * q) * 1024),
                                                     16, (int)ow[q], cw * 128, 0, 0);
        sw = sw + 1 == S ? 0 : sw + 1;
        if (++cw == ew) {                                    // uniform
            if (++qw == NG) {
                qw = 0;
                if (tw + G < ntile) tw += G;                 // past its last tile: that again
            }
            cw = start(qw ^ rot);
            ew = start((qw ^ rot) + 1);
        }
    };
    int m[MB], mc[MB];                                       // the lane's hidden rows of the pass
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        m[i] = (wc * MB + i) * 32 + r;
        mc[i] = m[i] < nb ? m[i] : nb - 1;
    }
    float sx[MB], swt;                                       // the next step's scales
    auto load_s = [&](int tile, int c) {
        const int vb = tile * 2 + (wr * VB * 32) / 128;      // the block of 128 vocab rows of the wave
        swt = Q.ws[(size_t)(vb * 128 < V ? vb : 0) * NK + c];
#pragma unroll
        for (int i = 0; i < MB; ++i) sx[i] = Q.xs[(size_t)(b0 + mc[i]) * NK + c];
    };
    int slot = 0;
    float acc[MB][VB][16];
    Lmh8Best best[MB];
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        best[i] = {0ull, -__builtin_inff(), 0.0f};
#pragma unroll
        for (int v = 0; v < VB; ++v)
#pragma unroll
            for (int k = 0; k < 16; ++k) acc[i][v][k] = 0.0f;
    }
    load_s((int)blockIdx.x, start(rot));
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int i = 0; i < S - 1; ++i) issue();
    const uint32_t rl = (uint32_t)(r * 128), rz = (uint32_t)(r >> 1 & 7);
    for (int tile = (int)blockIdx.x; tile < ntile; tile += G) {
        float low[K > 0 ? K : 1][MB][VB][16];                // sums of groups that wait for their counterpart
#pragma unroll
        for (int q = 0; q < NG; ++q) {
            const int ce = start((q ^ rot) + 1);
            const bool over = q + 1 == NG;                   // (compile time) the step after is the next tile's
            const int cnext = over ? start(rot) : start((q + 1) ^ rot);
            const int tnext = over && tile + G < ntile ? tile + G : tile;
            for (int c = start(q ^ rot); c < ce; ++c) {
                lmh_wait_barrier<(S - 2) * (LW + LX)>();     // the step's values have landed, the last one's are read
                const int cn = c + 1 < ce ? c + 1 : cnext, tn = c + 1 < ce ? tile : tnext;
                float sc[MB];
#pragma unroll
                for (int i = 0; i < MB; ++i) {
                    sc[i] = sx[i] * swt;
                    asm volatile("" : "+v"(sc[i]));          // now: later, the next scales would need a copy, and that a wait
                }
                load_s(tn, cn);
                __builtin_amdgcn_sched_barrier(0);           // before the requests: waited for without them
                issue();
                const uint8_t* wb = sm + slot * SB + wr * VB * 4096;
                const uint8_t* xb = sm + slot * SB + WB + wc * MB * 4096;
                const bool half = c * 128 + 64 >= H;         // uniform: H % 128 == 64, the last block
                // NE pieces of the block (two in the last one when H % 128 == 64); each
                // read one ahead of its conversion
                auto block = [&](auto ne) __attribute__((always_inline)) {
                    constexpr int NE = decltype(ne)::value;
                    lmh_acc p[MB][VB];
#pragma unroll
                    for (int i = 0; i < MB; ++i)
#pragma unroll
                        for (int v = 0; v < VB; ++v)
#pragma unroll
                            for (int k = 0; k < 16; ++k) p[i][v][k] = 0.0f;
                    llima_u32x4 w[2][VB], x[2][MB];
                    auto read = [&](int e) {
                        const uint32_t o = rl + ((((uint32_t)(2 * e + g)) ^ rz) << 4);
#pragma unroll
                        for (int v = 0; v < VB; ++v) w[e & 1][v] = *(const llima_u32x4*)(wb + v * 4096 + o);
#pragma unroll
                        for (int i = 0; i < MB; ++i) x[e & 1][i] = *(const llima_u32x4*)(xb + i * 4096 + o);
                    };
                    read(0);
#pragma unroll
                    for (int e = 0; e < NE; ++e) {
                        if (e + 1 < NE) read(e + 1);
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            lmh_b8 wv[VB], xv[MB];
#pragma unroll
                            for (int v = 0; v < VB; ++v) wv[v] = q ? lmh8_wide(w[e & 1][v].z, w[e & 1][v].w) : lmh8_wide(w[e & 1][v].x, w[e & 1][v].y);
#pragma unroll
                            for (int i = 0; i < MB; ++i) xv[i] = q ? lmh8_wide(x[e & 1][i].z, x[e & 1][i].w) : lmh8_wide(x[e & 1][i].x, x[e & 1][i].y);
#pragma unroll
                            for (int i = 0; i < MB; ++i)
#pragma unroll
                                for (int v = 0; v < VB; ++v) p[i][v] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wv[v], xv[i], p[i][v], 0, 0, 0);
                        }
                    }
#pragma unroll
                    for (int i = 0; i < MB; ++i)
#pragma unroll
                        for (int v = 0; v < VB; ++v)
#pragma unroll
                            for (int k = 0; k < 16; ++k) acc[i][v][k] = __builtin_fmaf(p[i][v][k], sc[i], acc[i][v][k]);
                };
                if (half) block(std::integral_constant<int, 2>{});
                else block(std::integral_constant<int, 4>{});
                slot = slot + 1 == S ? 0 : slot + 1;
            }
            if constexpr (K > 0) {                           // a pair of groups, then a pair of pairs
#pragma unroll
                for (int k = 0; k < K; ++k) {
                    if ((q & ((1 << k) - 1)) != (1 << k) - 1) continue;      // (compile time)
#pragma unroll
                    for (int i = 0; i < MB; ++i)
#pragma unroll
                        for (int v = 0; v < VB; ++v)
#pragma unroll
                            for (int x = 0; x < 16; ++x) {
                                if (q >> k & 1) {
                                    acc[i][v][x] += low[k][i][v][x];
                                } else {
                                    low[k][i][v][x] = acc[i][v][x];
                                    acc[i][v][x] = 0.0f;
                                }
                            }
                }
            }
        }
        const int n = tile * LMH8_NV + wr * VB * 32;
        if (n < V) {                                         // uniform
#pragma unroll
            for (int i = 0; i < MB; ++i) {
                float x[16 * VB];
#pragma unroll
                for (int k = 0; k < 16 * VB; ++k) x[k] = acc[i][k >> 4][k & 15];
                lmh8_slot_out<16 * VB, SC>(P, x, best[i], b0 + mc[i], m[i] < nb, n, V, g);
            }
        }
#pragma unroll
        for (int i = 0; i < MB; ++i)
#pragma unroll
            for (int v = 0; v < VB; ++v)
#pragma unroll
                for (int k = 0; k < 16; ++k) acc[i][v][k] = 0.0f;
    }
    asm volatile("s_waitcnt vmcnt(0)" ::: "memory");         // no request outlives the workgroup
#pragma unroll
    for (int i = 0; i < MB; ++i) {
        const size_t at = (size_t)(b0 + mc[i]) * P.NW + blockIdx.x * RWV + wr;
        if constexpr (SC) {                                  // the two lanes' sums under the pair's maximum
            const float mo = __shfl_xor(best[i].m, 32, 64), so = __shfl_xor(best[i].s, 32, 64);
            const float mn = mo > best[i].m ? mo : best[i].m, mw = mn > -__builtin_inff() ? mn : 0.0f;
            auto under = [&](float m, float s) { return m > -__builtin_inff() ? s * __builtin_amdgcn_exp2f((m - mw) * LMH_LOG2E) : s; };
            if (m[i] < nb && g == 0) P.sums[at] = under(best[i].m, best[i].s) + under(mo, so);
        }
        if (m[i] < nb && g == 0) P.keys[at] = best[i].key;
    }
}

// Workgroups: one per CU, or per tile where there are fewer.  (As many as give
// each the same number of tiles: 151936 rows, B = 64, 142 us with 198 of them, 138
// with 256.)
static int lmh8_groups(int V) {
    const int ntile = (V + LMH8_NV - 1) / LMH8_NV;
    return ntile < LMH8_CUS ? ntile : LMH8_CUS;
}

// Key slots per hidden row: one per wave along the vocab rows.
static int lmh8_slots(int B, int V) { return lmh8_groups(V) * (B <= 32 ? 8 : 4); }

template <bool SC>
static int lmh8_run(Lmh8Params& Q, hipStream_t st) {
    LmhParams& P = Q.P;
    P.NW = lmh8_slots(P.B, P.V);
    const dim3 g((uint32_t)lmh8_groups(P.V)), blk(512);
    const bool apart = P.H >= 4096 && P.B <= 64;              // K = 2
    for (int b0 = 0; b0 < P.B; b0 += 128) {
        const int nb = P.B - b0 < 128 ? P.B - b0 : 128;
        if (P.B <= 32 && apart) hipLaunchKernelGGL((lmh8_tiles<8, 1, 1, 1, 4, 2, SC>), g, blk, 0, st, Q, b0, nb);
        else if (P.B <= 32) hipLaunchKernelGGL((lmh8_tiles<8, 1, 1, 1, 4, 0, SC>), g, blk, 0, st, Q, b0, nb);
        else if (apart) hipLaunchKernelGGL((lmh8_tiles<4, 2, 2, 1, 4, 2, SC>), g, blk, 0, st, Q, b0, nb);
        else if (nb <= 64) hipLaunchKernelGGL((lmh8_tiles<4, 2, 2, 1, 4, 0, SC>), g, blk, 0, st, Q, b0, nb);
        else hipLaunchKernelGGL((lmh8_tiles<4, 2, 2, 2, 3, 0, SC>), g, blk, 0, st, Q, b0, nb);
    }
    if (SC) hipLaunchKernelGGL(lmh_score_finish, dim3((uint32_t)P.B), dim3(LLIMA_WG), 0, st, P);
    else hipLaunchKernelGGL(lmh_finish, dim3((uint32_t)P.B), dim3(LLIMA_WG), 0, st, P);
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}
