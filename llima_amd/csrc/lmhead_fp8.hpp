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
// instructions 2^-25 and 2^-22), which is not a sum in 32 bits.  xq [B][H] and xs [B][NK] are a hidden row's values
// and scales, wq [V][H] and ws [ceil(V/128)][NK] the weight's, NK = ceil(H/128).
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
    uint8_t* frag;                                           // hidden rows in operand order (lmh8_order)
    float* fs;                                               // and their scales
    int32_t NK;
};

// The hidden rows in the order the MFMAs read them, so that a wave's load is 1 KB
// of adjacent memory (read from the rows themselves, 32 pieces of 32 bytes, they
// and not the weight bound the product: B = 64, H = 4096, V = 128256 147 us): per
// group of 32 rows and block of 128 ids the pieces e < 4, lane (r, g)'s 16 bytes
// being ids 32 e + 16 g .. of row r; then the block's 32 scales, one per row.
// Rows past the batch repeat its last one, ids past H are 0.
__global__ __launch_bounds__(LLIMA_WG) void lmh8_order(Lmh8Params Q) {
    const int kb = (int)blockIdx.x, rg = (int)blockIdx.y, t = (int)threadIdx.x;
    const int H = Q.P.H, B = Q.P.B, lane = t & 63, m = rg * 32 + (lane & 31), mc = m < B ? m : B - 1;
    const int h = kb * 128 + (t >> 6) * 32 + (lane >> 5) * 16;
    llima_u32x4 v = {0u, 0u, 0u, 0u};
    if (h < H) v = *(const llima_u32x4*)(Q.xq + (size_t)mc * H + h);
    const size_t block = (size_t)rg * Q.NK + kb;
    *(llima_u32x4*)(Q.frag + (block * 256 + t) * 16) = v;
    if (t < 32) Q.fs[block * 32 + t] = Q.xs[(size_t)mc * Q.NK + kb];
}

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

// One slot (2 NX vocab rows from n) of one hidden row per lane pair (r, 0), (r, 1):
// x[k] of lane half g is row (k / 16) 32 + (k / 4 % 4) 8 + 4 g + k % 4 of the
// slot.  Writes the logits when asked, the slot's key, and with SC its sum and
// the target's logit.  b: the hidden row (row false: none).
template <int NX, bool SC>
__device__ __forceinline__ void lmh8_slot_out(const LmhParams& P, float (&x)[NX], int b, bool row,
                                              int n, int g) {
    const int left = P.V - n;                                // <= 0: the slot is past the vocabulary
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
    if (left < 2 * NX) {                                     // uniform: rows past the vocabulary
#pragma unroll
        for (int k = 0; k < NX; ++k) x[k] = col(k) < left ? x[k] : __builtin_nanf("");
    }
    // the greatest of the two lanes' logits (NaN only when all are), and its first row
    float best = lmh_max3(x[0], x[1], x[1]);
#pragma unroll
    for (int k = 2; k < NX; k += 2) best = lmh_max3(best, x[k], x[k + 1]);
    best = lmh_max3(best, __shfl_xor(best, 32, 64), best);
    int at = 255;
#pragma unroll
    for (int k = NX - 1; k >= 0; --k) at = x[k] == best ? (k >> 4) * 32 + (k >> 2 & 3) * 8 + (k & 3) : at;
    at = at == 255 ? 255 : at + 4 * g;
    const int other = __shfl_xor(at, 32, 64);
    at = at < other ? at : other;
    const size_t slot = (size_t)b * P.NW + n / (2 * NX);
    if (row && g == 0)
        P.keys[slot] = at < 255 ? ((uint64_t)f32_key(best) << 32) | (uint32_t)~(uint32_t)(n + at) : 0ull;
    if constexpr (SC) {
        const int32_t tg = row ? P.targets[b] : -1;
        if (left < 2 * NX) {                                 // uniform
#pragma unroll
            for (int k = 0; k < NX; ++k) x[k] = col(k) < left ? x[k] : -__builtin_inff();
        }
        const float mw = best > -__builtin_inff() ? best : 0.0f;
        float e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < NX; ++k) e[k & 3] += __builtin_amdgcn_exp2f((x[k] - mw) * LMH_LOG2E);
        float s = (e[0] + e[1]) + (e[2] + e[3]);
        s += __shfl_xor(s, 32, 64);
        if (row && g == 0) P.sums[slot] = s;
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

// A barrier of the workgroup that waits for the wave's LDS accesses and for no
// other request.
__device__ __forceinline__ void lmh8_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

// lmh8_rows: up to 32 CG hidden rows.  A workgroup (one per CU) takes tiles of
// 64 vocab rows (tile, tile + grid, ...) through k in chunks of 512 ids: a
// chunk is 512 contiguous bytes of each of 64 weight rows, in a ring of LMH8_S LDS
// slots (32 KB).  Four waves request the chunks straight into LDS, four
// multiply: requests return in order, so a wave that also loaded hidden rows
// would wait for the weight's whenever it waits for those.  CG waves take a group
// of 32 hidden rows each, KS = 4 / CG waves share a group and split a chunk's
// four blocks of 128 between them, so that a wave's hidden values are its own:
// it loads them from L2 into registers, each block of the next chunk when that
// of this one is used.  At a tile's end the waves of a group exchange their
// sums through LDS and each finishes 64 / KS of the tile's rows (a key slot),
// while the ring fills up.
//
// LDS rows are 512 bytes with their 16-byte columns exchanged by row % 16 (the
// request's source address does it): fragment reads have no bank conflicts.
// The weight is the MFMA's row operand: lane (r, g) has for hidden row r the
// sums of half of a slot's rows (the lane with the other g the others).  k order
// within a block: piece e of 16 ids of half g is ids 32 e + 16 g .. + 15, its
// halves two steps, for both operands.
//
// 512 contiguous bytes per row: read 128 bytes at a time (a tile of 256 rows)
// the weight streams at 4.8 TB/s, this way at 5.6 to 5.9 (0.53 GB, requests alone).
#define LMH8_W 512                     // bytes of a row per chunk
#define LMH8_NV 64                     // vocab rows per tile

template <int CG, int NC, int S, bool SC>
__global__ __launch_bounds__(64 * (NC + 4)) void lmh8_rows(Lmh8Params Q, int b0, int nb) {
    constexpr int KS = NC / CG;                              // waves that share a column group
    constexpr int KB = 4 / KS;                               // blocks of a chunk per wave
    constexpr int SB = LMH8_NV * LMH8_W;                     // bytes of a slot
    constexpr int NX = 32 / KS;                              // a lane's sums of a finished slot
    constexpr int RED = NC * (KS - 1) * NX * 64 * 4;         // the exchanged sums
    static_assert(KS * CG == NC && KS <= 4 && S * SB + RED <= 163840, "shape");
    __shared__ __align__(1024) uint8_t sm[S * SB + RED];
    const LmhParams& P = Q.P;
    const int t = (int)threadIdx.x, lane = t & 63, g = lane >> 5, r = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int H = P.H, V = P.V, NK = Q.NK, nch = (H + LMH8_W - 1) / LMH8_W;
    const int ntile = (V + LMH8_NV - 1) / LMH8_NV, G = (int)gridDim.x;
    const int rot = (int)(blockIdx.x >> 3) % nch;            // the tiles' first chunk
    const int ntot = (ntile - 1 - (int)blockIdx.x) / G * nch + nch;   // the workgroup's chunks (grid <= ntile)
    if (wave >= NC) {
        const int wq = wave - NC;
        int tw = (int)blockIdx.x, cw = rot, sw = 0;
        auto issue = [&]() {                                 // the next chunk; past the last one, that again
            const uint8_t* base = Q.wq + (size_t)tw * LMH8_NV * H + cw * LMH8_W;
            const int left = V - 1 - tw * LMH8_NV;           // the tile's last row
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const int row = 2 * (wq + 4 * q) + (lane >> 5), pos = lane & 31;
                const int col = (pos ^ (row & 15)) * 16;     // bytes past H read the chunk's first ones
                lmh_dma(base, (uint32_t)(row < left ? row : left) * (uint32_t)H + (uint32_t)(cw * LMH8_W + col < H ? col : 0),
                        sm + sw * SB + (wq + 4 * q) * 1024);
            }
            sw = sw + 1 == S ? 0 : sw + 1;
            cw = cw + 1 == nch ? 0 : cw + 1;
            if (cw == rot && tw + G < ntile) tw += G;        // past its last tile: that again
        };
#pragma unroll
        for (int i = 0; i < S - 1; ++i) issue();
        asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 2) * 8) : "memory");   // chunk 0 has landed
        for (int i = 0, c = 0; i < ntot; ++i) {
            issue();                                         // into the slot read before the last barrier
            if (++c == nch) {
                c = 0;
                if (KS > 1) asm volatile("s_barrier" ::: "memory");
            }
            asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((S - 2) * 8) : "memory");   // chunk i + 1 has
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");     // no request outlives the workgroup
        return;
    }
    const int cg = wave % CG, ks = wave / CG;
    const int m = cg * 32 + r;                               // the lane's hidden row of the pass
    const int mc = m < nb ? m : nb - 1;                      // rows past the batch repeat the last one
    const size_t block0 = (size_t)((b0 >> 5) + (cg * 32 < nb ? cg : 0)) * NK;   // the group's first block
    const uint8_t* const xf = Q.frag + block0 * 4096 + lane * 16;
    const float* const xsf = Q.fs + block0 * 32 + r;
    llima_u32x4 hx[KB][4];
    float sx[KB], sw[KB];
    auto load = [&](int tile, int c, int j) {                // block j of the wave in chunk c of tile
        const int kb = c * 4 + ks * KB + j, kc = kb < NK ? kb : 0;
        sx[j] = xsf[kc * 32];
        sw[j] = Q.ws[(size_t)(tile >> 1) * NK + kc];
#pragma unroll
        for (int p = 0; p < 4; ++p) hx[j][p] = *(const llima_u32x4*)(xf + (size_t)kc * 4096 + p * 1024);
    };
    int tile = (int)blockIdx.x, c = rot, slot = 0;
    float acc[2][16];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[j][i] = 0.0f;
#pragma unroll
    for (int j = 0; j < KB; ++j) load(tile, rot, j);
    asm volatile("s_barrier" ::: "memory");
    for (int it = 0; it < ntot; ++it) {
        const uint8_t* wb = sm + slot * SB;
        const int cn = c + 1 == nch ? 0 : c + 1;
        const bool end = cn == rot;                          // uniform: the tile's last chunk
        const int tn = end && tile + G < ntile ? tile + G : tile;
#pragma unroll
        for (int j = 0; j < KB; ++j) {
            const int kb = c * 4 + ks * KB + j;
            if (kb < NK) {                                   // uniform
                const bool half = kb * 128 + 64 >= H;        // uniform: H % 128 == 64, the last block
                lmh_acc p[2];
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int i = 0; i < 16; ++i) p[v][i] = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (e < 2 || !half) {
                        const llima_u32x4 x = hx[j][e];
                        const lmh_b8 x0 = lmh8_wide(x.x, x.y), x1 = lmh8_wide(x.z, x.w);
#pragma unroll
                        for (int v = 0; v < 2; ++v) {
                            const int row = v * 32 + r;
                            const llima_u32x4 w = *(const llima_u32x4*)(wb + row * LMH8_W + ((((ks * KB + j) * 8 + 2 * e + g) ^ (row & 15)) << 4));
                            p[v] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lmh8_wide(w.x, w.y), x0, p[v], 0, 0, 0);
                            p[v] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(lmh8_wide(w.z, w.w), x1, p[v], 0, 0, 0);
                        }
                    }
                }
                const float sc = sx[j] * sw[j];
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[v][i] = __builtin_fmaf(p[v][i], sc, acc[v][i]);
            }
            load(tn, cn, j);
        }
        if (end) {                                           // uniform
            float x[NX];
            if constexpr (KS > 1) {
                // wave ks keeps sums ks NX .. + NX - 1 of its 32 and gives the others to their waves
                float* red = (float*)(sm + S * SB);
#pragma unroll
                for (int d = 1; d < KS; ++d) {
                    const int to = (ks + d) % KS;
                    float* w = red + (((to * CG + cg) * (KS - 1) + d - 1) * NX) * 64 + lane;
#pragma unroll
                    for (int i = 0; i < NX; ++i) {
                        float v = 0.0f;
#pragma unroll
                        for (int q = 0; q < KS; ++q) v = to == q ? acc[(q * NX + i) >> 4][(q * NX + i) & 15] : v;
                        w[i * 64] = v;
                    }
                }
                lmh8_barrier();
#pragma unroll
                for (int i = 0; i < NX; ++i) {
                    float v = 0.0f;
#pragma unroll
                    for (int q = 0; q < KS; ++q) v = ks == q ? acc[(q * NX + i) >> 4][(q * NX + i) & 15] : v;
#pragma unroll
                    for (int d = 1; d < KS; ++d) v += red[(((ks * CG + cg) * (KS - 1) + d - 1) * NX + i) * 64 + lane];
                    x[i] = v;
                }
            } else {
#pragma unroll
                for (int i = 0; i < NX; ++i) x[i] = acc[i >> 4][i & 15];
            }
            const int n = tile * LMH8_NV + ks * 2 * NX;
            if (n < V) lmh8_slot_out<NX, SC>(P, x, b0 + mc, m < nb, n, g);   // uniform
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[j][i] = 0.0f;
        }
        c = cn;
        tile = tn;
        slot = slot + 1 == S ? 0 : slot + 1;
        lmh8_barrier();
    }
}

// Vocab rows per key slot: a wave finishes 64 / KS rows of a tile.
#ifndef LMH8_C2
#define LMH8_C2 8, 3
#define LMH8_T2 768
#define LMH8_R2 16
#endif
static int lmh8_slot_rows(int nb) { return nb <= 32 ? 16 : nb <= 64 ? LMH8_R2 : 32; }

template <bool SC>
static int lmh8_run(Lmh8Params& Q, hipStream_t st) {
    LmhParams& P = Q.P;
    const int ntile = (P.V + LMH8_NV - 1) / LMH8_NV;
    const int per = P.B < 128 ? P.B : 128;                   // rows per pass, one slot size for all
    P.NW = (P.V + lmh8_slot_rows(per) - 1) / lmh8_slot_rows(per);
    const dim3 g((uint32_t)(ntile < LMH_CUS ? ntile : LMH_CUS));
    hipLaunchKernelGGL(lmh8_order, dim3((uint32_t)Q.NK, (uint32_t)((P.B + 31) / 32)), dim3(LLIMA_WG), 0, st, Q);
    for (int b0 = 0; b0 < P.B; b0 += 128) {
        const int nb = P.B - b0 < 128 ? P.B - b0 : 128;
        if (per <= 32) hipLaunchKernelGGL((lmh8_rows<1, 4, 4, SC>), g, dim3(512), 0, st, Q, b0, nb);
        else if (per <= 64) hipLaunchKernelGGL((lmh8_rows<2, LMH8_C2, SC>), g, dim3(LMH8_T2), 0, st, Q, b0, nb);
        else hipLaunchKernelGGL((lmh8_rows<4, 8, 4, SC>), g, dim3(768), 0, st, Q, b0, nb);
    }
    if (SC) hipLaunchKernelGGL(lmh_score_finish, dim3((uint32_t)P.B), dim3(LLIMA_WG), 0, st, P);
    else hipLaunchKernelGGL(lmh_finish, dim3((uint32_t)P.B), dim3(LLIMA_WG), 0, st, P);
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}
