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
    int32_t NK;
};

// One slot (64 vocab rows from n) of one hidden row per lane pair (r, 0), (r, 1):
// x[k] of lane half g is row (k / 16) 32 + (k / 4 % 4) 8 + 4 g + k % 4 of the
// slot.  Writes the logits when asked, the slot's key, and with SC its sum and
// the target's logit.  b: the hidden row (row false: none).
template <bool SC>
__device__ __forceinline__ void lmh8_slot_out(const LmhParams& P, float (&x)[32], int b, bool row,
                                              int n, int g) {
    const int left = P.V - n;                                // > 0
    auto col = [&](int k) { return (k >> 4) * 32 + (k >> 2 & 3) * 8 + 4 * g + (k & 3); };
    lmh_logits32(P, x);
    if (P.out_logits) {                                      // uniform
        const bool wide = ((uintptr_t)P.out_logits & 15u) == 0 && P.V % 4 == 0;
        if (P.logits_bf16) {
            auto h = [](float v) { return v == v ? __float_as_uint(v) >> 16 : 0x7FC0u; };
            uint16_t* o = (uint16_t*)P.out_logits + (size_t)(row ? b : 0) * P.V + n;
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
                if (row && wide && col(k) < left) {
                    *(uint2*)(o + col(k)) = make_uint2(h(x[k]) | h(x[k + 1]) << 16, h(x[k + 2]) | h(x[k + 3]) << 16);
                } else if (row && !wide) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (col(k + e) < left) o[col(k + e)] = (uint16_t)h(x[k + e]);
                }
            }
        } else {
            float* o = P.out_logits + (size_t)(row ? b : 0) * P.V + n;
#pragma unroll
            for (int k = 0; k < 32; k += 4) {
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
    if (left < LMH_SLOT) {                                   // uniform: rows past the vocabulary
#pragma unroll
        for (int k = 0; k < 32; ++k) x[k] = col(k) < left ? x[k] : __builtin_nanf("");
    }
    float best;
    const int at = lmh_first_max(x, g, best);
    const size_t slot = (size_t)b * P.NW + n / LMH_SLOT;
    if (row && g == 0)
        P.keys[slot] = at < 255 ? ((uint64_t)f32_key(best) << 32) | (uint32_t)~(uint32_t)(n + at) : 0ull;
    if constexpr (SC) {
        const int32_t tg = row ? P.targets[b] : -1;
        if (left < LMH_SLOT) {                               // uniform
#pragma unroll
            for (int k = 0; k < 32; ++k) x[k] = col(k) < left ? x[k] : -__builtin_inff();
        }
        const float mw = best > -__builtin_inff() ? best : 0.0f;
        float e[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int k = 0; k < 32; ++k) e[k & 3] += __builtin_amdgcn_exp2f((x[k] - mw) * LMH_LOG2E);
        float s = (e[0] + e[1]) + (e[2] + e[3]);
        s += __shfl_xor(s, 32, 64);
        if (row && g == 0) P.sums[slot] = s;
        const int ts = tg >= 0 ? tg - n : -1;                // the target's column of the slot
        const bool hit = ts >= 0 && ts < LMH_SLOT && ts < left && (ts >> 2 & 1) == g;
        if (__any(hit)) {
            float v = 0.0f;
#pragma unroll
            for (int k = 0; k < 32; ++k) v = ts == col(k) ? x[k] : v;
            if (hit) P.tval[b] = v;
        }
    }
}

// lmh8_rows: up to 32 CG hidden rows.  A workgroup of four waves takes tiles of
// 64 vocab rows (tile, tile + grid, ...) through k in chunks of 512 ids: a
// chunk is 512 contiguous bytes of each of 64 weight rows, requested straight
// into one of two LDS slots (32 KB) while the other is read; two workgroups
// share a CU.  CG waves take a group of 32 hidden rows each, KS = 4 / CG waves
// share a group and split a chunk's four blocks of 128 between them, so that a
// wave's hidden values are its own: it loads them from L2 into registers one
// chunk ahead.  LDS rows are 512 bytes with their 16-byte columns exchanged by
// row % 16 (the request's source address does it): fragment reads have no bank
// conflicts.  The weight is the MFMA's row operand: lane (r, g) has for hidden
// row r the sums of 32 of the tile's 64 vocab rows (the lane with the other g
// the others).  k order within a block: piece e of 16 ids of half g is ids
// 32 e + 16 g .. + 15, its halves two steps, for both operands.
//
// 512 contiguous bytes per row: read 128 bytes at a time (a tile of 256 rows)
// the weight streams at 4.8 TB/s, this way at 5.6 to 5.9 (0.53 GB, requests alone).
#define LMH8_W 512                     // bytes of a row per chunk
#define LMH8_NV 64                     // vocab rows per tile

template <int CG, bool SC>
__global__ __launch_bounds__(256, 2) void lmh8_rows(Lmh8Params Q, int b0, int nb) {
    constexpr int KS = 4 / CG;                               // waves that share a column group
    constexpr int KB = 4 / KS;                               // blocks of a chunk per wave
    constexpr int SB = LMH8_NV * LMH8_W;                     // bytes of a slot
    __shared__ __align__(1024) uint8_t sm[2 * SB];
    const LmhParams& P = Q.P;
    const int t = (int)threadIdx.x, lane = t & 63, g = lane >> 5, r = lane & 31;
    const int wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const int cg = wave % CG, ks = wave / CG;
    const int H = P.H, V = P.V, NK = Q.NK, nch = (H + LMH8_W - 1) / LMH8_W;
    const int ntile = (V + LMH8_NV - 1) / LMH8_NV;
    const int m = cg * 32 + r;                               // the lane's hidden row of the pass
    const int mc = m < nb ? m : nb - 1;                      // rows past the batch repeat the last one
    const uint8_t* const xrow = Q.xq + (size_t)(b0 + mc) * H;
    const float* const xsrow = Q.xs + (size_t)(b0 + mc) * NK;
    // the request stream: a tile and a chunk of it
    int tw = (int)blockIdx.x, cw = 0;
    auto issue_w = [&](int slot) {
        const uint8_t* base = Q.wq + (size_t)tw * LMH8_NV * H + cw * LMH8_W;
        const int left = V - 1 - tw * LMH8_NV;               // the tile's last row
#pragma unroll
        for (int q = 0; q < 8; ++q) {
            const int row = 2 * (wave + 4 * q) + (lane >> 5), pos = lane & 31;
            const int col = (pos ^ (row & 15)) * 16;         // bytes past H read the chunk's first ones
            lmh_dma(base, (uint32_t)(row < left ? row : left) * (uint32_t)H + (uint32_t)(cw * LMH8_W + col < H ? col : 0),
                    sm + slot * SB + (wave + 4 * q) * 1024);
        }
    };
    llima_u32x4 hx[KB][4];
    float sc[KB];
    auto load_x = [&](llima_u32x4 (&h)[KB][4], float (&s)[KB]) {
#pragma unroll
        for (int j = 0; j < KB; ++j) {
            const int kb = cw * 4 + ks * KB + j, kc = kb < NK ? kb : 0;
            s[j] = xsrow[kc] * Q.ws[(size_t)(tw >> 1) * NK + kc];
#pragma unroll
            for (int p = 0; p < 4; ++p) {
                const int o = kc * 128 + p * 32 + g * 16;
                h[j][p] = *(const llima_u32x4*)(xrow + (o < H ? o : 0));
            }
        }
    };
    auto next = [&]() {                                      // false: past the last chunk
        if (++cw == nch) { cw = 0; tw += (int)gridDim.x; }
        return tw < ntile;
    };
    bool more = tw < ntile;                                  // uniform
    if (!more) return;
    load_x(hx, sc);
    issue_w(0);
    int slot = 0, c = 0, tile = tw;
    float acc[2][16];
#pragma unroll
    for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[j][i] = 0.0f;
    while (more) {
        asm volatile("s_waitcnt vmcnt(0)\n\ts_barrier" ::: "memory");   // the chunk has landed
        more = next();
        llima_u32x4 hn[KB][4];
        float sn[KB];
        if (more) {                                          // uniform
            load_x(hn, sn);
            issue_w(slot ^ 1);                               // its readers passed the barrier
        }
        const uint8_t* wb = sm + slot * SB;
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
#pragma unroll
                for (int v = 0; v < 2; ++v)
#pragma unroll
                    for (int i = 0; i < 16; ++i) acc[v][i] = __builtin_fmaf(p[v][i], sc[j], acc[v][i]);
            }
        }
        if (++c == nch) {                                    // uniform: the tile is summed
            c = 0;
            if constexpr (KS > 1) {                          // the groups' waves add up, in the order of ks
                asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");   // the slot is read
                float* red = (float*)(sm + slot * SB);
                if (ks > 0) {
#pragma unroll
                    for (int i = 0; i < 32; ++i)
                        red[(((ks - 1) * CG + cg) * 32 + i) * 64 + lane] = acc[i >> 4][i & 15];
                }
                __syncthreads();
                if (ks == 0) {
#pragma unroll
                    for (int k = 1; k < KS; ++k)
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            acc[i >> 4][i & 15] += red[(((k - 1) * CG + cg) * 32 + i) * 64 + lane];
                }
            }
            if (ks == 0) {
                float x[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) x[i] = acc[i >> 4][i & 15];
                lmh8_slot_out<SC>(P, x, b0 + mc, m < nb, tile * LMH8_NV, g);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[j][i] = 0.0f;
            tile += (int)gridDim.x;
        }
        slot ^= 1;
        if (more) {
#pragma unroll
            for (int j = 0; j < KB; ++j) {
                sc[j] = sn[j];
#pragma unroll
                for (int p = 0; p < 4; ++p) hx[j][p] = hn[j][p];
            }
        }
    }
}

template <bool SC>
static int lmh8_run(Lmh8Params& Q, hipStream_t st) {
    LmhParams& P = Q.P;
    const int ntile = (P.V + LMH8_NV - 1) / LMH8_NV;
    P.NW = (P.V + LMH_SLOT - 1) / LMH_SLOT;
    const dim3 g((uint32_t)(ntile < 512 ? ntile : 512));
    for (int b0 = 0; b0 < P.B; b0 += 128) {
        const int nb = P.B - b0 < 128 ? P.B - b0 : 128;
        if (nb <= 32) hipLaunchKernelGGL((lmh8_rows<1, SC>), g, dim3(256), 0, st, Q, b0, nb);
        else if (nb <= 64) hipLaunchKernelGGL((lmh8_rows<2, SC>), g, dim3(256), 0, st, Q, b0, nb);
        else hipLaunchKernelGGL((lmh8_rows<4, SC>), g, dim3(256), 0, st, Q, b0, nb);
    }
    if (SC) hipLaunchKernelGGL(lmh_score_finish, dim3((uint32_t)P.B), dim3(LLIMA_WG), 0, st, P);
    else hipLaunchKernelGGL(lmh_finish, dim3((uint32_t)P.B), dim3(LLIMA_WG), 0, st, P);
    return hipGetLastError() == hipSuccess ? LLIMA_OK : LLIMA_E_HIP;
}
