/*
 * k_rows_gemm.h — the weight-streaming linear of a few activation rows
 * (gfx950), as k_rows.hip (plain: MODE GHIP_EP_STORE) and k_ffn_rows.hip (with
 * an epilogue, one or two weight matrices) instantiate it. k_rows.hip's header
 * describes it. With an epilogue:
 *   - x's rows may be apart, and K need only be a multiple of 8: the chunk that
 *     K cuts is completed with zeros in LDS;
 *   - dual modes: a wave's weight groups alternate between gate and up, so that
 *     one pass of x serves both and the reduction finds g and u of a column
 *     side by side;
 *   - bias and residual are loaded before the products, so that their latency
 *     is not added to the reduction's.
 */
#ifndef K_ROWS_GEMM_H
#define K_ROWS_GEMM_H

#include "ghip_epilogue.h"
#include "k_rows_addr.h"

#define RW_NW 8                  /* waves per workgroup */
#define RW_LDS_MAX (160u * 1024u)

/* LDS: each wave's SL slots of x and weights; the partial sums reuse it */
template <bool BF, int MR, int NT, int SL>
__host__ __device__ constexpr uint32_t rw_wave_lds() {
    return SL * ((MR * (BF ? 128u : 256u) < 1024u ? 1024u : MR * (BF ? 128u : 256u)) + 2048u * NT);
}
template <bool BF, int MR, int NT, int SL>
constexpr uint32_t rw_lds() {
    const uint32_t ring = RW_NW * rw_wave_lds<BF, MR, NT, SL>();
    const uint32_t red = RW_NW * MR * 16u * NT * 4u;
    return ring > red ? ring : red;
}

/* Weight rows of FP8 may start at any 8 bytes (the forms with an epilogue). */
typedef ghip_u32x4 rw_u32x4 __attribute__((aligned(8)));

/* What the forms with an epilogue take besides: the up projection of the dual
 * modes, x's row stride, and the epilogue. */
struct RwMore {
    const uint8_t *W2;
    const float *S2;
    uint32_t ldx;
    int exact;
    GhipEp ep;
};

template <bool BF, int MR, int NT, int KS, int NA, int SL, int MODE>
__global__ __launch_bounds__(RW_NW * 64, 1) void k_rows_gemm(
    const uint8_t *__restrict__ W, const float *__restrict__ S, const uint16_t *__restrict__ X,
    uint16_t *__restrict__ Y, uint32_t M, uint32_t O, uint32_t K,
    const uint32_t *__restrict__ exact_flag, uint32_t blk0, uint32_t tile0, RwMore more) {
    constexpr bool EPI = MODE != GHIP_EP_STORE, DUAL = ghip_ep_dual(MODE);
    /* weights that are read again stay in the caches: by the backward's dx next, or
     * by the other row tiles (linear BF16 37 x 1537 x 4096 9.7 -> 8.6 us). The forms
     * of up to 8 rows, which have one, are spared the branch (3 to 4%) */
    constexpr bool GRAD = MODE == GHIP_EP_DLINEAR || MODE == GHIP_EP_DGATED;
    const bool again = GRAD || (EPI && MR >= 16 && gridDim.y > 1u);
    constexpr uint32_t GPP = RW_NW / KS;                 /* row groups per workgroup */
    constexpr uint32_t OG = DUAL ? NT / 2 : NT;          /* output groups of 16 a wave */
    static_assert(!DUAL || NT % 2 == 0, "gate and up groups alternate");
    constexpr uint32_t MT = MR < 16 ? 1 : MR / 16;
    constexpr uint32_t XI = BF ? (MR < 8 ? 1 : MR / 8) : MR / 4;  /* x loads per chunk */
    constexpr uint32_t XROW = BF ? 128u : 256u;          /* x bytes of a row in a chunk */
    constexpr uint32_t XB = XI * 1024u, SLOT = XB + 2048u * NT;
    static_assert(SL * SLOT == rw_wave_lds<BF, MR, NT, SL>() &&
                      rw_lds<BF, MR, NT, SL>() <= RW_LDS_MAX, "LDS layout");
    static_assert(SL == 1 || SL == NA, "one LDS slot, or one per register set");
    extern __shared__ __attribute__((aligned(1024))) uint8_t rl[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t n = lane & 15u, g = lane >> 4;
    uint8_t *ring = rl + wv * (SL * SLOT);
    const uint32_t KB = BF ? 2u * K : K;                 /* weight row stride, bytes */
    const uint32_t nch = EPI ? (KB + 127u) >> 7 : KB >> 7, nkb = EPI ? (K + 127u) >> 7 : K >> 7;
    const uint32_t ldx = EPI ? more.ldx : K;
    /* pieces of a last chunk that K cuts; FP8 with K % 16 == 8: the last one is
     * half */
    const uint32_t end = EPI ? rw_end(KB) : 0u;
    const bool half = EPI && !BF && (K & 8u);
    const uint32_t part = wv % KS, slot = wv / KS;
    const uint32_t c0 = part * nch / KS, c1 = (part + 1u) * nch / KS, nc = c1 - c0;
    const uint32_t blk = blk0 + blockIdx.x, grp = blk * GPP + slot, row0 = grp * (16u * OG);
    const uint32_t m0 = (tile0 + blockIdx.y) * MR;
    const uint32_t mrows = min(M - m0, (uint32_t)MR);
    ghip_f32x4 acc[MT][NT];
#pragma unroll
    for (uint32_t a = 0; a < MT; a++)
#pragma unroll
        for (int b = 0; b < NT; b++) acc[a][b] = (ghip_f32x4){0.f, 0.f, 0.f, 0.f};

    /* the epilogue's inputs, on their way during the products: value v of the
     * workgroup's outputs is of thread v % 512 */
    constexpr uint32_t NOUT = GPP * MR * 16u * OG, NV = (NOUT + RW_NW * 64u - 1u) / (RW_NW * 64u);
    auto place = [&](uint32_t v, uint32_t &m, uint32_t &o) {
        const uint32_t sl = v / (MR * 16u * OG), e = v - sl * (MR * 16u * OG);
        m = e / (16u * OG);
        o = (blk * GPP + sl) * (16u * OG) + e % (16u * OG);
        return v < NOUT && m < mrows && o < O;
    };
    constexpr bool EARLY = EPI && NV <= 4;               /* more would spill (64 rows) */
    uint16_t ein[EARLY ? NV : 1], ebias[EARLY ? NV : 1];
    if constexpr (EARLY) {
#pragma unroll
        for (uint32_t i = 0; i < NV; i++) {
            uint32_t m, o;
            const bool live = place(tid + i * (RW_NW * 64u), m, o);
            ein[i] = live && more.ep.in ? more.ep.in[(size_t)(m0 + m) * more.ep.ldin + o] : (uint16_t)0;
            ebias[i] = live && more.ep.bias ? more.ep.bias[o] : (uint16_t)0;
        }
        __builtin_amdgcn_sched_barrier(0);
    }
    if (row0 < O && nc > 0u) {
        const uint8_t *rows = W + (size_t)row0 * KB;
        const uint8_t *rows2 = DUAL ? more.W2 + (size_t)row0 * KB : rows;
        ghip_cdma d[NT];
#pragma unroll
        for (int b = 0; b < NT; b++) {
            const uint32_t left = O - 1u - row0, ob = DUAL ? b >> 1 : b;
            if (left >= 16u * ob + 15u) {
                d[b] = ghip_cdma_offsets(lane, KB);
                d[b].off0 += 16u * ob * KB;
                d[b].off1 += 16u * ob * KB;
            } else {
                const uint32_t r0 = min(16u * ob + (lane >> 3), left);
                const uint32_t r1 = min(16u * ob + 8u + (lane >> 3), left);
                /* the piece swizzle is by the LDS row, not the clamped one */
                d[b].off0 = r0 * KB + 16u * ((lane & 7u) ^ ((lane >> 4) & 7u));
                d[b].off1 = r1 * KB + 16u * ((lane & 7u) ^ ((4u + (lane >> 4)) & 7u));
            }
        }
        /* x load u: BF rows 8u + l/8, piece l % 8; FP8 rows 4u + l/16, piece
         * l % 16 */
        constexpr uint32_t LPR = XROW / 16u;             /* lanes per row */
        const uint8_t *xb = (const uint8_t *)(X + (size_t)m0 * ldx);
        uint32_t xo[XI], xq[XI];
#pragma unroll
        for (uint32_t u = 0; u < XI; u++) {
            const uint32_t r = u * (64u / LPR) + lane / LPR;
            const uint32_t sw = BF ? (r >> 1) & 7u : r & 15u;
            xq[u] = (lane & (LPR - 1u)) ^ sw;
            xo[u] = min(r, mrows - 1u) * ldx * 2u + 16u * xq[u];
        }
        /* the chunk that K cuts (k_rows_addr.h) */
        const uint32_t q0 = rw_piece(lane, 0), q1 = rw_piece(lane, 1), xend = rw_xend(BF, end, half);
        auto cut = [&](uint32_t c) { return EPI && end && c == nch - 1u; };
        auto from = [&](uint32_t c, const uint8_t *wb, uint32_t off, uint32_t q) {
            return (const rw_u32x4 *)rw_from(wb, off, q, cut(c), half, end);
        };
        ghip_u32x4 xr[NA][XI], wr[NA][2 * NT];
        auto load = [&](auto set_c, uint32_t c) {
            constexpr int A = decltype(set_c)::value;
            const uint8_t *xc = xb + (size_t)c * XROW, *wc = rows + (size_t)c * 128u;
#pragma unroll
            for (uint32_t u = 0; u < XI; u++)
                xr[A][u] = *(const ghip_u32x4 *)(xc + rw_x(xo[u], xq[u], cut(c), xend));
#pragma unroll
            for (int b = 0; b < NT; b++) {
                const uint8_t *wb = DUAL && (b & 1) ? rows2 + (size_t)c * 128u : wc;
                if (again) {
                    wr[A][2 * b] = *from(c, wb, d[b].off0, q0);
                    wr[A][2 * b + 1] = *from(c, wb, d[b].off1, q1);
                } else {
                    wr[A][2 * b] = __builtin_nontemporal_load(from(c, wb, d[b].off0, q0));
                    wr[A][2 * b + 1] = __builtin_nontemporal_load(from(c, wb, d[b].off1, q1));
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        const float *srow = BF ? nullptr : S + (size_t)(row0 >> 7) * nkb;
        const float *srow2 = DUAL && !BF ? more.S2 + (size_t)(row0 >> 7) * nkb : srow;
        const bool exact = !BF && (EPI ? more.exact != 0 : exact_flag != nullptr && *exact_flag != 0u);
        auto step = [&](auto set_c, auto refill_c, uint32_t t) {
            constexpr int A = decltype(set_c)::value;
            uint8_t *xs = ring + (SL == 1 ? 0u : A * SLOT), *ws = xs + XB;
            if (cut(c0 + t)) {
                const ghip_u32x4 zero = {0u, 0u, 0u, 0u};
#pragma unroll
                for (uint32_t u = 0; u < XI; u++)
                    if (xq[u] >= xend) xr[A][u] = zero;
#pragma unroll
                for (int b = 0; b < NT; b++) {
                    auto tail = [&](uint32_t q, ghip_u32x4 &v) {
                        if (q >= end) v = zero;
                        else if (half && q == end - 1u) v = (ghip_u32x4){v[2], v[3], 0u, 0u};
                    };
                    tail(q0, wr[A][2 * b]);
                    tail(q1, wr[A][2 * b + 1]);
                }
            }
#pragma unroll
            for (uint32_t u = 0; u < XI; u++)
                *(ghip_u32x4 *)(xs + u * 1024u + lane * 16u) = xr[A][u];
#pragma unroll
            for (int b = 0; b < NT; b++)
                ghip_rl_store(ws + 2048u * b, lane, wr[A][2 * b], wr[A][2 * b + 1]);
            if constexpr (decltype(refill_c)::value) {
                __builtin_amdgcn_sched_barrier(0);
                load(set_c, c0 + t + NA);
            }
            ghip_chunk cw[NT];
#pragma unroll
            for (int b = 0; b < NT; b++) cw[b] = ghip_cdma_read(ws + 2048u * b, n, g);
            if constexpr (BF) {
#pragma unroll
                for (uint32_t a = 0; a < MT; a++) {
                    const uint32_t r = MR < 16 ? n & (MR - 1u) : 16u * a + n;
                    const uint32_t sw = (r >> 1) & 7u;
                    const ghip_bf16x8 x0 = *(const ghip_bf16x8 *)(xs + r * 128u + 16u * ((2u * g) ^ sw));
                    const ghip_bf16x8 x1 = *(const ghip_bf16x8 *)(xs + r * 128u + 16u * ((2u * g + 1u) ^ sw));
#pragma unroll
                    for (int b = 0; b < NT; b++) {
                        acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            x0, __builtin_bit_cast(ghip_bf16x8, cw[b].lo), acc[a][b], 0, 0, 0);
                        acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                            x1, __builtin_bit_cast(ghip_bf16x8, cw[b].hi), acc[a][b], 0, 0, 0);
                    }
                }
            } else {
                const float sg = ghip_sload(srow, c0 + t);
                const float su = DUAL ? ghip_sload(srow2, c0 + t) : sg;
                ghip_bf16x8 w4[NT][4];
#pragma unroll
                for (int b = 0; b < NT; b++) {
                    const float sc = DUAL && (b & 1) ? su : sg;
                    if (exact) {
                        ghip_deq16<true>(cw[b].lo, sc, w4[b][0], w4[b][1]);
                        ghip_deq16<true>(cw[b].hi, sc, w4[b][2], w4[b][3]);
                    } else {
                        ghip_deq16<false>(cw[b].lo, sc, w4[b][0], w4[b][1]);
                        ghip_deq16<false>(cw[b].hi, sc, w4[b][2], w4[b][3]);
                    }
                }
#pragma unroll
                for (uint32_t a = 0; a < MT; a++) {
                    const uint32_t r = MR < 16 ? n & (MR - 1u) : 16u * a + n;
#pragma unroll
                    for (uint32_t i = 0; i < 4; i++) {
                        const ghip_bf16x8 xv = *(const ghip_bf16x8 *)(
                            xs + r * 256u + 16u * ((4u * g + i) ^ (r & 15u)));
#pragma unroll
                        for (int b = 0; b < NT; b++)
                            acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(xv, w4[b][i],
                                                                               acc[a][b], 0, 0, 0);
                    }
                }
            }
        };
        using RF = std::true_type;
        using NR = std::false_type;
        using S0 = std::integral_constant<int, 0>;
        using S1 = std::integral_constant<int, NA - 1>;
        load(S0{}, c0);
        if constexpr (NA == 2) load(S1{}, min(c0 + 1u, nch - 1u));
        uint32_t t = 0;
        if constexpr (NA == 1) {
            for (; t + 1u < nc; t++) step(S0{}, RF{}, t);
            step(S0{}, NR{}, t);
        } else {
            for (; t + 3u < nc; t += 2u) {
                step(S0{}, RF{}, t);
                step(S1{}, RF{}, t + 1u);
            }
            if (nc - t == 3u) {
                step(S0{}, RF{}, t);
                step(S1{}, NR{}, t + 1u);
                step(S0{}, NR{}, t + 2u);
            } else if (nc - t == 2u) {
                step(S0{}, NR{}, t);
                step(S1{}, NR{}, t + 1u);
            } else {
                step(S0{}, NR{}, t);
            }
        }
    }
    /* the KS partial sums of each group, added in order */
    __syncthreads();
    float *red = (float *)rl;                            /* [8 waves][MR][16 NT] */
#pragma unroll
    for (uint32_t a = 0; a < MT; a++)
#pragma unroll
        for (int b = 0; b < NT; b++)
#pragma unroll
            for (uint32_t i = 0; i < 4; i++) {
                const uint32_t m = 16u * a + 4u * g + i;
                if (MR >= 16 || m < (uint32_t)MR)
                    red[(wv * MR + m) * (16u * NT) + 16u * b + n] = acc[a][b][i];
            }
    __syncthreads();
    if constexpr (!EPI) {
        for (uint32_t v = tid; v < GPP * MR * 16u * NT; v += RW_NW * 64u) {
            const uint32_t sl = v / (MR * 16u * NT), e = v - sl * (MR * 16u * NT);
            const uint32_t m = e / (16u * NT), c = e - m * (16u * NT);
            const uint32_t o = (blk * GPP + sl) * (16u * NT) + c;
            if (m < mrows && o < O) {
                float s = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; k++) s += red[((sl * KS + k) * MR) * (16u * NT) + e];
                Y[(size_t)(m0 + m) * O + o] = (uint16_t)ghip_bf16_bits(s);
            }
        }
    } else {
        ghip_with_act(more.ep.act, [&](auto act) {
#pragma unroll
            for (uint32_t i = 0; i < NV; i++) {
                uint32_t m, o;
                const uint32_t v = tid + i * (RW_NW * 64u);
                if (!place(v, m, o)) {
                    /* the output's own columns behind its width */
                    if (GRAD && more.ep.pad && v < NOUT
                        && m < mrows && o < ((O + 7u) & ~7u)) {
                        more.ep.out[(size_t)(m0 + m) * more.ep.ldout + o] = 0;
                        if (DUAL) more.ep.out2[(size_t)(m0 + m) * more.ep.ldout + o] = 0;
                    }
                    continue;
                }
                const uint32_t sl = v / (MR * 16u * OG), c = v % (16u * OG);
                /* dual: gate group, up group, ... of 16 columns */
                const uint32_t e = m * (16u * NT) + (DUAL ? 32u * (c >> 4) + (c & 15u) : c);
                float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
                for (int k = 0; k < KS; k++) {
                    const float *p = red + ((sl * KS + k) * MR) * (16u * NT) + e;
                    s0 += p[0];
                    if (DUAL) s1 += p[16];
                }
                if constexpr (EARLY)
                    ghip_ep_put<MODE, decltype(act)::value>(more.ep, more.ep.out, m0 + m, o, s0, s1,
                                                            ghip_bf16_f32(ebias[i]),
                                                            ghip_bf16_f32(ein[i]));
                else
                    ghip_ep_store<MODE, decltype(act)::value>(more.ep, more.ep.out, m0 + m, o, s0, s1);
            }
        });
    }
}

#endif /* K_ROWS_GEMM_H */
