/*
 * k_mx_gemm.h — x W^T on tiles, W in MXFP4, x in MXFP8, MXFP4 or BF16 (gfx950).
 *
 *   y[m, n] = sum over blocks b of 32 k: 2^(sx + sw - 254) sum_k x[m, k] w[n, k]
 *
 * Microscaled x goes to v_mfma_scale_f32_16x16x128_f8f6f4 as it lies: the instruction
 * multiplies the block's two scales in, so nothing is dequantized, and MXFP4 against
 * MXFP4 has twice the rate of MXFP8 (dense peaks 10 and 5 PFLOP/s). BF16 x takes W's
 * codes to BF16 at the operand, exactly, by the conversion that takes a scale: two
 * codes an instruction, over the second half of the step before.
 *
 * Bound by the MFMAs at the chip's power limit for large products, by what a step costs
 * with few workgroups. Four waves; a step of 128 k (BF16 64) comes straight to LDS, R
 * steps in a ring; a wave waits for its own loads by count, so those of R - 2 steps stay
 * in flight over the one barrier of a step. Between the MFMAs of a step, in places set
 * by hand, stand the next step's operand reads and the loads of step j + R. The
 * accumulators of the largest tile fill all 256 AGPRs and stay in place through an
 * assembly MFMA; what the compiler then does not know is read from the built code by
 * tests/test_mx_asm.py.
 *
 * Measured (us; TFLOP/s): MXFP4 8192 x 8192 x 8192 266 (4130), 4096^3 45.6 (3010);
 * MXFP8 8192^3 362 (3035), 4096^3 57.8 (2380), gated 8192 x 12288 x 4096 603-625 (2640-2740);
 * BF16 8192^3 791 (1390). The library's plain products of 8192^3 in the same types run at
 * 2990, 1290 and 1390.
 */
#ifndef K_MX_GEMM_H
#define K_MX_GEMM_H

#include "ghip_mx.h"
#include "k_ffn_gemm.h"
#include "k_mx_addr.h"

typedef int mg_i32x8 __attribute__((ext_vector_type(8)));

/* acc += w (16 rows of MXFP4) . x^T over 128 k, in place; byte Q of sw and sx: the
 * blocks' scales. As fg_mfma the compiler knows no MFMA in it. */
template <int Q>
__device__ __forceinline__ void mg_mfma(ghip_f32x4 &acc, const ghip_u32x4 &w, const mg_i32x8 &x, uint32_t sw,
                                        uint32_t sx) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] cbsz:4"
        : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx), "n"(Q & 1), "n"(Q >> 1));
#endif
}
template <int Q>
__device__ __forceinline__ void mg_mfma(ghip_f32x4 &acc, const ghip_u32x4 &w, const ghip_u32x4 &x, uint32_t sw,
                                        uint32_t sx) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel:[%5,%5,0] op_sel_hi:[%6,%6,0] cbsz:4 blgp:4"
        : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx), "n"(Q & 1), "n"(Q >> 1));
#endif
}

/* 4 words of 4 bytes in each of 64 lanes, lane (n, b) a row of scales of block b of 16
 * rows: out[b] of lane (n, g) is byte g of the words of block b's row n. */
__device__ __forceinline__ ghip_u32x4 mg_turn(const ghip_u32x4 &v) {
    const uint32_t lo01 = __builtin_amdgcn_perm(v[1], v[0], 0x05010400u), hi01 = __builtin_amdgcn_perm(v[1], v[0], 0x07030602u);
    const uint32_t lo23 = __builtin_amdgcn_perm(v[3], v[2], 0x05010400u), hi23 = __builtin_amdgcn_perm(v[3], v[2], 0x07030602u);
    /* byte g of the words, then bytes against lane groups */
    const auto a = __builtin_amdgcn_permlane16_swap(__builtin_amdgcn_perm(lo23, lo01, 0x05040100u), __builtin_amdgcn_perm(lo23, lo01, 0x07060302u), false, false);
    const auto b = __builtin_amdgcn_permlane16_swap(__builtin_amdgcn_perm(hi23, hi01, 0x05040100u), __builtin_amdgcn_perm(hi23, hi01, 0x07060302u), false, false);
    const auto e = __builtin_amdgcn_permlane32_swap(a[0], b[0], false, false);
    const auto o = __builtin_amdgcn_permlane32_swap(a[1], b[1], false, false);
    return (ghip_u32x4){e[0], o[0], e[1], o[1]};
}

/* v, in a register of its own from here on: a copy that the compiler makes of it later could
 * be too near an MFMA, which it knows nothing of. */
__device__ __forceinline__ uint32_t mg_keep(uint32_t v) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("" : "+v"(v));
#endif
    return v;
}

/* Whether one of the n steps before one of quarter qu is of quarter 2, steps before the
 * first among them: n up to 4, so at most one is. */
constexpr int mg_third(int qu, int n) {
    int c = 0;
    for (int i = 1; i <= (n < 4 ? n : 4); i++) c += (qu + 8 - i) % 4 == 2;
    return c;
}
template <int N>
__device__ __forceinline__ void mg_wait() {
    constexpr int M = N < 63 ? N : 63;
    GHIP_VMCNT(M);
}

template <int MODE, int XT, int WM, int WN, int RB, int CB, int R>
struct MgTile {
    static constexpr bool DUAL = ghip_ep_dual(MODE), BF = XT == GHIP_BF16;
    static constexpr uint32_t NW = WM * WN, BM = 16u * RB * WM, BN = 16u * CB * WN, OUTN = DUAL ? BN / 2 : BN;
    /* a step: k, bytes of a row of x and of W */
    static constexpr uint32_t KS = BF ? 64u : 128u, XB = XT == GHIP_MXFP4 ? 64u : 128u, WB = BF ? 32u : 64u;
    static constexpr uint32_t AST = BM * XB, BST = BN * WB;
    static constexpr uint32_t SLOT = AST + BST, RING = R * SLOT;
    static constexpr uint32_t NAL = AST / 1024u / NW, NBL = BST / 1024u / NW, LPS = NAL + NBL;
    /* scales of four words of k, 16 bytes a row: x's rows, W's, the second matrix's, each
     * in units of 64 rows */
    static constexpr uint32_t XU = BF ? 0u : (BM + 63u) / 64u, WU = (OUTN + 63u) / 64u, NU = XU + WU * (DUAL ? 2u : 1u);
    static constexpr uint32_t NSL = (NU + NW - 1u) / NW, LDS = RING + NU * 1024u;
    static_assert(AST % (1024u * NW) == 0 && BST % (1024u * NW) == 0, "whole loads");
    static_assert(LDS <= FG_LDS_MAX && R >= 3 && (R - 2) * LPS <= 63, "ring, waits");
    static_assert(!DUAL || CB % 2 == 0, "gate and up blocks alternate");
};

template <int MODE, int XT, int WM, int WN, int RB, int CB, int R>
__global__ __launch_bounds__(64 * WM * WN, 1) void k_mx_gemm(GhipMxProd p, GhipEp ep, uint32_t mt,
                                                             uint32_t nt) {
    using T = MgTile<MODE, XT, WM, WN, RB, CB, R>;
    constexpr bool DUAL = T::DUAL, BF = T::BF;
    constexpr uint32_t NW = T::NW, BM = T::BM, BN = T::BN, OUTN = T::OUTN, XB = T::XB, WB = T::WB, KS = T::KS;
    constexpr uint32_t NAL = T::NAL, NBL = T::NBL, LPS = T::LPS, SLOT = T::SLOT;
    constexpr int NM = RB * CB;
    extern __shared__ __attribute__((aligned(1024))) uint8_t mg_lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wr = wv / WN, wc = wv % WN, n = lane & 15u, g = lane >> 4;

    /* the tile: an XCD's workgroups take a run of consecutive ones, 4 row tiles before
     * the next column */
    uint32_t t;
    {
        const uint32_t x = blockIdx.x & 7u, i = blockIdx.x >> 3, q = gridDim.x >> 3, r = gridDim.x & 7u;
        t = x * q + (x < r ? x : r) + i;
    }
    const uint32_t strip = t / (4u * nt), in_strip = t - strip * (4u * nt);
    const uint32_t sr = min(4u, mt - strip * 4u);
    const uint32_t row0 = (strip * 4u + in_strip % sr) * BM, col0 = in_strip / sr * OUTN;
    const uint32_t rows = min(p.M - row0, BM), cols = min(p.N - col0, OUTN);
    const uint32_t nst = (p.K + KS - 1u) / KS, words = (p.K + 127u) >> 7, lds = 4u * words, wb = p.K >> 1, xld = (uint32_t)p.xld;
    const bool up = DUAL && (wv & 1u);

    /* loads: this lane's place in the first one; the others are a whole number of
     * rows behind it. Rows past the matrix are past the buffer, pieces past K are put
     * there */
    const uint8_t *pa = p.x + (size_t)row0 * p.xld, *pb = (up ? p.w2 : p.w) + (size_t)col0 * wb;
    const uint32_t aspan = rows * xld, bspan = cols * wb;
    const uint32_t ar = mg_row<XB>(wv, lane), aq = mg_byte<XB>(lane, ar), ao = ar * xld + aq;
    const uint32_t br = mg_row<WB>(DUAL ? wv >> 1 : wv, lane), bq = mg_byte<WB>(lane, br), bo = br * wb + bq;
    const uint32_t astep = mg_rows_apart<XB, NW>(false) * xld, bstep = mg_rows_apart<WB, NW>(DUAL) * wb;
    const uint32_t xrow = BF ? 2u * p.K : XT == GHIP_MXFP8 ? p.K : wb;   /* bytes of x's row */
    uint32_t sl = 0;                                     /* slot of the next step to load */
    int32_t xleft = (int32_t)xrow, wleft = (int32_t)wb;
    auto load = [&](uint32_t i) {
        if (i < NAL) {
            const uint32_t off = mg_cut(ao + i * astep, aq, xleft);
            fg_dma16(pa, aspan, off, mg_lds + sl + (wv + NW * i) * 1024u);
        } else {
            const uint32_t off = mg_cut(bo + (i - NAL) * bstep, bq, wleft);
            fg_dma16(pb, bspan, off, mg_lds + sl + T::AST + (wv + NW * (i - NAL)) * 1024u);
        }
    };
    auto next_load = [&]() {
        pa += XB;
        pb += WB;
        xleft -= (int32_t)XB;
        wleft -= (int32_t)WB;
        sl = sl == (R - 1u) * SLOT ? 0u : sl + SLOT;
    };

    /* Operands. W's are read one step ahead into the other set. x's row block r is read
     * again, for the next step, once its products are issued; the last one has two
     * sets, as its step ends with it */
    using XReg = std::conditional_t<XT == GHIP_MXFP4, ghip_u32x4, mg_i32x8>;
    using WReg = std::conditional_t<BF, mg_i32x8, ghip_u32x4>;
    XReg xa[RB], xl[2];
    WReg wa[2][CB];
    ghip_u32x2 codes[BF ? CB : 1];
    const uint32_t a0 = mg_at_x<XB>(wr * RB, n, g, 0, BF), a1 = mg_at_x<XB>(wr * RB, n, g, 1, BF);
    const uint32_t b0 = mg_at_w<WB, CB>(T::AST, wc, n, g, DUAL);
    auto read_x = [&](XReg &x, int r, const uint8_t *st) {
        const ghip_u32x4 lo = *(const ghip_u32x4 *)(st + a0 + r * (16u * XB));
        if constexpr (XB == 128u) {
            const ghip_u32x4 hi = *(const ghip_u32x4 *)(st + a1 + r * (16u * XB));
            x = (mg_i32x8){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
        } else {
            x = lo;
        }
    };
    auto read_a = [&](auto set_c, auto r_c, const uint8_t *st) {
        constexpr int S = decltype(set_c)::value, r = decltype(r_c)::value;
        if constexpr (r == RB - 1) read_x(xl[S], r, st);
        else read_x(xa[r], r, st);
    };
    auto read_b = [&](auto set_c, auto c_c, const uint8_t *st) {
        constexpr int S = decltype(set_c)::value, c = decltype(c_c)::value;
        if constexpr (BF) codes[c] = *(const ghip_u32x2 *)(st + b0 + mg_w_step<WB>(c, DUAL));
        else wa[S][c] = *(const ghip_u32x4 *)(st + b0 + mg_w_step<WB>(c, DUAL));
    };

    /* Scales. The workgroup's waves share out its rows, 64 a load: 16 bytes of a row, the
     * scales of four steps (eight of 64 k), go through registers to LDS four steps behind
     * their load. From there a wave reads its blocks', four at a time, and turns them
     * (mg_turn) into words that the MFMA picks a step's byte from by number. Each of the
     * simpler ways costs more than a small tile's step: 4 bytes a row every step, as the
     * line is in flight already and the loads wait for it one after the other (64 x 64
     * tiles, 4096 x 4096 x 4096: 193 us, 93 with no scales at all, 112 so); every wave its
     * own blocks', as the waves of a row of tiles ask for the same lines (256 x 256, 8192 x
     * 8192 x 8192 in MXFP4: 302 us, 277 so) */
    constexpr uint32_t NSL = T::NSL, XU = T::XU, WU = T::WU, NU = T::NU;
    constexpr int XQ = BF ? 0 : (RB + 3) / 4, WQ = DUAL ? (CB / 2 + 3) / 4 : (CB + 3) / 4, NQD = XQ + WQ * (DUAL ? 2 : 1);
    constexpr int GS = BF ? 8 : 4, WB16 = DUAL ? CB / 2 : CB;
    uint8_t *const sc = mg_lds + T::RING;
    ghip_u32x4 next[NSL], raw[NQD];
    uint32_t sx[BF ? 1 : RB], sw[BF ? 2 * CB : CB];
    auto scale_load = [&](uint32_t word) {
        fg_each<NSL>([&](auto i_c) {
            constexpr uint32_t i = decltype(i_c)::value;
            const uint32_t u = wv + NW * i, first = u < XU ? 0u : u < XU + WU ? XU : XU + WU;
            const uint8_t *const s = u < XU ? p.xs : !DUAL || u < XU + WU ? p.ws : p.ws2;
            const uint32_t base = u < XU ? row0 : col0, live = u < XU ? rows : u < NU ? cols : 0u;
            const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc((void *)(s + (size_t)base * lds), 0, live * lds, 0x20000);
            const uint32_t row = 64u * (u - first) + lane;
            if (word + 4u <= words) {
                next[i] = __builtin_amdgcn_raw_buffer_load_b128(r, mg_scale(row, word, words), 0, 0);
            } else {
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) next[i][e] = __builtin_amdgcn_raw_buffer_load_b32(r, mg_scale(row, word + e, words), 0, 0);
            }
        });
    };
    auto scale_store = [&]() {
        fg_each<NSL>([&](auto i_c) {
            constexpr uint32_t i = decltype(i_c)::value;
            const uint32_t u = wv + NW * i;
            if (NU % NW == 0 || u < NU) *(ghip_u32x4 *)(sc + 1024u * u + 16u * lane) = next[i];
        });
    };
    /* quad q of a wave's blocks: x's, W's, the second matrix's; of two or one, lanes
     * behind these read the same rows again */
    const uint32_t scx = mg_scale_at(0u, wr * RB, RB, lane), scw = mg_scale_at(XU, wc * WB16, WB16, lane);
    auto scale_read = [&](auto q_c) {
        constexpr int q = decltype(q_c)::value;
        constexpr uint32_t at = q < XQ ? 1024u * q : q < XQ + WQ ? 1024u * (q - XQ) : 1024u * (q - XQ - WQ + WU);
        raw[q] = *(const ghip_u32x4 *)(sc + (q < XQ ? scx : scw) + at);
    };
    auto scale_turn = [&](auto q_c) { raw[decltype(q_c)::value] = mg_turn(raw[decltype(q_c)::value]); };
    /* BF16: a row's steps take half a word each; sw[c] has the even ones' scales (lane
     * groups 0 and 1 block 0 of the word, 2 and 3 block 1), sw[CB + c] the odd ones' */
    auto scale_take = [&]() {
        if constexpr (!BF)
            fg_each<RB>([&](auto r_c) {
                constexpr int r = decltype(r_c)::value;
                sx[r] = mg_keep(raw[r / 4][r % 4]);
            });
        fg_each<CB>([&](auto c_c) {
            constexpr int c = decltype(c_c)::value, i = DUAL ? c >> 1 : c;
            const uint32_t v = raw[XQ + (DUAL && (c & 1) ? WQ : 0) + i / 4][i % 4];
            if constexpr (BF) {
                const auto h = __builtin_amdgcn_permlane32_swap(v, v, false, false);
#pragma unroll
                for (int e = 0; e < 2; e++) {
                    const auto q = __builtin_amdgcn_permlane16_swap(h[e], h[e], false, false);
                    sw[e * CB + c] = g & 2u ? q[1] : q[0];
                }
            } else {
                sw[c] = mg_keep(v);
            }
        });
    };
    /* BF16: half h of W's block c of step j, of set S; past: its k is past K, where the
     * codes are zeros and the scale is any byte */
    auto dequant = [&](auto set_c, auto c_c, auto h_c, uint32_t j, bool past) {
        if constexpr (BF) {
            constexpr int S = decltype(set_c)::value, c = decltype(c_c)::value, h = decltype(h_c)::value;
            const uint32_t b = sw[S * CB + c] >> (8u * ((j >> 1) & 3u)) & 255u;
            const ghip_u32x4 d = mx_fp4_bf16(codes[c][h], past ? 1.0f : __uint_as_float(b << 23));
#pragma unroll
            for (int e = 0; e < 4; e++) wa[S][c][4 * h + e] = (int)d[e];
        }
    };
    /* The step that K cuts: its blocks past K have any scale. A step past K (an odd
     * number of them) has zeros for codes and scales */
    const uint32_t nb = p.K >> 5, rem = nb & 3u;
    ghip_f32x4 acc[RB][CB];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int c = 0; c < CB; c++) acc[r][c] = (ghip_f32x4){0.f, 0.f, 0.f, 0.f};

    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    const uint32_t all = (nst + 1u) & ~1u;               /* steps, in pairs */
    scale_load(0u);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (uint32_t j = 0; j < (uint32_t)R; j++)
        if (j < all) {
#pragma unroll
            for (uint32_t i = 0; i < LPS; i++) load(i);
            next_load();
        }
    ghip_wait_stages<LPS, R - 1>(min(all, (uint32_t)R) - 1u);
    scale_store();
    __builtin_amdgcn_sched_barrier(0);
    scale_load(4u);
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    fg_each<NQD>(scale_read);
    fg_each<NQD>(scale_turn);
    scale_take();
    fg_each<CB>([&](auto c) { read_b(S0{}, c, mg_lds); });
    fg_each<RB>([&](auto r) { read_a(S0{}, r, mg_lds); });
    if constexpr (BF)
        fg_each<2 * CB>([&](auto q) {
            constexpr int Q = decltype(q)::value;
            dequant(S0{}, std::integral_constant<int, Q / 2>{}, std::integral_constant<int, Q % 2>{}, 0u, (g >> 1) >= nb);
        });

    uint32_t rs = 0;                                     /* slot of step j */
    auto step = [&](uint32_t j, auto quarter_c, auto main_c) {
        constexpr int QU = decltype(quarter_c)::value, S = QU & 1;
        constexpr bool MAIN = decltype(main_c)::value;
        const bool more = MAIN || j + 1u < all, loads = MAIN || j + R < all;
        /* own loads of step j + 1 done, own reads of step j done; after the barrier that holds
         * for every wave. Behind them are those of R - 2 steps, and scales where one of these
         * loaded some (fewer are assumed where that is not known: a longer wait) */
        if (MAIN) mg_wait<(R - 2) * LPS + (BF ? 0 : NSL * mg_third(QU, R - 2))>();
        else ghip_wait_stages<LPS, R - 2>(more ? all - 2u - j : 0u);
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!MAIN && !BF)
            if (rem && j + 1u >= nst && g >= rem) {
                fg_each<RB>([&](auto r) { sx[decltype(r)::value] = 0x7f7f7f7fu; });
                fg_each<CB>([&](auto c) { sw[decltype(c)::value] = 0x7f7f7f7fu; });
                asm volatile("s_nop 3");                 /* VALU to MFMA */
                __builtin_amdgcn_sched_barrier(0);
            }
        /* the next scales: to LDS in a third step, from there in the fourth */
        const bool scales = !BF || (j & 4u);
        if constexpr (QU == 2)
            if (scales) {
                scale_store();
                __builtin_amdgcn_sched_barrier(0);
                scale_load(4u * (j / GS + 2u));
                __builtin_amdgcn_sched_barrier(0);
            }
        if constexpr (QU == 3)
            if (scales) {
                fg_each<NQD>(scale_read);
                __builtin_amdgcn_sched_barrier(0);
            }
        const uint32_t ns = !more ? rs : rs == (R - 1u) * SLOT ? 0u : rs + SLOT;
        const uint8_t *st = mg_lds + ns;
        using NS = std::integral_constant<int, S ^ 1>;
        const bool past = !MAIN && 2u * (j + 1u) + (g >> 1) >= nb;
        constexpr int NL = (int)LPS, CU = CB + 1, TE = BF ? NM / 2 : NM;
        fg_each<NM>([&](auto slot) {
            constexpr int I = decltype(slot)::value, Rr = I / CB, K = I % CB;
            constexpr int C = Rr & 1 ? CB - 1 - K : K;
            const XReg &x = Rr == RB - 1 ? xl[S] : xa[Rr];
            if constexpr (BF) {
                const auto half = [](const mg_i32x8 &v, auto h) {
                    constexpr int H = 4 * decltype(h)::value;
                    return __builtin_bit_cast(ghip_bf16x8, __builtin_shufflevector(v, v, H, H + 1, H + 2, H + 3));
                };
                fg_mfma(acc[Rr][C], half(wa[S][C], S0{}), half(x, S0{}));
                fg_mfma(acc[Rr][C], half(wa[S][C], S1{}), half(x, S1{}));
            } else {
                mg_mfma<QU>(acc[Rr][C], wa[S][C], x, sw[C], sx[Rr]);
            }
            /* W and x's last block over the first RB - 1 rows (codes for BF16 over the first
             * third, dequantized behind), x's others behind their own */
            constexpr int BE = BF ? NM / 3 : NM - CB, NQ = BF ? 2 * CB : 0;
            constexpr int B0 = fg_spread(CU, I, 0, BE), B1 = fg_spread(CU, I + 1, 0, BE);
            constexpr int Q0 = fg_spread(NQ, I, NM / 2, NM), Q1 = fg_spread(NQ, I + 1, NM / 2, NM);
            constexpr int L0 = fg_spread(NL, I, 0, NM), L1 = fg_spread(NL, I + 1, 0, NM);
            fg_each<B1 - B0>([&](auto k) {
                constexpr int O = B0 + decltype(k)::value;
                if constexpr (O < CB) read_b(NS{}, std::integral_constant<int, O>{}, st);
                else read_a(NS{}, std::integral_constant<int, RB - 1>{}, st);
            });
            constexpr int T0 = QU == 3 ? fg_spread(NQD, I, TE / 4, TE) : 0, T1 = QU == 3 ? fg_spread(NQD, I + 1, TE / 4, TE) : 0;
            if constexpr (T1 > T0)
                if (scales) {
                    fg_each<T1 - T0>([&](auto k) { scale_turn(std::integral_constant<int, T0 + decltype(k)::value>{}); });
                    if constexpr (BF && T1 == NQD) scale_take();   /* all of this step's are used up */
                }
            fg_each<Q1 - Q0>([&](auto k) {
                constexpr int Q = Q0 + decltype(k)::value;
                dequant(NS{}, std::integral_constant<int, Q / 2>{}, std::integral_constant<int, Q % 2>{}, j + 1u, past);
            });
            constexpr bool A = Rr > 0 && K == 0;
            if constexpr (A) read_a(NS{}, std::integral_constant<int, Rr - 1>{}, st);
            if constexpr (L1 > L0)
                if (loads) fg_each<L1 - L0>([&](auto k) { load(L0 + decltype(k)::value); });
            if constexpr (A || B1 > B0 || Q1 > Q0 || L1 > L0 || T1 > T0) __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (!BF && QU == 3) scale_take();
        if (loads) next_load();
        __builtin_amdgcn_sched_barrier(0);
        rs = ns;
    };
    uint32_t j = 0;
    for (; j + 3u + R < all; j += 4u) fg_each<4>([&](auto q) { step(j + decltype(q)::value, q, std::true_type{}); });
    for (; j < all; j += 4u)
        fg_each<4>([&](auto q) {
            if (j + decltype(q)::value < all) step(j + decltype(q)::value, q, std::false_type{});
        });
    fg_settle(acc);

    /* the sums through LDS, 8 columns of a row a lane (as k_ffn_gemm.h) */
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    constexpr uint32_t PER = T::RING / NW;
    constexpr int G = PER >= 1024u * CB * RB ? RB : PER >= 512u * CB * RB ? RB / 2 : PER >= 256u * CB * RB ? RB / 4 : 1;
    static_assert(PER >= 1024u * CB * G && RB % G == 0, "epilogue staging");
    static_assert(G * (DUAL ? CB : 2 * CB) % 4 == 0, "whole passes over the staged rows");
    constexpr uint32_t RBY = 64u * CB;
    constexpr uint32_t LPR = DUAL ? CB : 2u * CB;
    constexpr int IT = G * (int)LPR / 4, U = IT % 8 == 0 ? 8 : IT % 4 == 0 ? 4 : IT % 2 == 0 ? 2 : 1;
    uint8_t *stg = mg_lds + wv * (1024u * CB * G);
    auto spot = [&](uint32_t row, uint32_t q) {
        return row * RBY + 16u * (q ^ (CB >= 4 ? row & 15u : CB == 2 ? (row >> 1) & 7u : (row >> 2) & 3u));
    };
    const uint32_t pc = lane % LPR, c0 = (DUAL ? 8u : 16u) * CB * wc + 8u * pc, n0 = col0 + c0;
    const uint32_t m0 = row0 + 16u * wr * RB + lane / LPR;
    const uint32_t q0 = DUAL ? 8u * (pc >> 1) + 2u * (pc & 1u) : 2u * pc;
    constexpr bool BIAS = MODE == GHIP_EP_LINEAR;
    const bool live = c0 < cols, whole = n0 + 8u <= p.N;
    const bool fast = (p.N & 7u) == 0u || cols == OUTN;
    const uint32_t nc = live ? n0 : col0;
    auto load8 = [&](auto fast_c, const uint16_t *row, float (&v)[8]) {
        if (decltype(fast_c)::value) {
            ghip_u32x4 d;
            __builtin_memcpy(&d, row + nc, 16);
            fg_unpack(d, v);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) v[e] = n0 + e < p.N ? ghip_bf16_f32(row[n0 + e]) : 0.0f;
        }
    };
    auto store8 = [&](auto fast_c, uint16_t *row, const float (&v)[8]) {
        const ghip_u32x4 d = fg_pack(v);
        if (decltype(fast_c)::value || whole) {
            __builtin_memcpy(row + n0, &d, 16);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++)
                if (n0 + e < p.N) row[n0 + e] = (uint16_t)(d[e >> 1] >> (16u * (e & 1u)));
        }
    };
    float bias[8] = {};
    if constexpr (BIAS)
        if (ep.bias) {
            if (fast) load8(std::true_type{}, ep.bias, bias);
            else load8(std::false_type{}, ep.bias, bias);
        }
    /* The residual, U rows ahead: the first ones come while the sums are laid out, the next
     * while U are computed (4096 x 4096 x 12288 in MXFP4, one round of 256 x 256 tiles: 112
     * us, 118 with each batch loaded where it was needed) */
    ghip_u32x4 res[U];
    const bool ahead = BIAS && fast && ep.in;
    auto fetch = [&](int at) {
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint32_t m = min(m0 + (at + u) * (64u / LPR), p.M - 1u);
            __builtin_memcpy(&res[u], ep.in + (size_t)m * ep.ldin + nc, 16);
        }
    };
    if constexpr (BIAS)
        if (ahead) fetch(0);
    ghip_with_act(ep.act, [&](auto act) {
        auto values = [&](uint32_t lr, const float (&in)[8], float (&o)[8]) {
            float s0[8], s1[8] = {}, none;
            auto read8 = [&](uint32_t q, float (&v)[8]) {
#pragma unroll
                for (uint32_t d = 0; d < 2; d++) {
                    const ghip_f32x4 x = *(const ghip_f32x4 *)(stg + spot(lr, q + d));
#pragma unroll
                    for (int e = 0; e < 4; e++) v[4 * d + e] = x[e];
                }
            };
            read8(q0, s0);
            if constexpr (DUAL) read8(q0 + 4u, s1);
#pragma unroll
            for (int e = 0; e < 8; e++)
                ghip_ep_value<MODE, decltype(act)::value>(s0[e], s1[e], bias[e], in[e], ep.limit, o[e], none);
        };
#pragma unroll
        for (int rg = 0; rg < RB; rg += G) {
#pragma unroll
            for (int r = 0; r < G; r++)
#pragma unroll
                for (uint32_t c = 0; c < CB; c++)
                    *(ghip_f32x4 *)(stg + spot(16u * r + n, 4u * c + g)) = acc[rg + r][c];
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_wave_barrier();
            const uint32_t mg = m0 + 16u * rg;
            auto rows_out = [&](auto fast_c, auto u_c) {
                constexpr int UU = decltype(u_c)::value;
#pragma unroll 1
                for (int it = 0; it < IT; it += UU) {
                    float in[UU][8] = {};
                    if constexpr (BIAS && decltype(fast_c)::value) {
                        if (ahead) {
#pragma unroll
                            for (int u = 0; u < UU; u++) fg_unpack(res[u], in[u]);
                            const int next = rg * (int)LPR / 4 + it + U;
                            if (next < RB * (int)LPR / 4) fetch(next);
                        }
                    } else if constexpr (BIAS) {
                        if (ep.in) load8(fast_c, ep.in + (size_t)min(mg + it * (64u / LPR), p.M - 1u) * ep.ldin, in[0]);
                    }
#pragma unroll
                    for (int u = 0; u < UU; u++) {
                        const uint32_t dr = (it + u) * (64u / LPR), m = mg + dr;
                        float o[8];
                        values(lane / LPR + dr, in[u], o);
                        if (m < p.M && live) store8(fast_c, ep.out + (size_t)m * ep.ldout, o);
                    }
                }
            };
            if (fast) rows_out(std::true_type{}, std::integral_constant<int, U>{});
            else rows_out(std::false_type{}, std::integral_constant<int, 1>{});
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_wave_barrier();
        }
    });
}

#endif /* K_MX_GEMM_H */
