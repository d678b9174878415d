/*
 * k_mx_gemm.h — the tiled product with MXFP4 weights (gfx950).
 */
#ifndef K_MX_GEMM_H
#define K_MX_GEMM_H

#include "ghip_mx.h"
#include "k_ffn_gemm.h"
#include "k_mx_addr.h"

typedef int mg_i32x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ void mg_dma4(const void *src, void *lds_wave) {
    __builtin_amdgcn_global_load_lds((ghip_glb_t *)src, (ghip_lds_t *)lds_wave, 4, 0, 0);
}

/* acc += w (16 rows of MXFP4) . x^T over 128 k, in place; sw, sx: the blocks' scales
 * in the low byte. As fg_mfma the compiler knows no MFMA in it. */
__device__ __forceinline__ void mg_mfma(ghip_f32x4 &acc, const ghip_u32x4 &w, const mg_i32x8 &x, uint32_t sw,
                                        uint32_t sx) {
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4"
        : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
}
__device__ __forceinline__ void mg_mfma(ghip_f32x4 &acc, const ghip_u32x4 &w, const ghip_u32x4 &x, uint32_t sw,
                                        uint32_t sx) {
    asm("v_mfma_scale_f32_16x16x128_f8f6f4 %0, %1, %2, %0, %3, %4 op_sel_hi:[0,0,0] cbsz:4 blgp:4"
        : "+a"(acc) : "v"(w), "v"(x), "v"(sw), "v"(sx));
}

template <int MODE, int XT, int WM, int WN, int RB, int CB, int R>
struct MgTile {
    static constexpr bool DUAL = ghip_ep_dual(MODE), BF = XT == GHIP_BF16;
    static constexpr uint32_t NW = WM * WN, BM = 16u * RB * WM, BN = 16u * CB * WN, OUTN = DUAL ? BN / 2 : BN;
    /* a step: k, bytes of a row of x and of W, words of scales */
    static constexpr uint32_t KS = BF ? 64u : 128u, XB = XT == GHIP_MXFP4 ? 64u : 128u, WB = BF ? 32u : 64u;
    static constexpr uint32_t SBM = BF ? 0u : BM, NSL = (SBM + BN + 64u * NW - 1u) / (64u * NW);
    static constexpr uint32_t AST = BM * XB, BST = BN * WB, SST = NSL * NW * 256u;
    static constexpr uint32_t SLOT = AST + BST + SST, RING = R * SLOT;
    static constexpr uint32_t NAL = AST / 1024u / NW, NBL = BST / 1024u / NW, LPS = NAL + NBL + NSL;
    static_assert(AST % (1024u * NW) == 0 && BST % (1024u * NW) == 0, "whole loads");
    static_assert(RING <= FG_LDS_MAX && R >= 2 && (R - 2) * LPS <= 63, "ring, waits");
    static_assert(!DUAL || CB % 2 == 0, "gate and up blocks alternate");
};

template <int MODE, int XT, int WM, int WN, int RB, int CB, int R>
__global__ __launch_bounds__(64 * WM * WN, 1) void k_mx_gemm(GhipMxProd p, GhipEp ep, uint32_t mt,
                                                             uint32_t nt) {
    using T = MgTile<MODE, XT, WM, WN, RB, CB, R>;
    constexpr bool DUAL = T::DUAL, BF = T::BF;
    constexpr uint32_t NW = T::NW, BM = T::BM, BN = T::BN, OUTN = T::OUTN, XB = T::XB, WB = T::WB, KS = T::KS;
    constexpr uint32_t NAL = T::NAL, NBL = T::NBL, NSL = T::NSL, LPS = T::LPS, SLOT = T::SLOT;
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
    const uint8_t *ps[NSL];
#pragma unroll
    for (uint32_t i = 0; i < NSL; i++) {
        const uint32_t e = (wv + NW * i) * 64u + lane;
        bool second;
        const uint32_t c = mg_scale_row(e, T::SBM, BN, DUAL, second);
        ps[i] = e < T::SBM ? p.xs + (size_t)min(row0 + e, p.M - 1u) * lds
                       : (second ? p.ws2 : p.ws) + (size_t)min(col0 + c, p.N - 1u) * lds;
    }
    uint32_t jl = 0, sl = 0;                             /* the next step to load, its slot */
    int32_t xleft = (int32_t)xrow, wleft = (int32_t)wb;
    auto load = [&](uint32_t i) {
        if (i < NAL) {
            const uint32_t off = mg_cut(ao + i * astep, aq, xleft);
            fg_dma16(pa, aspan, off, mg_lds + sl + (wv + NW * i) * 1024u);
        } else if (i < NAL + NBL) {
            const uint32_t off = mg_cut(bo + (i - NAL) * bstep, bq, wleft);
            fg_dma16(pb, bspan, off, mg_lds + sl + T::AST + (wv + NW * (i - NAL)) * 1024u);
        } else {
            const uint32_t k = i - NAL - NBL;
            mg_dma4(ps[k] + 4u * min(BF ? jl >> 1 : jl, words - 1u), mg_lds + sl + T::AST + T::BST + (wv + NW * k) * 256u);
        }
    };
    auto next_load = [&]() {
        jl++;
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
    uint32_t sx[RB], sl_[2], sw[2][CB];
    constexpr uint32_t SC = T::AST + T::BST;
    const uint32_t a0 = mg_at_x<XB>(wr * RB, n, g, 0, BF), a1 = mg_at_x<XB>(wr * RB, n, g, 1, BF);
    const uint32_t b0 = mg_at_w<WB, CB>(T::AST, wc, n, g, DUAL);
    const uint32_t as = mg_at_sx(SC, wr * RB, n) + g, bs = mg_at_sw(SC, T::SBM, wc * CB, n, DUAL) + (BF ? g >> 1 : g);
    auto read_x = [&](XReg &x, uint32_t &s, int r, const uint8_t *st) {
        const ghip_u32x4 lo = *(const ghip_u32x4 *)(st + a0 + r * (16u * XB));
        if constexpr (XB == 128u) {
            const ghip_u32x4 hi = *(const ghip_u32x4 *)(st + a1 + r * (16u * XB));
            x = (mg_i32x8){(int)lo[0], (int)lo[1], (int)lo[2], (int)lo[3], (int)hi[0], (int)hi[1], (int)hi[2], (int)hi[3]};
        } else {
            x = lo;
        }
        if constexpr (!BF) s = st[as + 64u * r];
    };
    auto read_a = [&](auto set_c, auto r_c, const uint8_t *st) {
        constexpr int S = decltype(set_c)::value, r = decltype(r_c)::value;
        if constexpr (r == RB - 1) read_x(xl[S], sl_[S], r, st);
        else read_x(xa[r], sx[r], r, st);
    };
    /* beside BF16: steps start in pairs, so that set S has bytes 2 S and 2 S + 1 of the word */
    auto read_b = [&](auto set_c, auto c_c, const uint8_t *st) {
        constexpr int S = decltype(set_c)::value, c = decltype(c_c)::value;
        if constexpr (BF) codes[c] = *(const ghip_u32x2 *)(st + b0 + mg_w_step<WB>(c, DUAL));
        else wa[S][c] = *(const ghip_u32x4 *)(st + b0 + mg_w_step<WB>(c, DUAL));
        sw[S][c] = st[bs + mg_sw_step(c, BN, DUAL) + (BF ? 2 * S : 0)];
    };
    /* BF16: half h of W's block c of the next step; past: its k is past K, where the codes
     * are zeros and the scale is any byte */
    auto dequant = [&](auto set_c, auto c_c, auto h_c, bool past) {
        if constexpr (BF) {
            constexpr int S = decltype(set_c)::value, c = decltype(c_c)::value, h = decltype(h_c)::value;
            const ghip_u32x4 d = mx_fp4_bf16(codes[c][h], past ? 1.0f : __uint_as_float(sw[S][c] << 23));
#pragma unroll
            for (int e = 0; e < 4; e++) wa[S][c][4 * h + e] = (int)d[e];
        }
    };
    /* The step that K cuts: its blocks past K have any scale. A step past K (an odd
     * number of them) has zeros for codes, and the last one's scales */
    const uint32_t nb = p.K >> 5, rem = nb & 3u;
    ghip_f32x4 acc[RB][CB];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int c = 0; c < CB; c++) acc[r][c] = (ghip_f32x4){0.f, 0.f, 0.f, 0.f};

    using S0 = std::integral_constant<int, 0>;
    using S1 = std::integral_constant<int, 1>;
    const uint32_t all = (nst + 1u) & ~1u;               /* steps, in pairs */
#pragma unroll
    for (uint32_t j = 0; j < (uint32_t)R; j++)
        if (j < all) {
#pragma unroll
            for (uint32_t i = 0; i < LPS; i++) load(i);
            next_load();
        }
    ghip_wait_stages<LPS, R - 1>(min(all, (uint32_t)R) - 1u);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    fg_each<CB>([&](auto c) { read_b(S0{}, c, mg_lds); });
    fg_each<RB>([&](auto r) { read_a(S0{}, r, mg_lds); });
    if constexpr (BF)
        fg_each<2 * CB>([&](auto q) {
            constexpr int Q = decltype(q)::value;
            dequant(S0{}, std::integral_constant<int, Q / 2>{}, std::integral_constant<int, Q % 2>{}, g >= 2u * nb);
        });

    uint32_t rs = 0;                                     /* slot of step j */
    auto step = [&](uint32_t j, auto set_c, auto main_c) {
        constexpr int S = decltype(set_c)::value;
        constexpr bool MAIN = decltype(main_c)::value;
        const bool more = MAIN || j + 1u < all;
        /* own loads of step j + 1 done, own reads of step j done; after the barrier that
         * holds for every wave */
        if (MAIN) GHIP_VMCNT((R - 2) * LPS);
        else ghip_wait_stages<LPS, R - 2>(more ? all - 2u - j : 0u);
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (!MAIN && !BF)
            if (rem && j + 1u >= nst && g >= rem) {
                fg_each<RB - 1>([&](auto r) { sx[decltype(r)::value] = 127u; });
                sl_[S] = 127u;
                fg_each<CB>([&](auto c) { sw[S][decltype(c)::value] = 127u; });
                asm volatile("s_nop 3");                 /* VALU to MFMA */
                __builtin_amdgcn_sched_barrier(0);
            }
        const uint32_t ns = !more ? rs : rs == (R - 1u) * SLOT ? 0u : rs + SLOT;
        const uint8_t *st = mg_lds + ns;
        using NS = std::integral_constant<int, S ^ 1>;
        const bool past = !MAIN && 2u * (j + 1u) + (g >> 1) >= nb;
        constexpr int NL = MAIN ? (int)LPS : 0, CU = CB + 1;
        fg_each<NM>([&](auto slot) {
            constexpr int I = decltype(slot)::value, Rr = I / CB, K = I % CB;
            constexpr int C = Rr & 1 ? CB - 1 - K : K;
            auto mma = [&](const XReg &x, uint32_t s) {
                if constexpr (BF) {
                    const auto half = [](const mg_i32x8 &v, auto h) {
                        constexpr int H = 4 * decltype(h)::value;
                        return __builtin_bit_cast(ghip_bf16x8, __builtin_shufflevector(v, v, H, H + 1, H + 2, H + 3));
                    };
                    fg_mfma(acc[Rr][C], half(wa[S][C], S0{}), half(x, S0{}));
                    fg_mfma(acc[Rr][C], half(wa[S][C], S1{}), half(x, S1{}));
                } else {
                    mg_mfma(acc[Rr][C], wa[S][C], x, sw[S][C], s);
                }
            };
            if constexpr (Rr == RB - 1) mma(xl[S], sl_[S]);
            else mma(xa[Rr], sx[Rr]);
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
            fg_each<Q1 - Q0>([&](auto k) {
                constexpr int Q = Q0 + decltype(k)::value;
                dequant(NS{}, std::integral_constant<int, Q / 2>{}, std::integral_constant<int, Q % 2>{}, past);
            });
            constexpr bool A = Rr > 0 && K == 0;
            if constexpr (A) read_a(NS{}, std::integral_constant<int, Rr - 1>{}, st);
            fg_each<L1 - L0>([&](auto k) { load(L0 + decltype(k)::value); });
            if constexpr (A || B1 > B0 || Q1 > Q0 || L1 > L0) __builtin_amdgcn_sched_barrier(0);
        });
        if constexpr (MAIN) next_load();
        __builtin_amdgcn_sched_barrier(0);
        rs = ns;
    };
    uint32_t j = 0;
    for (; j + R + 1u < all; j += 2u) {
        step(j, S0{}, std::true_type{});
        step(j + 1u, S1{}, std::true_type{});
    }
    if constexpr (R & 1)                                 /* one more to load */
        if (j + R < all) {
            step(j, S0{}, std::true_type{});
            step(j + 1u, S1{}, std::false_type{});
            j += 2u;
        }
    for (; j < all; j += 2u) {
        step(j, S0{}, std::false_type{});
        step(j + 1u, S1{}, std::false_type{});
    }
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
    constexpr int IT = G * (int)LPR / 4, U = IT % 4 == 0 ? 4 : IT % 2 == 0 ? 2 : 1;
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
                    if constexpr (BIAS)
                        if (ep.in) {
#pragma unroll
                            for (int u = 0; u < UU; u++) {
                                const uint32_t m = min(mg + (it + u) * (64u / LPR), p.M - 1u);
                                load8(fast_c, ep.in + (size_t)m * ep.ldin, in[u]);
                            }
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
