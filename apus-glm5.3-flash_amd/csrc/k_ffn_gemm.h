/*
 * k_ffn_gemm.h — the tiled MFMA product of the dense feed-forward operators
 * (gfx950): out[m, n] = epilogue(sum_k A(m, k) B(n, k)); instantiated by
 * k_ffn_nt.hip (forward) and k_ffn_bwd.hip (backward).
 *
 * A workgroup of WM x WN = 4 waves owns 16 RB WM rows of A x 16 CB WN rows of B;
 * wave (wr, wc) computes 16 RB x 16 CB outputs with v_mfma_f32_16x16x32_bf16, B
 * as the A operand of the instruction, so a lane ends with four consecutive
 * columns of one output row. k is walked in stages of 64, two MFMA steps each.
 *
 * What bounds it, and what follows. A full chip of these products is at its
 * power limit (4096 x 4096 x 4096 of zeros runs at 1800 TFLOP/s, of normal
 * values at 1430), so what costs energy or idles counts:
 *   - 16x16x32 MFMAs, which move half the accumulators of 32x32x16 a product
 *     (1180 -> 1290), walked in a snake so that one operand stays (+2%);
 *   - accumulators of the largest tile fill all 256 AGPRs; the MFMAs are inline
 *     asm that updates them in place, which the compiler's register allocation
 *     does not keep (it moved half of them every stage: 1116);
 *   - 128 x 128 outputs a wave, the least LDS reads a product; one wave a SIMD,
 *     whose order of MFMAs, operand reads and loads is written out (evenly
 *     spread loads: +4%; in a burst after the barrier they block the issue);
 *   - loads go straight to LDS and are issued L stages ahead: A's in the first
 *     step (a ring of L + 1 slots), B's after the stage's one barrier, which
 *     frees their slot (a ring of L). L = 2 with the largest tile fills the
 *     160 KB (one stage ahead: 1380 against 1505 at 4096 x 4096 x 12288, from
 *     HBM).
 *
 * Operand layouts. 0: k is the fast index in memory (x, W in the forward). The
 * stage is [row][64 k], whole 128-byte lines, 16-byte piece p of row r at p ^
 * fg_rot8(r); an operand of 8 k values is one ds_read_b128. 1: the row is
 * (W in dx, dz and x in dW). The stage is [64 k][rows], 32-byte slots XORed
 * with k (fg_swizzle), and an operand is two ds_read_b64_tr_b16: each
 * transposes 4 k x 16 rows inside 16 lanes, so no transposed copy of a matrix
 * is made. In both, lane group g of MFMA step s takes k = 16 g + 8 s + [0, 8),
 * so either layout may meet the other. SQ_LDS_BANK_CONFLICT is 0 to 3% of the
 * LDS cycles.
 *
 * Rows past the matrix and k past its end are given an offset outside the
 * buffer, which loads zeros: no other row is read in their place and a ragged
 * K needs no separate kernel.
 *
 * FP8 weights lie in LDS as codes, [row][64 codes], 16-byte piece p of row r at
 * p ^ fg_rot4(r): one read gives the 16 codes of both steps, which are
 * dequantized bit-exactly in registers between the MFMAs of the step before
 * (against writing bf16 back to LDS it takes half the loads and writes). Its
 * waves lie side by side (WM = 1), so that no two dequantize the same codes.
 *
 * Dual modes (gate and up): the tile's B rows alternate in blocks of 16 between
 * the two matrices, so a lane holds g and u of the same columns and the product
 * of the two needs no exchange.
 *
 * The epilogue passes the sums through a wave-private piece of the ring 16 rows
 * at a time, so that bias, residual and output are 16-byte accesses along a
 * row.
 */
#ifndef K_FFN_GEMM_H
#define K_FFN_GEMM_H

#include <utility>

#include "ghip_epilogue.h"
#include "k_ffn_addr.h"

typedef short fg_s16x4 __attribute__((ext_vector_type(4)));

#define FG_LDS_MAX (160u * 1024u)

__device__ __forceinline__ void fg_dma16(const void *base, uint32_t span, uint32_t off,
                                         void *lds_wave) {
    const __amdgpu_buffer_rsrc_t r =
        __builtin_amdgcn_make_buffer_rsrc((void *)base, 0, span, 0x20000);
    __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (ghip_lds_t *)lds_wave, 16, off, 0, 0, 0);
}

/* acc += b . a, in place. The compiler knows no MFMA in it: operands are
 * written (by LDS reads or VALU) at least two instructions ahead, which
 * tests/test_ffn_asm.py checks in the built code, and sums are read after
 * fg_settle. */
__device__ __forceinline__ void fg_mfma(ghip_f32x4 &acc, const ghip_bf16x8 &b,
                                        const ghip_bf16x8 &a) {
    asm("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc) : "v"(b), "v"(a));
}
/* The last MFMAs have written their sums (32 wait states; they need 4 passes). */
template <int R, int C>
__device__ __forceinline__ void fg_settle(ghip_f32x4 (&acc)[R][C]) {
    asm volatile("s_nop 15\n\ts_nop 15" : "+a"(acc[R - 1][C - 1]));
#pragma unroll
    for (int r = 0; r < R; r++)
#pragma unroll
        for (int c = 0; c < C; c++) asm volatile("" : "+a"(acc[r][c]));
}

/* 4 k x 16 rows of a layout-1 stage, transposed inside 16 lanes: lane i gives
 * the address of 4 values of k row i / 4 and gets the 4 k of row i. The
 * restrict keeps the compiler from waiting for every load to LDS in flight
 * before each of these reads, as it does for a pointer it knows nothing of (dx
 * of 1024 x 4096 x 4096: 52 -> 38 us); the stages' own waits and barriers order
 * the two. */
typedef __attribute__((address_space(3))) fg_s16x4 fg_lds_s16x4;
__device__ __forceinline__ fg_s16x4 fg_read_tr(fg_lds_s16x4 *__restrict p) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16(p);
}

/* f(0), f(1), ... f(N - 1), the argument a constant */
template <typename F, int... I>
__device__ __forceinline__ void fg_each_of(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void fg_each(F f) {
    fg_each_of(f, std::make_integer_sequence<int, N>{});
}
/* Of n things spread over slots [from, to): how many come in slots before i. */
constexpr int fg_spread(int n, int i, int from, int to) {
    return i <= from ? 0 : i >= to ? n : (n * (i - from) + (to - from) - 1) / (to - from);
}

/* 8 bf16 values as f32, and back with one rounding */
__device__ __forceinline__ void fg_unpack(const ghip_u32x4 &d, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e++) v[e] = ghip_bf16_f32(e & 1 ? d[e >> 1] >> 16 : d[e >> 1] & 0xffffu);
}
__device__ __forceinline__ ghip_u32x4 fg_pack(const float (&v)[8]) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    ghip_u32x4 d;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        bf2 t;
        t[0] = (__bf16)v[2 * e];
        t[1] = (__bf16)v[2 * e + 1];
        d[e] = __builtin_bit_cast(uint32_t, t);
    }
    return d;
}

/* W8: 0 bf16 weights, 1 FP8 codes, 2 FP8 codes with NaN codes among them */
template <int MODE, int W8, int AL, int BL, int WM, int RB, int CB, int L>
__device__ __forceinline__ void fg_product(const GhipProd &p, const GhipEp &ep, uint32_t mt,
                                           uint32_t nt, uint32_t block, uint32_t blocks) {
    constexpr bool DUAL = ghip_ep_dual(MODE), FP8 = W8 != 0;
    constexpr uint32_t WN = 4 / WM, BM = 16u * RB * WM, BN = 16u * CB * WN;
    constexpr uint32_t OUTN = DUAL ? BN / 2 : BN;        /* output columns of a tile */
    constexpr uint32_t AST = BM * 128u, BST = BN * (FP8 ? 64u : 128u);  /* slot bytes */
    constexpr uint32_t NAL = BM / 32u, NBL = FP8 ? BN / 64u : BN / 32u, LPS = NAL + NBL;
    constexpr uint32_t RING = (L + 1u) * AST + L * BST;
    constexpr int NM = RB * CB;                          /* MFMAs of a step */
    static_assert(RING <= FG_LDS_MAX, "ring");
    static_assert(WM * WN == 4 && BM % 32 == 0 && BN % (FP8 ? 64 : 32) == 0, "waves, whole loads");
    static_assert(L >= 2 && (L - 1) * NAL + (L - 2) * NBL <= 63 && (L - 1) * LPS <= 63, "waits");
    static_assert((!DUAL || CB % 2 == 0) && (!FP8 || (BL == 0 && 128 % (16 * CB) == 0)), "columns");
    extern __shared__ __attribute__((aligned(1024))) uint8_t fg_lds[];
    uint8_t *bring = fg_lds + (L + 1u) * AST;
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wr = wv / WN, wc = wv % WN, n = lane & 15u, g = lane >> 4;

    /* tile t of block b: the workgroups of one XCD (b % 8) take a run of consecutive
     * tiles, which go down 4 row tiles before the next column, so that an XCD's
     * L2 holds few rows of A and of B at a time (8192 x 24576 x 4096: 4 1.148
     * ms, 8 1.157, 16 1.18). A batch of two: the second half of the tiles is the
     * second product. Splits of k: each walks its share of the stages. */
    uint32_t t;
    {
        const uint32_t x = block & 7u, i = block >> 3, q = blocks >> 3, r = blocks & 7u;
        t = x * q + (x < r ? x : r) + i;
    }
    bool second = false;
    uint32_t split = 0;
    if constexpr (MODE == GHIP_EP_STORE) {
        split = t / (mt * nt);
        t -= split * (mt * nt);
        second = p.batch && split >= p.splits;
        if (second) split -= p.splits;
    }
    const uint32_t strip = t / (4u * nt), in_strip = t - strip * (4u * nt);
    const uint32_t sr = min(4u, mt - strip * 4u);
    const uint32_t row0 = (strip * 4u + in_strip % sr) * BM, col0 = in_strip / sr * OUTN;
    const uint32_t rows = min(p.M - row0, BM), cols = min(p.N - col0, OUTN);
    const uint32_t nst1 = (p.K + 63u) >> 6;              /* stages of one product */
    const uint32_t all = MODE == GHIP_EP_STORE && p.a2 && !p.batch ? 2u * nst1 : nst1;
    const uint32_t j0 = MODE == GHIP_EP_STORE ? (uint32_t)((uint64_t)all * split / p.splits) : 0u;
    const uint32_t nst =                                 /* of this split */
        MODE == GHIP_EP_STORE ? (uint32_t)((uint64_t)all * (split + 1u) / p.splits) - j0 : all;
    const size_t astep = AL == 0 ? 128u : (size_t)p.aks * 128u;
    const size_t bstep = BL == 0 ? (FP8 ? 64u : 128u) : (size_t)p.bks * 128u;
    const uint32_t lda = (uint32_t)(AL == 0 ? p.ars : p.aks);
    const uint32_t ldb = (uint32_t)(BL == 0 ? p.brs : p.bks);
    /* dual modes: this wave's loads are all of one matrix (16-row blocks of B
     * rows alternate, and a wave's lie an even number of blocks apart) */
    const bool up = DUAL && (FP8 ? wv & 1u : wv >> 1);
    auto base_a = [&](const uint16_t *a) {
        return (const uint8_t *)(a + (AL == 0 ? (size_t)row0 * p.ars : row0));
    };
    auto base_b = [&](const void *b) {
        return (const uint8_t *)b
               + (BL == 0 ? (size_t)col0 * p.brs : col0) * (FP8 ? (size_t)1 : (size_t)2);
    };
    /* the next stage to load: its address, number and slots */
    const bool late = second || j0 >= nst1;              /* starts in the second product */
    const uint8_t *pa = base_a(late ? p.a2 : p.a), *pb = base_b(late || up ? p.b2 : p.b);
    uint32_t ja = j0, jb = j0, sa = 0, sb = 0;
    if constexpr (MODE == GHIP_EP_STORE) {
        const size_t from = j0 >= nst1 ? j0 - nst1 : j0;
        pa += from * astep;
        pb += from * bstep;
    }

    /* this lane's offsets in a stage's loads (k_ffn_addr.h) */
    uint32_t ao[NAL], bo[NBL], akq = 0, bkq = 0;
    using LA = std::integral_constant<int, AL>;
    using LB = std::integral_constant<int, BL>;
    using WA = std::integral_constant<uint32_t, BM>;
    using WB = std::integral_constant<uint32_t, BN>;
#pragma unroll
    for (uint32_t i = 0; i < NAL; i++) ao[i] = fg_place<AL, BM>(wv + 4u * i, lane, rows, lda, akq);
#pragma unroll
    for (uint32_t i = 0; i < NBL; i++) {
        if constexpr (FP8) bo[i] = fg_place_codes(DUAL, wv + 4u * i, lane, cols, ldb, bkq);
        else if constexpr (DUAL) bo[i] = fg_place_dual(wv + 4u * i, lane, cols, ldb, bkq);
        else bo[i] = fg_place<BL, BN>(wv + 4u * i, lane, cols, ldb, bkq);
    }
    /* load i of the next stage of A (of B) */
    auto left = [&](uint32_t j) { return p.K - (j >= nst1 ? j - nst1 : j) * 64u; };
    auto load_a = [&](uint32_t i) {
        const uint32_t lf = left(ja);
        fg_dma16(pa, fg_span<AL>(lf, lda), AL == 0 ? fg_cut(ao[i], lf, akq) : ao[i], fg_lds + sa + (wv + 4u * i) * 1024u);
    };
    /* FP8 rows of K % 16 == 8 codes end in half a piece: the last stage's is read 8
     * bytes early, and its codes move down when they are read from LDS */
    const bool half = FP8 && (p.K & 8u);
    auto half_loads = [&]() {
        if (half && jb + 1u == nst1) {
            pb -= 8;
#pragma unroll
            for (uint32_t i = 0; i < NBL; i++) bo[i] = fg_half(bo[i], left(jb), bkq);
        }
    };
    auto load_b = [&](uint32_t i) {
        const uint32_t lf = left(jb);
        fg_dma16(pb, fg_span<BL>(lf, ldb), BL == 0 ? fg_cut(bo[i], lf, bkq) : bo[i], bring + sb + (wv + 4u * i) * 1024u);
    };
    auto next_a = [&]() {
        ja++;
        pa += astep;
        if (MODE == GHIP_EP_STORE && ja == nst1 && all > nst1) pa = base_a(p.a2);
        sa = sa == L * AST ? 0u : sa + AST;
    };
    auto next_b = [&]() {
        jb++;
        pb += bstep;
        if (MODE == GHIP_EP_STORE && jb == nst1 && all > nst1) pb = base_b(p.b2);
        sb = sb == (L - 1u) * BST ? 0u : sb + BST;
        if constexpr (FP8) half_loads();
    };
    if constexpr (FP8) half_loads();                     /* one stage */

    /* operand reads: block blk of 16 rows, step s */
    uint32_t off0[2];
#pragma unroll
    for (uint32_t s = 0; s < 2; s++) off0[s] = fg_at0(n, 2u * g + s);
    auto frag = [&](auto layout_c, auto w_c, const uint8_t *st, uint32_t blk, int s) -> ghip_bf16x8 {
        constexpr uint32_t W = decltype(w_c)::value;
        if constexpr (decltype(layout_c)::value == 0) {
            return *(const ghip_bf16x8 *)(st + blk * 2048u + off0[s]);
        } else {
            const uint32_t k = 16u * g + 8u * (uint32_t)s + (n >> 2);
            const uint8_t *q = fg_at1<W>(st, k, blk) + (n & 3u) * 8u;
            /* k + 4 has the same swizzle */
            const fg_s16x4 lo = fg_read_tr((fg_lds_s16x4 *)q);
            const fg_s16x4 hi = fg_read_tr((fg_lds_s16x4 *)(q + 8u * W));
            return __builtin_bit_cast(ghip_bf16x8,
                                      __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };
    ghip_f32x4 acc[RB][CB];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (int c = 0; c < CB; c++) acc[r][c] = (ghip_f32x4){0.f, 0.f, 0.f, 0.f};
    ghip_bf16x8 xa[2][RB], wa[2][CB];
    ghip_u32x4 codes[FP8 ? CB : 1];
    auto read_a = [&](int set, int r, const uint8_t *st, int s) {
        xa[set][r] = frag(LA{}, WA{}, st, wr * RB + r, s);
    };
    auto read_b = [&](int set, int c, const uint8_t *st, int s) {
        if constexpr (FP8)
            codes[c] = *(const ghip_u32x4 *)(st + (wc * CB + c) * 1024u + fg_at_codes(n, g));
        else
            wa[set][c] = frag(LB{}, WB{}, st, wc * CB + c, s);
    };
    auto half_codes = [&]() {                            /* of the last stage */
        if (half && left(nst1 - 1u) - 16u * g == 8u) {
#pragma unroll
            for (int c = 0; c < CB; c++) codes[FP8 ? c : 0] = (ghip_u32x4){codes[FP8 ? c : 0][2], codes[FP8 ? c : 0][3], 0u, 0u};
        }
    };
    /* FP8: quarter q of column block c's operand of step s (4 codes) */
    float sc0 = 0.0f, sc1 = 0.0f;
    uint32_t srow0 = 0, srow1 = 0;
    if constexpr (FP8) {
        /* the wave's rows of a matrix lie in one block of 128 (tiles start at
         * multiples of their width, which divides it or is 256) */
        const uint32_t nkb = (p.K + 127u) >> 7, last = (p.N - 1u) >> 7;
        const uint32_t w0 = col0 + wc * (DUAL ? 8u * CB : 16u * CB);
        srow0 = srow1 = min(w0 >> 7, last) * nkb;
    }
    auto scales = [&](uint32_t j) {                      /* of stage j */
        sc0 = ghip_sload(p.s, srow0 + (j >> 1));
        if constexpr (DUAL) sc1 = ghip_sload(p.s2, srow1 + (j >> 1));
    };
    auto dequant = [&](int set, int c, int s, int h) {
        const float sc = DUAL && (c & 1) ? sc1 : sc0;
        const ghip_u32x2 d = ghip_deq4<W8 == 2>(codes[c][2 * s + h], sc);
        ghip_u32x4 v = __builtin_bit_cast(ghip_u32x4, wa[set][c]);
        v[2 * h] = d[0];
        v[2 * h + 1] = d[1];
        wa[set][c] = __builtin_bit_cast(ghip_bf16x8, v);
    };

    /* L stages in flight, then the first step's operands */
#pragma unroll
    for (uint32_t j = 0; j < (uint32_t)L; j++)
        if (j < nst) {
#pragma unroll
            for (uint32_t i = 0; i < NAL; i++) load_a(i);
            next_a();
#pragma unroll
            for (uint32_t i = 0; i < NBL; i++) load_b(i);
            next_b();
        }
    if constexpr (FP8) scales(0);
    ghip_wait_stages<LPS, L - 1>(nst - 1u);
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int c = 0; c < CB; c++) read_b(0, c, bring, 0);
#pragma unroll
    for (int r = 0; r < RB; r++) read_a(0, r, fg_lds, 0);
    if constexpr (FP8) {
        if (nst == 1u) half_codes();
#pragma unroll
        for (int c = 0; c < CB; c++)
#pragma unroll
            for (int h = 0; h < 2; h++) dequant(0, c, 0, h);
    }
    uint32_t ra = 0, rb = 0;                             /* slots of stage j */
    /* MAIN: stage j + L exists and is loaded during this one. Operands are read
     * one step ahead; the barrier sits between the steps, when the stage's last
     * operands are in registers, and frees its B slot (its A slot is written
     * again from the next stage's first step on). */
    auto stage = [&](uint32_t j, auto main_c) {
        constexpr bool MAIN = decltype(main_c)::value;
        const bool more = MAIN || j + 1u < nst;          /* else re-read this stage, unused */
        const uint32_t na = !more ? ra : ra == L * AST ? 0u : ra + AST;
        const uint32_t nb = !more ? rb : rb == (L - 1u) * BST ? 0u : rb + BST;
        fg_each<2>([&](auto step) {
            constexpr int S = decltype(step)::value;
            if constexpr (S == 1) {
                /* own loads of stage j + 1 done, own reads of stage j done;
                 * after the barrier that holds for every wave */
                if (MAIN) GHIP_VMCNT((L - 1) * NAL + (L - 2) * NBL);
                else ghip_wait_stages<LPS, L - 2>(more ? nst - 2u - j : 0u);
                __builtin_amdgcn_s_waitcnt(0xc07f);
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (FP8) scales(more ? j + 1u : j);
            }
            const uint8_t *as = fg_lds + (S == 0 ? ra : na), *bs = bring + (S == 0 ? rb : nb);
            /* between the MFMAs: the next step's reads (FP8: in the first half,
             * codes only in step 1, which serve both steps), its dequantization
             * (in step 1 in the second half), and the loads */
            constexpr int B0 = FP8 && S == 0 ? (int)CB : 0, NR = RB + (int)CB - B0;
            constexpr int RE = FP8 ? NM / 2 : NM, DF = S == 1 ? NM / 2 : 0, NQ = FP8 ? 2 * CB : 0;
            constexpr int NL = !MAIN ? 0 : S == 0 ? (int)NAL : (int)NBL;
            fg_each<NM>([&](auto slot) {
                constexpr int I = decltype(slot)::value, R = I / CB;
                constexpr int C = R & 1 ? CB - 1 - I % CB : I % CB;
                fg_mfma(acc[R][C], wa[S][C], xa[S][R]);
                constexpr int R0 = fg_spread(NR, I, 0, RE), R1 = fg_spread(NR, I + 1, 0, RE);
                constexpr int Q0 = fg_spread(NQ, I, DF, NM), Q1 = fg_spread(NQ, I + 1, DF, NM);
                constexpr int L0 = fg_spread(NL, I, 0, NM), L1 = fg_spread(NL, I + 1, 0, NM);
                fg_each<R1 - R0>([&](auto k) {
                    constexpr int O = R0 + decltype(k)::value + B0;
                    if constexpr (O < (int)CB) read_b(S ^ 1, O, bs, S ^ 1);
                    else read_a(S ^ 1, O - CB, as, S ^ 1);
                });
                if constexpr (FP8 && S == 1 && !MAIN && I == DF)
                    if (more && j + 2u == nst) half_codes();
                fg_each<Q1 - Q0>([&](auto k) {
                    constexpr int Q = Q0 + decltype(k)::value;
                    dequant(S ^ 1, Q >> 1, S ^ 1, Q & 1);
                });
                fg_each<L1 - L0>([&](auto k) {
                    constexpr uint32_t O = L0 + decltype(k)::value;
                    if constexpr (S == 0) load_a(O);
                    else load_b(O);
                });
                if constexpr (R1 > R0 || Q1 > Q0 || L1 > L0) __builtin_amdgcn_sched_barrier(0);
            });
            if constexpr (MAIN) {
                if constexpr (S == 0) next_a();
                else next_b();
            }
            __builtin_amdgcn_sched_barrier(0);
        });
        ra = na;
        rb = nb;
    };
    uint32_t j = 0;
    for (; j + L < nst; j++) stage(j, std::true_type{});
    for (; j < nst; j++) stage(j, std::false_type{});
    fg_settle(acc);

    /* register i of block (r, c): row 16 r + n, column 16 c + 4 g + i. G blocks of
     * 16 rows of f32 at a time, 16-byte piece q of a row at q XOR a function of
     * the row; then 8 columns of a row a lane, the same columns every time */
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    constexpr int G = RING / 4u >= 1024u * CB * RB ? RB : RING / 4u >= 512u * CB * RB ? RB / 2 : RB / 4;
    static_assert(RING / 4u >= 1024u * CB * G && RB % G == 0, "epilogue staging");
    constexpr uint32_t RBY = 64u * CB;                   /* bytes of a staged row */
    constexpr uint32_t LPR = DUAL ? CB : 2u * CB;        /* groups of 8 columns of a row */
    constexpr int IT = G * (int)LPR / 4, U = IT % 4 == 0 ? 4 : IT % 2 == 0 ? 2 : 1;
    uint8_t *sw = fg_lds + wv * (1024u * CB * G);
    auto spot = [&](uint32_t row, uint32_t q) {
        return row * RBY + 16u * (q ^ (CB >= 4 ? row & 15u : CB == 2 ? (row >> 1) & 7u : (row >> 2) & 3u));
    };
    const uint32_t pc = lane % LPR, c0 = (DUAL ? 8u : 16u) * CB * wc + 8u * pc, n0 = col0 + c0;
    const uint32_t m0 = row0 + 16u * wr * RB + lane / LPR;
    /* dual: block c of 16 output columns is staged as gate block 2c, up block 2c + 1 */
    const uint32_t q0 = DUAL ? 8u * (pc >> 1) + 2u * (pc & 1u) : 2u * pc;
    constexpr bool BIAS = MODE == GHIP_EP_LINEAR || MODE == GHIP_EP_DLINEAR;
    constexpr bool IN = BIAS || MODE == GHIP_EP_DGATED;
    uint16_t *out = second ? ep.out2 : ep.out;
    /* 8 values at any alignment: the device takes 16-byte accesses at 2 bytes. A
     * tile that holds a row's last piece where that is a part (!fast) goes by
     * elements there; columns behind it up to the next multiple of 8 get zeros
     * where they are the output's own */
    const bool live = c0 < cols, whole = n0 + 8u <= p.N;
    const bool fast = (p.N & 7u) == 0u || cols == OUTN;
    const uint32_t nc = live ? n0 : col0;                /* loads of dead lanes stay inside */
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
            for (uint32_t e = 0; e < 8; e++) {
                if (n0 + e < p.N) row[n0 + e] = (uint16_t)(d[e >> 1] >> (16u * (e & 1u)));
                else if (ep.pad) row[n0 + e] = 0;
            }
        }
    };
    float bias[8] = {};
    if constexpr (BIAS)
        if (ep.bias) {
            if (fast) load8(std::true_type{}, ep.bias, bias);
            else load8(std::false_type{}, ep.bias, bias);
        }
    ghip_with_act(MODE == GHIP_EP_STORE ? GHIP_ACT_NONE : ep.act, [&](auto act) {
        auto values = [&](uint32_t lr, const float (&in)[8], float (&o0)[8], float (&o1)[8]) {
            float s0[8], s1[8] = {};
            auto read8 = [&](uint32_t q, float (&v)[8]) {
#pragma unroll
                for (uint32_t d = 0; d < 2; d++) {
                    const ghip_f32x4 x = *(const ghip_f32x4 *)(sw + spot(lr, q + d));
#pragma unroll
                    for (int e = 0; e < 4; e++) v[4 * d + e] = x[e];
                }
            };
            read8(q0, s0);
            if constexpr (DUAL) read8(q0 + 4u, s1);
#pragma unroll
            for (int e = 0; e < 8; e++)
                ghip_ep_value<MODE, decltype(act)::value>(s0[e], s1[e], bias[e], in[e], ep.limit,
                                                          o0[e], o1[e]);
        };
#pragma unroll
        for (int rg = 0; rg < RB; rg += G) {
#pragma unroll
            for (int r = 0; r < G; r++)
#pragma unroll
                for (uint32_t c = 0; c < CB; c++)
                    *(ghip_f32x4 *)(sw + spot(16u * r + n, 4u * c + g)) = acc[rg + r][c];
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_wave_barrier();
            const uint32_t mg = m0 + 16u * rg;           /* this lane's first row */
            auto rows_out = [&](auto fast_c, auto u_c) {
                constexpr int UU = decltype(u_c)::value;
#pragma unroll 1
                for (int it = 0; it < IT; it += UU) {
                    float in[UU][8] = {};
                    if constexpr (IN)
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
                        float o0[8], o1[8];
                        values(lane / LPR + dr, in[u], o0, o1);
                        if (m < p.M && live) {
                            if (MODE == GHIP_EP_STORE && p.part) {
                                /* f32 partial sums, rows of whole pieces */
                                const size_t ld = (p.N + 7u) & ~7u;
                                float *q = p.part
                                           + (((second ? p.splits : 0u) + split) * (size_t)p.M + m) * ld + n0;
                                *(ghip_f32x4 *)q = (ghip_f32x4){o0[0], o0[1], o0[2], o0[3]};
                                *(ghip_f32x4 *)(q + 4) = (ghip_f32x4){o0[4], o0[5], o0[6], o0[7]};
                            } else {
                                store8(fast_c, out + (size_t)m * ep.ldout, o0);
                                if constexpr (MODE == GHIP_EP_DGATED)
                                    store8(fast_c, ep.out2 + (size_t)m * ep.ldout, o1);
                            }
                        }
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

template <int MODE, int W8, int AL, int BL, int WM, int RB, int CB, int L>
__global__ __launch_bounds__(256, 1) void k_ffn_gemm(GhipProd p, GhipEp ep, uint32_t mt,
                                                     uint32_t nt) {
    fg_product<MODE, W8, AL, BL, WM, RB, CB, L>(p, ep, mt, nt, blockIdx.x, gridDim.x);
}

#endif /* K_FFN_GEMM_H */
