/*
 * k_ffn_gemm.h — the tiled MFMA product of the dense feed-forward operators
 * (gfx950): out[m, n] = epilogue(sum_k A(m, k) B(n, k)); instantiated by
 * k_ffn_nt.hip (forward), k_ffn_nn.hip (dx) and k_ffn_tn.hip (dW).
 *
 * A workgroup of WM x WN waves owns 32 RB WM rows (of A) x 64 WN rows of B;
 * wave (wr, wc) computes 32 RB x 64 outputs with v_mfma_f32_32x32x16_bf16, B
 * as the A operand of the instruction, so a lane ends with four consecutive
 * columns of one output row. k is walked in stages of 64 through a ring of NS
 * stages in LDS.
 *
 * Operand layouts. 0: k is the fast index in memory (x, W in the forward). The
 * stage is [row][64 k], whole 128-byte lines, 16-byte piece p of row r at p ^
 * ((r >> 1) & 7); an operand of 8 k values is one ds_read_b128. 1: the row is
 * (W in dx, dz and x in dW). The stage is [64 k][rows], 32-byte slot s of k at
 * s ^ 2 (k & 3), and an operand is two ds_read_b64_tr_b16: each transposes 4 k
 * x 16 rows inside 16 lanes, so no transposed copy of a matrix is made. In
 * both, lane half h of MFMA step s takes k = 32 h + 8 s + [0, 8), so either
 * layout may meet the other. (Rows of 64 values: slot s at s ^ 2 ((k >> 1) & 1).)
 *
 * Loads go straight to LDS (buffer loads, 16 bytes a lane). Rows past the
 * matrix and k past its end are given an offset outside the buffer, which
 * loads zeros: no other row is read in their place and a ragged K needs no
 * separate kernel. FP8 weights go through registers instead: 16 codes a load,
 * dequantized bit-exactly while the products of the stage before run, and
 * written in the same layout.
 *
 * Dual modes (gate and up): the tile's B rows alternate in blocks of 32 between
 * the two matrices, so a wave holds g and u of the same 32 columns and the
 * product of the two needs no exchange.
 *
 * The epilogue passes the sums through a wave-private piece of the ring 32 rows
 * at a time, so that bias, residual and output are 16-byte accesses along a
 * row.
 */
#ifndef K_FFN_GEMM_H
#define K_FFN_GEMM_H

#include "ghip_epilogue.h"

typedef float fg_f32x16 __attribute__((ext_vector_type(16)));
typedef short fg_s16x4 __attribute__((ext_vector_type(4)));
typedef short fg_s16x8 __attribute__((ext_vector_type(8)));

#define FG_LDS_MAX (160u * 1024u)
#define FG_OOB 0xFFFFFFF0u                       /* past every buffer: loads zeros */
#define FG_SPAN 0x80000000u                      /* valid offsets are below */

__device__ __forceinline__ __amdgpu_buffer_rsrc_t fg_buf(const void *p) {
    return __builtin_amdgcn_make_buffer_rsrc((void *)p, 0, FG_SPAN, 0x20000);
}
__device__ __forceinline__ void fg_dma16(const void *base, uint32_t off, void *lds_wave) {
    __builtin_amdgcn_raw_ptr_buffer_load_lds(fg_buf(base), (ghip_lds_t *)lds_wave, 16, off, 0, 0, 0);
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

/* Layout 1: what the 32-byte slots of k's row of W values are XORed with, so that
 * the 4 k x 32 rows a half wave reads lie in distinct banks. */
template <uint32_t W>
__device__ __forceinline__ uint32_t fg_swizzle(uint32_t k) {
    static_assert(W == 64 || W == 128 || W == 256, "whole rounds of the banks");
    return W == 64 ? k & 2u : (k & 3u) << 1;
}

/* 8 outputs of row m from column n0 on: s0 (and s1) their sums. */
template <int MODE, int ACT>
__device__ __forceinline__ void fg_store8(const GhipEp &ep, uint16_t *out, uint32_t m, uint32_t n0,
                                          uint32_t N, const float (&s0)[8], const float (&s1)[8],
                                          bool vin, bool vout, bool vbias) {
    float b[8] = {}, in[8] = {}, o0[8], o1[8];
    const bool whole = n0 + 8u <= N;
    auto load = [&](const uint16_t *p, bool vec, float (&v)[8]) {
        if (whole && vec) {
            const ghip_u32x4 d = *(const ghip_u32x4 *)p;
#pragma unroll
            for (int e = 0; e < 8; e++)
                v[e] = ghip_bf16_f32(e & 1 ? d[e >> 1] >> 16 : d[e >> 1] & 0xffffu);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) v[e] = n0 + e < N ? ghip_bf16_f32(p[e]) : 0.0f;
        }
    };
    if constexpr (MODE == GHIP_EP_LINEAR || MODE == GHIP_EP_DLINEAR)
        if (ep.bias) load(ep.bias + n0, vbias, b);
    if constexpr (MODE != GHIP_EP_STORE && MODE != GHIP_EP_GATED)
        if (ep.in) load(ep.in + (size_t)m * ep.ldin + n0, vin, in);
#pragma unroll
    for (int e = 0; e < 8; e++)
        ghip_ep_value<MODE, ACT>(s0[e], s1[e], b[e], in[e], ep.limit, o0[e], o1[e]);
    auto store = [&](uint16_t *p, const float (&v)[8]) {
        typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
        ghip_u32x4 d;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const bool pad = n0 + 2u * e >= N, half = n0 + 2u * e + 1u >= N;
            bf2 t;
            t[0] = (__bf16)(!whole && pad ? 0.0f : v[2 * e]);
            t[1] = (__bf16)(!whole && half ? 0.0f : v[2 * e + 1]);
            d[e] = __builtin_bit_cast(uint32_t, t);
        }
        if (vout && (whole || ep.pad)) {
            *(ghip_u32x4 *)p = d;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++)
                if (n0 + e < N) p[e] = (uint16_t)(d[e >> 1] >> (16u * (e & 1u)));
        }
    };
    store(out + (size_t)m * ep.ldout + n0, o0);
    if constexpr (MODE == GHIP_EP_DGATED) store(ep.out2 + (size_t)m * ep.ldout + n0, o1);
}

template <int MODE, bool FP8, int AL, int BL, int WM, int WN, int RB, int NS>
__global__ __launch_bounds__(WM *WN * 64, 1) void k_ffn_gemm(GhipProd p, GhipEp ep, uint32_t mt,
                                                              uint32_t nt) {
    constexpr bool DUAL = ghip_ep_dual(MODE);
    constexpr uint32_t CB = 2, NW = WM * WN, BM = 32u * RB * WM, BN = 64u * WN;
    constexpr uint32_t OUTN = DUAL ? BN / 2 : BN;        /* output columns of a tile */
    constexpr uint32_t ASTG = BM * 128u, STG = (BM + BN) * 128u;
    constexpr uint32_t NAL = BM / 8u / NW, NBL = FP8 ? 0 : BN / 8u / NW, LPS = NAL + NBL;
    constexpr uint32_t NC = FP8 ? BN / 16u / NW : 1u;    /* code loads of a lane a stage */
    static_assert(NAL * NW * 8u == BM && BN / 8u % NW == 0 && BN / 16u % NW == 0, "loads");
    static_assert(NS * STG <= FG_LDS_MAX && NS >= 2 && LPS * (NS - 1) <= 63, "ring");
    static_assert(NS * STG / NW >= 8192u, "epilogue staging");
    static_assert(!FP8 || (NS == 2 && BL == 0), "codes are staged through two slots");
    extern __shared__ __attribute__((aligned(1024))) uint8_t fg_lds[];
    const uint32_t tid = threadIdx.x, lane = tid & 63u;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t wr = wv / WN, wc = wv % WN, n = lane & 31u, h = lane >> 5;

    /* tile t: the workgroups of one XCD (b % 8) take a run of consecutive
     * tiles, which go down 8 row tiles before the next column, so that an XCD's
     * L2 holds few rows of A and of B at a time. A batch of two: the second
     * half of the tiles is the second product. */
    uint32_t t;
    {
        const uint32_t T = gridDim.x, x = blockIdx.x & 7u, i = blockIdx.x >> 3;
        const uint32_t q = T >> 3, r = T & 7u;
        t = x * q + (x < r ? x : r) + i;
    }
    bool second = false;
    if constexpr (MODE == GHIP_EP_STORE) {
        second = p.batch && t >= mt * nt;
        if (second) t -= mt * nt;
    }
    const uint32_t strip = t / (8u * nt), in_strip = t - strip * (8u * nt);
    const uint32_t sr = min(8u, mt - strip * 8u);
    const uint32_t row0 = (strip * 8u + in_strip % sr) * BM, col0 = in_strip / sr * OUTN;
    const uint32_t rows = min(p.M - row0, BM), cols = min(p.N - col0, OUTN);
    const uint32_t nst1 = (p.K + 63u) >> 6;              /* stages of one product */
    const uint32_t nst = MODE == GHIP_EP_STORE && p.a2 && !p.batch ? 2u * nst1 : nst1;
    const size_t astep = AL == 0 ? 128u : (size_t)p.aks * 128u;
    const size_t bstep = BL == 0 ? (FP8 ? 64u : 128u) : (size_t)p.bks * 128u;
    auto base_a = [&](const uint16_t *a) {
        return (const uint8_t *)(a + (AL == 0 ? (size_t)row0 * p.ars : row0));
    };
    auto base_b = [&](const void *b) {
        return (const uint8_t *)b
               + (BL == 0 ? (size_t)col0 * p.brs : col0) * (FP8 ? (size_t)1 : (size_t)2);
    };
    const uint8_t *a0 = base_a(second ? p.a2 : p.a), *b0 = base_b(second ? p.b2 : p.b);
    const uint8_t *a1 = nst > nst1 ? base_a(p.a2) : a0;
    const uint8_t *b1 = DUAL || nst > nst1 ? base_b(p.b2) : b0;

    /* Byte offset of this lane's 16 bytes of 1 KB load c in a stage of W rows,
     * `live` of them inside the matrix; kq: the k (layout 0: of the piece) it
     * holds. The load's lane l goes to byte 16 l of the KB. */
    auto place = [&](auto layout_c, auto w_c, uint32_t c, uint32_t live, uint32_t ld,
                     uint32_t &kq) -> uint32_t {
        constexpr uint32_t W = decltype(w_c)::value;
        if constexpr (decltype(layout_c)::value == 0) {
            const uint32_t r = 8u * c + (lane >> 3), q = (lane & 7u) ^ ((r >> 1) & 7u);
            kq = 8u * q;
            return r < live ? r * ld * 2u + 16u * q : FG_OOB;
        } else {
            const uint32_t e = c * 64u + lane, k = e / (W / 8u);
            const uint32_t q = e % (W / 8u) ^ 2u * fg_swizzle<W>(k);
            kq = k;
            return 8u * q < live ? k * ld * 2u + 16u * q : FG_OOB;
        }
    };
    using LA = std::integral_constant<int, AL>;
    using LB = std::integral_constant<int, BL>;
    using WA = std::integral_constant<uint32_t, BM>;
    using WB = std::integral_constant<uint32_t, BN>;
    const uint32_t lda = (uint32_t)(AL == 0 ? p.ars : p.aks);
    const uint32_t ldb = (uint32_t)(BL == 0 ? p.brs : p.bks);
    /* B row r of the tile: in the dual modes row 32 (r / 64) + r % 32 of the
     * gate (even blocks of 32) or up matrix */
    uint32_t ao[NAL], ak[NAL], bo[NBL ? NBL : 1], bk[NBL ? NBL : 1];
#pragma unroll
    for (uint32_t i = 0; i < NAL; i++) ao[i] = place(LA{}, WA{}, wv + NW * i, rows, lda, ak[i]);
    if constexpr (!FP8) {
#pragma unroll
        for (uint32_t i = 0; i < NBL; i++) {
            const uint32_t c = wv + NW * i;
            bo[i] = place(LB{}, WB{}, c, DUAL ? BN : cols, ldb, bk[i]);
            if constexpr (DUAL) {
                const uint32_t r = 8u * c + (lane >> 3), mr = 32u * (r >> 6) + (r & 31u);
                bo[i] = mr < cols ? bo[i] - (r - mr) * ldb * 2u : FG_OOB;
            }
        }
    }
    /* FP8: load i of wave wv covers 16 rows (wv + NW i), 4 lanes a row */
    uint32_t co[NC], cw[NC][2], ck = 0;
    if constexpr (FP8) {
        ck = 16u * (lane & 3u);
#pragma unroll
        for (uint32_t i = 0; i < NC; i++) {
            const uint32_t r = 16u * (wv + NW * i) + (lane >> 2);
            const uint32_t mr = DUAL ? 32u * (r >> 6) + (r & 31u) : r;
            co[i] = mr < cols ? mr * ldb + ck : FG_OOB;
#pragma unroll
            for (uint32_t d = 0; d < 2; d++)
                cw[i][d] = ASTG + r * 128u + 16u * ((2u * (lane & 3u) + d) ^ ((r >> 1) & 7u));
        }
    }
    /* whether 1 KB load c (FP8: of 16 rows) is of the up matrix: wave-uniform */
    auto up = [&](uint32_t c) { return DUAL && (((FP8 ? 2u * c : c) >> 2) & 1u); };

    auto issue = [&](uint32_t j) {
        uint8_t *st = fg_lds + (j % NS) * STG;
        const bool nd = j >= nst1;
        const uint32_t jj = nd ? j - nst1 : j, k0 = jj * 64u, left = p.K - k0;
        const uint8_t *aj = (nd ? a1 : a0) + jj * astep;
        const uint8_t *bj = (nd && !DUAL ? b1 : b0) + jj * bstep, *uj = b1 + jj * bstep;
        if (left >= 64u) {
#pragma unroll
            for (uint32_t i = 0; i < NAL; i++) fg_dma16(aj, ao[i], st + (wv + NW * i) * 1024u);
#pragma unroll
            for (uint32_t i = 0; i < NBL; i++)
                fg_dma16(up(wv + NW * i) ? uj : bj, bo[i], st + ASTG + (wv + NW * i) * 1024u);
        } else {                                         /* the stage that ends at K */
#pragma unroll
            for (uint32_t i = 0; i < NAL; i++)
                fg_dma16(aj, ak[i] < left ? ao[i] : FG_OOB, st + (wv + NW * i) * 1024u);
#pragma unroll
            for (uint32_t i = 0; i < NBL; i++)
                fg_dma16(up(wv + NW * i) ? uj : bj, bk[i] < left ? bo[i] : FG_OOB,
                         st + ASTG + (wv + NW * i) * 1024u);
        }
    };
    /* FP8: stage j's codes into registers, and from there dequantized into its
     * slot. A load's rows share a scale (whole blocks of 128, or half of one) */
    ghip_u32x4 codes[NC];
    float sc[NC];
    auto fetch_codes = [&](uint32_t j) {
        const uint32_t left = p.K - j * 64u, nkb = (p.K + 127u) >> 7;
#pragma unroll
        for (uint32_t i = 0; i < NC; i++) {
            const uint32_t c = wv + NW * i, r = 16u * c, mr = DUAL ? 32u * (r >> 6) + (r & 31u) : r;
            const bool u = up(c);
            codes[i] = __builtin_bit_cast(
                ghip_u32x4, __builtin_amdgcn_raw_buffer_load_b128(
                                fg_buf((u ? b1 : b0) + j * bstep), ck < left ? co[i] : FG_OOB, 0, 0));
            const uint32_t last = (p.N - 1u) >> 7, sb = min((col0 + mr) >> 7, last);
            sc[i] = ghip_sload(u ? p.s2 : p.s, sb * nkb + (j >> 1));
        }
    };
    auto put_codes = [&](uint32_t j, uint32_t i) {
        uint8_t *st = fg_lds + (j % NS) * STG;
        ghip_u32x4 lo, hi;
        if (p.exact) ghip_deq16_u32<true>(codes[i], sc[i], lo, hi);
        else ghip_deq16_u32<false>(codes[i], sc[i], lo, hi);
        *(ghip_u32x4 *)(st + cw[i][0]) = lo;
        *(ghip_u32x4 *)(st + cw[i][1]) = hi;
    };

    uint32_t off0[4];                                    /* layout 0 operand reads */
#pragma unroll
    for (uint32_t s = 0; s < 4; s++) off0[s] = n * 128u + 16u * ((4u * h + s) ^ ((n >> 1) & 7u));
    const uint32_t i16 = lane & 15u, c16 = (lane >> 4) & 1u;
    auto frag = [&](auto layout_c, auto w_c, const uint8_t *st, uint32_t blk, int s) -> ghip_bf16x8 {
        constexpr uint32_t W = decltype(w_c)::value;
        if constexpr (decltype(layout_c)::value == 0) {
            return *(const ghip_bf16x8 *)(st + blk * 4096u + off0[s]);
        } else {
            const uint32_t k = 32u * h + 8u * (uint32_t)s + (i16 >> 2);
            const uint32_t slot = (2u * blk + c16) ^ fg_swizzle<W>(k);
            const uint8_t *q = st + k * (2u * W) + slot * 32u + (i16 & 3u) * 8u;
            const fg_s16x4 lo = fg_read_tr((fg_lds_s16x4 *)q);
            const fg_s16x4 hi = fg_read_tr((fg_lds_s16x4 *)(q + 8u * W));
            return __builtin_bit_cast(ghip_bf16x8,
                                      __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7));
        }
    };
    fg_f32x16 acc[RB][CB];
#pragma unroll
    for (int r = 0; r < RB; r++)
#pragma unroll
        for (uint32_t c = 0; c < CB; c++)
#pragma unroll
            for (int i = 0; i < 16; i++) acc[r][c][i] = 0.0f;
    ghip_bf16x8 xa[2][RB], wa[2][CB];
    auto fetch = [&](int set, uint32_t j, int s) {
        const uint8_t *st = fg_lds + (j % NS) * STG;
#pragma unroll
        for (uint32_t r = 0; r < RB; r++) xa[set][r] = frag(LA{}, WA{}, st, wr * RB + r, s);
#pragma unroll
        for (uint32_t c = 0; c < CB; c++) wa[set][c] = frag(LB{}, WB{}, st + ASTG, wc * CB + c, s);
    };
    /* all NS stages in flight, then the first step's operands */
    if constexpr (FP8) {
        issue(0);
        fetch_codes(0);
#pragma unroll
        for (uint32_t i = 0; i < NC; i++) put_codes(0, i);
        GHIP_VMCNT(0);
        __builtin_amdgcn_s_waitcnt(0xc07f);
        if (nst > 1u) {
            issue(1);
            fetch_codes(1);
        }
    } else {
#pragma unroll
        for (uint32_t i = 0; i < NS; i++)
            if (i < nst) issue(i);
        ghip_wait_stages<LPS, NS - 1>(nst - 1u);
    }
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    fetch(0, 0u, 0);
    constexpr int READS = (AL ? 2 : 1) * RB + (BL ? 2 : 1) * (int)CB;
    constexpr int PER = (READS + RB * (int)CB - 1) / (RB * (int)CB);

    /* MAIN: stage j + NS exists and is loaded during this one. Operands are
     * read one MFMA step ahead; the stage's one barrier sits before its last
     * step, when its last operands are in registers, and frees its slot. FP8:
     * the codes of stage j + 1 are written during the first two steps (its slot
     * is free since the barrier of stage j - 1), those of stage j + 2 loaded in
     * the third. */
    auto stage = [&](uint32_t j, auto main_c) {
        constexpr bool MAIN = decltype(main_c)::value;
        const uint32_t jn = MAIN ? j + 1u : min(j + 1u, nst - 1u);
#pragma unroll
        for (int s = 0; s < 4; s++) {
            if (s == 3) {
                /* own loads of stage j + 1 done, own reads of stage j done;
                 * after the barrier that holds for every wave */
                if constexpr (FP8) {
                    /* the x loads of stage j + 1 are older than the codes of
                     * stage j + 2 */
                    if (MAIN) GHIP_VMCNT(NC);
                    else GHIP_VMCNT(0);
                } else if (MAIN) {
                    GHIP_VMCNT(LPS * (NS - 2));
                } else {
                    ghip_wait_stages<LPS, NS - 2>(nst - 1u - jn);
                }
                __builtin_amdgcn_s_waitcnt(0xc07f);
                __builtin_amdgcn_s_barrier();
                __builtin_amdgcn_sched_barrier(0);
                if (MAIN) issue(j + NS);
            }
            const int cur = s & 1, nxt = cur ^ 1;
            if constexpr (FP8) {
                if (s < 2 && (MAIN || j + 1u < nst)) {
#pragma unroll
                    for (uint32_t i = (uint32_t)s; i < NC; i += 2) put_codes(j + 1u, i);
                }
                if (s == 2 && MAIN) {
                    fetch_codes(j + 2u);
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
            if (s < 3) fetch(nxt, j, s + 1);
            else fetch(nxt, jn, 0);
#pragma unroll
            for (int r = 0; r < RB; r++)
#pragma unroll
                for (uint32_t c = 0; c < CB; c++)
                    acc[r][c] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(wa[cur][c], xa[cur][r],
                                                                       acc[r][c], 0, 0, 0);
            if constexpr (!FP8) {
#pragma unroll
                for (int i = 0; i < RB * (int)CB; i++) {
                    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                    if (i * PER < READS) __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    uint32_t j = 0;
    for (; j + NS < nst; j++) stage(j, std::true_type{});
    for (; j < nst; j++) stage(j, std::false_type{});

    /* register 4q + i of block (r, c) is row 32 r + n, column 32 c + 8 q + 4 h +
     * i: 32 rows x 64 columns of f32 at a time, 16-byte piece p of row n at p ^
     * (n & 15) */
    __builtin_amdgcn_s_waitcnt(0xc07f);
    __builtin_amdgcn_s_barrier();
    uint8_t *sw = fg_lds + wv * 8192u;
    uint16_t *out = second ? ep.out2 : ep.out;
    const bool vin = ((uintptr_t)ep.in & 15u) == 0u && (ep.ldin & 7u) == 0u;
    const bool vout = (((uintptr_t)out | (uintptr_t)ep.out2) & 15u) == 0u && (ep.ldout & 7u) == 0u;
    const bool vbias = ((uintptr_t)ep.bias & 15u) == 0u;
    constexpr uint32_t LPR = DUAL ? 4u : 8u;             /* lanes of a row */
    ghip_with_act(MODE == GHIP_EP_STORE ? GHIP_ACT_NONE : ep.act, [&](auto act) {
#pragma unroll
        for (int r = 0; r < RB; r++) {
#pragma unroll
            for (uint32_t c = 0; c < CB; c++)
#pragma unroll
                for (uint32_t q = 0; q < 4; q++) {
                    ghip_f32x4 v;
#pragma unroll
                    for (int i = 0; i < 4; i++) v[i] = acc[r][c][4 * q + i];
                    *(ghip_f32x4 *)(sw + n * 256u + 16u * ((8u * c + 2u * q + h) ^ (n & 15u))) = v;
                }
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_wave_barrier();
#pragma unroll 1
            for (uint32_t i = 0; i < LPR / 2u; i++) {
                const uint32_t lr = lane / LPR + 64u / LPR * i, pc = lane % LPR;
                auto read8 = [&](uint32_t first, float (&s)[8]) {
#pragma unroll
                    for (uint32_t d = 0; d < 2; d++) {
                        const ghip_f32x4 v =
                            *(const ghip_f32x4 *)(sw + lr * 256u + 16u * ((first + d) ^ (lr & 15u)));
#pragma unroll
                        for (int e = 0; e < 4; e++) s[4 * d + e] = v[e];
                    }
                };
                float s0[8], s1[8] = {};
                read8(2u * pc, s0);
                if constexpr (DUAL) read8(8u + 2u * pc, s1);
                const uint32_t m = row0 + 32u * (wr * RB + r) + lr;
                const uint32_t c0 = (DUAL ? 32u : 64u) * wc + 8u * pc;
                if (m < p.M && c0 < cols)
                    fg_store8<MODE, decltype(act)::value>(ep, out, m, col0 + c0, p.N, s0, s1, vin,
                                                          vout, vbias);
            }
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_wave_barrier();
        }
    });
}

#endif /* K_FFN_GEMM_H */
