/*
 * k_mx_rows.hip — gated products of a few rows of x with MXFP4 weights (gfx950).
 *
 * Bound by HBM: the weights are read once, 17/32 bytes a value, in whole lines of 128
 * bytes (256 k of a row). A wave copies its share of x's rows to LDS once and streams
 * blocks of weight rows past them, four steps of 128 k in registers ahead of the four in
 * use; a grid as large as the chip, or a whole fraction of the blocks, so that x is
 * copied few times and the stream does not end with a block. The codes cross LDS on
 * their way, as a line's 16 bytes are loaded by lanes beside each other and used by
 * lanes a row apart; each line is asked for once, because a second load from a line that
 * is in flight waits for it and then makes a trip of its own (operands loaded straight
 * into their registers, 64 bytes of a line at a time: gated 5 x 12288 x 4096 27.1 us, 11.8
 * so).
 * k is split over 8 or 4 waves, whose sums meet in LDS in a fixed order.
 *
 * Measured: gated BF16 5 x 12288 x 4096 11.8 us (53.5 MB, 4.5 TB/s), from launch to end: an
 * empty launch takes 2.5 to 3.
 */
#include <type_traits>
#include <utility>

#include "ghip_epilogue.h"
#include "ghip_mx.h"
#include "k_mx_rows_addr.h"

typedef int mx_i32x8 __attribute__((ext_vector_type(8)));

/* acc += W (MXFP4, 16 rows) . x^T (16 rows) over 128 k. Lane (n, g): W's row n, block
 * g; x's row n, bytes as its type has them (MXFP8: k 16 g + [0, 16) and 64 + 16 g +
 * [0, 16), as the instruction takes 8-bit operands; MXFP4 block g). */
template <int XT>
__device__ __forceinline__ void mx_mfma(ghip_f32x4 &acc, const ghip_u32x4 &w, uint32_t sw,
                                        const ghip_u32x4 (&x)[XT == GHIP_MXFP8 ? 2 : 1], uint32_t sx) {
    const mx_i32x8 a = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
    mx_i32x8 b;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        b[e] = (int)x[0][e];
        b[e + 4] = XT == GHIP_MXFP8 ? (int)x[XT == GHIP_MXFP8 ? 1 : 0][e] : 0;
    }
    acc = __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(a, b, acc, 4, XT == GHIP_MXFP8 ? 0 : 4, 0, sw, 0, sx);
}

/* f(0), f(1), ... f(N - 1), the argument a constant */
template <typename F, int... I>
__device__ __forceinline__ void mr_each_of(F f, std::integer_sequence<int, I...>) {
    (f(std::integral_constant<int, I>{}), ...);
}
template <int N, typename F>
__device__ __forceinline__ void mr_each(F f) {
    mr_each_of(f, std::make_integer_sequence<int, N>{});
}

/* Words of four steps, lane group g's that of step g, as bytes: byte s of lane group
 * g's result is block g of step s. Two exchanges between lane groups, a byte
 * permutation behind each. */
struct MrBytes {
    uint32_t s16, s32;                                   /* this lane's selectors */
};
__device__ __forceinline__ MrBytes mr_bytes(uint32_t g) {
    return {g & 1u ? 0x07030501u : 0x06020400u, g & 2u ? 0x07060302u : 0x05040100u};
}
__device__ __forceinline__ uint32_t mr_transpose(uint32_t v, const MrBytes &b) {
    /* even and odd lane groups' words, then the lower and upper pair's */
    const auto e = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    const uint32_t u = __builtin_amdgcn_perm(e[1], e[0], b.s16);
    const auto h = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    return __builtin_amdgcn_perm(h[1], h[0], b.s32);
}

/* Bytes of x's row in a step. */
constexpr uint32_t mr_xrow(int xt) { return xt == GHIP_BF16 ? 256u : xt == GHIP_MXFP8 ? 128u : 64u; }

/* A workgroup's 8 waves: 8 / KS slots of 16 rows of both matrices, k over KS waves; mr (up
 * to 16) rows of x. It takes every gridDim.x-th block of weight rows: a wave copies its share
 * of x to LDS once, and its stream of weights, four steps of 128 k ahead with one load
 * of scales for four, runs on from one block into the next. */
template <int XT, int KS>
__global__ __launch_bounds__(MR_WAVES * 64, 1) void k_mx_rows(GhipMxProd p, GhipEp ep, uint32_t blocks,
                                                              uint32_t row0, uint32_t mr) {
    constexpr bool BF = XT == GHIP_BF16;
    constexpr uint32_t GPP = MR_WAVES / KS, XR = mr_xrow(XT);
    constexpr int XI = BF ? 4 : XT == GHIP_MXFP8 ? 2 : 1;          /* 16-byte pieces of x a step */
    extern __shared__ __attribute__((aligned(16))) float red[];    /* the sums, W's way to its operands, x */
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, g = lane >> 4;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t part = wv % KS, slot = wv / KS;
    const uint32_t nst = mr_steps(p.K), nb = p.K >> 5, lds = 4u * nst;
    const MrShare share = mr_share<KS>(part, nst);
    const uint32_t c0 = share.from, c1 = share.to, nc = c1 - c0, nq = (nc + 3u) >> 2;
    const uint32_t m0 = row0 + blockIdx.y * mr, mrows = min(p.M - m0, mr);

    /* x's rows over the wave's share: [step][row][XR], zeros past K. The first loads go
     * ahead of the weights', the rest behind them */
    uint8_t *const wl = (uint8_t *)red + mr_lds_codes(wv);
    uint8_t *const xl = (uint8_t *)red + mr_lds_x(wv, mrows, XR, mr_share_most(nst, KS));
    const uint32_t all = mrows * nc * (XR / 16u), xbytes = p.K * (BF ? 4u : XT == GHIP_MXFP8 ? 2u : 1u) / 2u;
    ghip_u32x4 xd[8];
    uint32_t xat[8];
    auto x_load = [&](uint32_t v0) {
#pragma unroll
        for (int i = 0; i < 8; i++) {
            const uint32_t v = v0 + 64u * i + lane;
            const MrPiece at = mr_piece<XR>(v, nc);
            const uint32_t byte = (c0 + at.t) * XR + 16u * at.q;
            xd[i] = (ghip_u32x4){0u, 0u, 0u, 0u};
            xat[i] = v < all ? at.t * (mrows * XR) + mr_spot<XR>(at.r, at.q) : ~0u;
            if (v < all && byte < xbytes) xd[i] = *(const ghip_u32x4 *)(p.x + (size_t)(m0 + at.r) * p.xld + byte);
        }
        __builtin_amdgcn_sched_barrier(0);
    };
    auto x_store = [&]() {
#pragma unroll
        for (int i = 0; i < 8; i++)
            if (xat[i] != ~0u) *(ghip_u32x4 *)(xl + xat[i]) = xd[i];
    };
    if (nc) x_load(0);

    /* the weights' stream: block lblk, quad lq of the wave's share */
    const uint32_t wb = p.K >> 1, wend = min(64u * c1, wb);
    uint32_t lblk = blockIdx.x, lq = 0;
    const uint32_t mine = min(n, mrows - 1u);
    const uint8_t *const xs = BF ? nullptr : p.xs + (size_t)(m0 + mine) * lds;
    ghip_u32x4 wr[4][2];
    uint32_t sw[2], sx = 0u, bw[2], bx = 0u;
    /* The stream's next four steps: their scales, and half h of their codes (two steps).
     * What lies past the wave's share, a row's end, the matrix or the stream is past the
     * buffer: zeros, and no access (a second load from a line on its way costs a trip of
     * its own) */
    auto stream = [&](const uint8_t *m, uint32_t ld) {
        const uint32_t first = mr_first<KS>(lblk, slot);
        /* a vector instruction counts: back to a scalar, or the load goes lane by lane */
        const uint32_t live = __builtin_amdgcn_readfirstlane(mr_live(first, p.N));
        return __builtin_amdgcn_make_buffer_rsrc((void *)(m + (size_t)mr_base(first, p.N) * ld), 0, live * ld, 0x20000);
    };
    auto load_scales = [&]() {
        const uint32_t t = c0 + 4u * lq + g;
#pragma unroll
        for (int b = 0; b < 2; b++)
            sw[b] = __builtin_amdgcn_raw_buffer_load_b32(stream(b ? p.ws2 : p.ws, lds), mr_scale(n, t, nst), 0, 0);
        if constexpr (!BF) sx = *(const uint32_t *)(xs + 4u * min(t, nst - 1u));
    };
    auto load_codes = [&](auto h_c) {
        constexpr int h = decltype(h_c)::value;
#pragma unroll
        for (int b = 0; b < 2; b++) {
            const __amdgpu_buffer_rsrc_t m = stream(b ? p.w2 : p.w, wb);
#pragma unroll
            for (int i = 0; i < 2; i++)
                wr[2 * h + i][b] = __builtin_amdgcn_raw_buffer_load_b128(m, mr_code(i, lane, c0 + 4u * lq + 2u * h, wend, wb), 0, 0);
        }
    };
    auto advance = [&]() {
        if (++lq == nq) {
            lq = 0;
            lblk += gridDim.x;
        }
    };
    if (nc) {
        load_scales();
        mr_each<2>(load_codes);
        advance();
        __builtin_amdgcn_sched_barrier(0);
        x_store();
        for (uint32_t v0 = 512u; v0 < all; v0 += 512u) {
            x_load(v0);
            x_store();
        }
    }

    uint32_t blk = blockIdx.x, j = 0;
    ghip_f32x4 acc[2];
#pragma unroll
    for (int b = 0; b < 2; b++) acc[b] = (ghip_f32x4){0.f, 0.f, 0.f, 0.f};
    /* a block's end: the KS partial sums of each slot, added in order (register i: weight
     * row 4 g + i, x's row n); its outputs, one a thread */
    auto finish = [&]() {
        if (blk != blockIdx.x) {                         /* the block before has been read */
            __builtin_amdgcn_s_waitcnt(0xc07f);
            __builtin_amdgcn_s_barrier();
        }
#pragma unroll
        for (int b = 0; b < 2; b++) {
            *(ghip_f32x4 *)(red + mr_sum_put(wv, n, b, g)) = acc[b];
            acc[b] = (ghip_f32x4){0.f, 0.f, 0.f, 0.f};
        }
        __builtin_amdgcn_s_waitcnt(0xc07f);
        __builtin_amdgcn_s_barrier();
        const MrOut at = mr_out(tid);
        const uint32_t o = mr_first<KS>(blk, at.slot) + at.c;
        if (at.slot < GPP && at.m < mrows && o < p.N) {
            const float *q = red + mr_sum_get<KS>(at.slot, at.m, at.c);
            float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                s0 += q[k * 512u];
                s1 += q[k * 512u + 16u];
            }
            ghip_with_act(ep.act, [&](auto act) {
                ghip_ep_put<GHIP_EP_GATED, decltype(act)::value>(ep, ep.out, m0 + at.m, o, s0, s1, 0.0f, 0.0f);
            });
        }
        blk += gridDim.x;
    };
    if (nc == 0u) {                                      /* fewer steps than waves */
        while (blk < blocks) finish();
        return;
    }
    const MrBytes bytes = mr_bytes(g);
    uint32_t xo[XI];
#pragma unroll
    for (int i = 0; i < XI; i++) xo[i] = mr_spot<XR>(mine, mr_operand<XR>(g, i));
    const uint32_t w0 = mr_code_get(n, g, 0), w1 = mr_code_get(n, g, 1);
    for (;;) {
        const uint32_t t = c0 + 4u * j;
#pragma unroll
        for (int b = 0; b < 2; b++) bw[b] = mr_transpose(sw[b], bytes);
        if constexpr (!BF) bx = mr_transpose(sx, bytes);
        load_scales();
        mr_each<2>([&](auto h_c) {
            constexpr int h = decltype(h_c)::value;
            /* two steps of W to LDS as they were loaded, the registers' next load, and back
             * as operands; a wave's LDS accesses are in order */
#pragma unroll
            for (int b = 0; b < 2; b++)
#pragma unroll
                for (int i = 0; i < 2; i++) *(ghip_u32x4 *)(wl + 2048 * b + mr_code_put(i, lane)) = wr[2 * h + i][b];
            __builtin_amdgcn_sched_barrier(0);
            load_codes(h_c);
            __builtin_amdgcn_sched_barrier(0);
            if (t + 2u * h >= c1) return;
            ghip_u32x4 wo[2][2];
#pragma unroll
            for (int i = 0; i < 2; i++)
#pragma unroll
                for (int b = 0; b < 2; b++) wo[i][b] = *(const ghip_u32x4 *)(wl + 2048 * b + (i ? w1 : w0));
            mr_each<2>([&](auto i_c) {
                constexpr int i = decltype(i_c)::value, s = 2 * h + i;
                if (i && t + s >= c1) return;
                const bool past = 4u * (t + s) + g >= nb;    /* codes and x are zeros there */
                const uint8_t *const xt = xl + (t + s - c0) * (mrows * XR);
                ghip_u32x4 xr[XI];
#pragma unroll
                for (int k = 0; k < XI; k++) xr[k] = *(const ghip_u32x4 *)(xt + xo[k]);
#pragma unroll
                for (int b = 0; b < 2; b++) {
                    const uint32_t sb = past ? 127u : bw[b] >> (8 * s) & 255u;
                    if constexpr (BF) {
                        const float f = __uint_as_float(sb << 23);
#pragma unroll
                        for (int k = 0; k < 4; k++)
                            acc[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                __builtin_bit_cast(ghip_bf16x8, mx_fp4_bf16(wo[i][b][k], f)),
                                __builtin_bit_cast(ghip_bf16x8, xr[k]), acc[b], 0, 0, 0);
                    } else {
                        mx_mfma<XT>(acc[b], wo[i][b], sb, xr, past ? 127u : bx >> (8 * s) & 255u);
                    }
                }
            });
            __builtin_amdgcn_sched_barrier(0);
        });
        advance();
        if (++j == nq) {
            j = 0;
            finish();
            if (blk >= blocks) break;
        }
    }
}

/* One launchable form: k's waves, and microseconds of the launch, of four steps of
 * a wave, of a block besides, and of a KB of a wave's share of x; two: how much longer
 * these are where CUs hold two workgroups. The times are least-squares fits to sweeps of
 * 1 to 192 rows over N x K of 256 x 1024 to 12288 x 4096, 4096 x 12288, 8192 x 512 and 512 x
 * 8192, every form timed (0.05 to 0.1 rms of the logarithm). 8 waves along k shorten a
 * wave's chain and 4 halve the joins; BF16, us:
 *                         8 waves   4
 *   4 x 12288 x 4096         15.6   13.6
 *   1 x 256 x 1024            4.2    4.8 */
struct MrForm {
    uint32_t ks;
    float base, quad, over, copy, two;
    const void *kern;
    void (*launch)(dim3, uint32_t, hipStream_t, const GhipMxProd &, const GhipEp &, uint32_t, uint32_t,
                   uint32_t);
};
template <int XT, int KS>
static void mr_run(dim3 grid, uint32_t lds, hipStream_t st, const GhipMxProd &p, const GhipEp &ep,
                   uint32_t blocks, uint32_t row0, uint32_t mr) {
    hipLaunchKernelGGL((k_mx_rows<XT, KS>), grid, dim3(MR_WAVES * 64), lds, st, p, ep, blocks, row0, mr);
}
template <int XT, int KS>
static constexpr MrForm mr_form(float base, float quad, float over, float copy, float two) {
    return {KS, base, quad, over, copy, two, (const void *)k_mx_rows<XT, KS>, mr_run<XT, KS>};
}

static const MrForm mr_bf16[] = {
    mr_form<GHIP_BF16, 8>(1.6f, 1.70f, 0.47f, 0.19f, 0.95f),
    mr_form<GHIP_BF16, 4>(1.9f, 1.86f, 0.20f, 0.16f, 0.87f),
};
static const MrForm mr_mxfp8[] = {
    mr_form<GHIP_MXFP8, 8>(1.8f, 1.49f, 0.57f, 0.17f, 0.90f),
    mr_form<GHIP_MXFP8, 4>(1.7f, 1.39f, 0.94f, 0.17f, 0.87f),
};
static const MrForm mr_mxfp4[] = {
    mr_form<GHIP_MXFP4, 8>(1.6f, 0.84f, 1.28f, 0.32f, 1.34f),
    mr_form<GHIP_MXFP4, 4>(2.1f, 1.56f, 0.48f, 0.10f, 0.95f),
};
/* The gated mode's only. */
static const MrForm *mr_forms(int mode, int xt, int *n) {
    *n = mode == GHIP_EP_GATED ? 2 : 0;
    if (mode != GHIP_EP_GATED) return nullptr;
    return xt == GHIP_MXFP8 ? mr_mxfp8 : xt == GHIP_MXFP4 ? mr_mxfp4 : mr_bf16;
}

#define MR_MAX_TILES 65535u

static uint32_t g_mr_ncu = 256;

static MrCut cut(const MrForm *c, const GhipMxProd *p) {
    return mr_cut(p->M, p->N, p->K, mr_xrow(p->xt), c->ks, g_mr_ncu);
}

/* Estimated microseconds: the rounds of the chip, or the weights at 6.5 TB/s, and a
 * tenth of the other. */
static float form_us(const MrForm *c, const GhipMxProd *p, const MrCut &r) {
    const uint32_t most = mr_share_most(mr_steps(p->K), c->ks);
    const double quads = (double)((most / 2 + 1) / 2), chip = (double)g_mr_ncu * r.occ;
    const double rounds = (double)(size_t)(((double)r.grid * r.tiles + chip - 1.0) / chip);
    const double two = (size_t)r.grid * r.tiles > g_mr_ncu ? c->two : 1.0;
    const double copy = (double)r.mr * mr_xrow(p->xt) * most / 1024.0;
    const double chain = c->base + two * rounds * (r.turns * (quads * c->quad + c->over) + copy * c->copy);
    const double hbm = 2.6 + 2.0 * p->N * p->K * 17.0 / 32.0 / 6.5e6;
    return (float)(chain > hbm ? chain + 0.1 * hbm : hbm + 0.1 * chain);
}

extern "C" int ghip_mx_rows_forms(int mode, int xt) {
    int n;
    mr_forms(mode, xt, &n);
    return n;
}

extern "C" int ghip_mx_rows_fits(int mode, int form, const GhipMxProd *p) {
    int n;
    const MrForm *c = mr_forms(mode, p->xt, &n);
    return form >= 0 && form < n && cut(c + form, p).mr != 0u;
}

extern "C" int ghip_mx_rows_pick(int mode, const GhipMxProd *p, float *us) {
    int n, best = -1;
    const MrForm *c = mr_forms(mode, p->xt, &n);
    for (int i = 0; i < n; i++) {
        const MrCut r = cut(c + i, p);
        if (r.mr == 0u) continue;
        const float t = form_us(c + i, p, r);
        if (best < 0 || t < *us) {
            best = i;
            *us = t;
        }
    }
    return best;
}

extern "C" hipError_t ghip_launch_mx_rows(int mode, int form, const GhipMxProd *p, const GhipEp *ep, hipStream_t st) {
    int n;
    const MrForm *c = mr_forms(mode, p->xt, &n);
    if (p->M == 0 || p->N == 0 || p->K == 0 || p->K % 32 || !ghip_mx_rows_fits(mode, form, p))
        return hipErrorInvalidValue;
    c += form;
    const MrCut r = cut(c, p);
    for (uint32_t t = 0; t < r.tiles; t += MR_MAX_TILES) {
        const uint32_t nt = r.tiles - t < MR_MAX_TILES ? r.tiles - t : MR_MAX_TILES;
        c->launch(dim3(r.grid, nt), r.lds, st, *p, *ep, r.blocks, t * r.mr, r.mr);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

extern "C" hipError_t ghip_mx_rows_init(uint32_t n_cu) {
    for (int xt = GHIP_BF16; xt <= GHIP_MXFP4; xt++) {
        int n;
        const MrForm *c = mr_forms(GHIP_EP_GATED, xt, &n);
        for (int k = 0; k < n; k++) {
            const hipError_t e = hipFuncSetAttribute(c[k].kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)MR_LDS_MAX);
            if (e != hipSuccess) return e;
        }
    }
    g_mr_ncu = n_cu;
    return hipSuccess;
}
