/*
 * k_mx_rows.hip — products of a few rows with MXFP4 weights (gfx950): every wave
 * loads its weights' codes straight into the operand registers of the matrix
 * instruction.
 */
#include <type_traits>

#include "ghip_epilogue.h"
#include "ghip_mx.h"

typedef int mx_i32x8 __attribute__((ext_vector_type(8)));

#define MR_WAVES 8

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

/* A workgroup's 8 waves: 8 / KS groups of 16 NT weight rows, k over KS waves; 16 MT
 * rows of x. */
template <int XT, int MT, int NT, int KS, int MODE>
__global__ __launch_bounds__(MR_WAVES * 64, 1) void k_mx_rows(GhipMxProd p, GhipEp ep, uint32_t blk0,
                                                              uint32_t tile0) {
    constexpr bool DUAL = ghip_ep_dual(MODE), BF = XT == GHIP_BF16;
    constexpr uint32_t GPP = MR_WAVES / KS, OG = DUAL ? NT / 2 : NT, MR = 16 * MT;
    constexpr int XI = BF ? 4 : XT == GHIP_MXFP8 ? 2 : 1;          /* 16-byte pieces of x a step */
    static_assert(!DUAL || NT % 2 == 0, "gate and up groups alternate");
    extern __shared__ __attribute__((aligned(16))) float red[];    /* [8 waves][MR][16 NT] */
    const uint32_t tid = threadIdx.x, lane = tid & 63u, n = lane & 15u, g = lane >> 4;
    const uint32_t wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t part = wv % KS, slot = wv / KS;
    const uint32_t nst = (p.K + 127u) >> 7, nb = p.K >> 5, lds = 4u * nst;
    const uint32_t c0 = part * nst / KS, c1 = (part + 1u) * nst / KS;
    const uint32_t blk = blk0 + blockIdx.x, row0 = (blk * GPP + slot) * (16u * OG);
    const uint32_t m0 = (tile0 + blockIdx.y) * MR, mrows = min(p.M - m0, MR);
    ghip_f32x4 acc[MT][NT];
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
        for (int b = 0; b < NT; b++) acc[a][b] = (ghip_f32x4){0.f, 0.f, 0.f, 0.f};
    if (row0 < p.N) {
        const uint8_t *w[NT], *ws[NT], *x[MT], *xs[MT];
#pragma unroll
        for (int b = 0; b < NT; b++) {
            const size_t r = min(row0 + 16u * (DUAL ? b >> 1 : b) + n, p.N - 1u);
            w[b] = (DUAL && (b & 1) ? p.w2 : p.w) + r * (p.K / 2u);
            ws[b] = (DUAL && (b & 1) ? p.ws2 : p.ws) + r * lds;
        }
#pragma unroll
        for (int a = 0; a < MT; a++) {
            const size_t r = m0 + min(16u * a + n, mrows - 1u);
            x[a] = p.x + r * p.xld;
            if (!BF) xs[a] = p.xs + r * lds;
        }
        for (uint32_t t = c0; t < c1; t++) {
            const bool past = 4u * t + g >= nb;          /* the step that K cuts */
            const uint32_t blkg = past ? 4u * t : 4u * t + g;
            ghip_u32x4 wr[NT], xr[MT][XI];
            uint32_t sw[NT], sx[MT];
#pragma unroll
            for (int b = 0; b < NT; b++) {
                wr[b] = *(const ghip_u32x4 *)(w[b] + 16u * blkg);
                sw[b] = past ? 127u : *(const uint32_t *)(ws[b] + 4u * t) >> (8u * g) & 255u;
            }
#pragma unroll
            for (int a = 0; a < MT; a++) {
                if constexpr (!BF) sx[a] = past ? 127u : *(const uint32_t *)(xs[a] + 4u * t) >> (8u * g) & 255u;
#pragma unroll
                for (int i = 0; i < XI; i++) {
                    /* byte offset of the piece, and the block it lies in */
                    const uint32_t q = BF ? 256u * t + 64u * g + 16u * i
                                     : XT == GHIP_MXFP8 ? 128u * t + 64u * i + 16u * g : 64u * t + 16u * g;
                    const uint32_t at = XT == GHIP_MXFP8 ? 4u * t + 2u * i + (g >> 1) : 4u * t + g;
                    xr[a][i] = *(const ghip_u32x4 *)(x[a] + (at < nb ? q : 0u));
                    if (at >= nb) xr[a][i] = (ghip_u32x4){0u, 0u, 0u, 0u};
                }
            }
#pragma unroll
            for (int b = 0; b < NT; b++) {
                if constexpr (BF) {
                    const float s = __uint_as_float(sw[b] << 23);
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const ghip_bf16x8 wb = __builtin_bit_cast(ghip_bf16x8, mx_fp4_bf16(wr[b][i], s));
#pragma unroll
                        for (int a = 0; a < MT; a++)
                            acc[a][b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                                wb, __builtin_bit_cast(ghip_bf16x8, xr[a][i]), acc[a][b], 0, 0, 0);
                    }
                } else {
#pragma unroll
                    for (int a = 0; a < MT; a++) mx_mfma<XT>(acc[a][b], wr[b], sw[b], xr[a], sx[a]);
                }
            }
        }
    }
    /* the KS partial sums of each group, added in order; register i of a block: weight
     * row 4 g + i, x's row n */
#pragma unroll
    for (int a = 0; a < MT; a++)
#pragma unroll
        for (int b = 0; b < NT; b++)
            *(ghip_f32x4 *)(red + (wv * MR + 16u * a + n) * (16u * NT) + 16u * b + 4u * g) = acc[a][b];
    __syncthreads();
    ghip_with_act(ep.act, [&](auto act) {
        for (uint32_t v = tid; v < GPP * MR * 16u * OG; v += MR_WAVES * 64u) {
            const uint32_t sl = v / (MR * 16u * OG), e = v - sl * (MR * 16u * OG);
            const uint32_t m = e / (16u * OG), c = e % (16u * OG), o = (blk * GPP + sl) * (16u * OG) + c;
            if (m >= mrows || o >= p.N) continue;
            const float *q = red + (sl * KS * MR + m) * (16u * NT) + (DUAL ? 32u * (c >> 4) + (c & 15u) : c);
            float s0 = 0.0f, s1 = 0.0f;
#pragma unroll
            for (int k = 0; k < KS; k++) {
                s0 += q[k * MR * 16u * NT];
                if (DUAL) s1 += q[k * MR * 16u * NT + 16u];
            }
            ghip_ep_store<MODE, decltype(act)::value>(ep, ep.out, m0 + m, o, s0, s1);
        }
    });
}

struct MrForm {
    uint32_t mr, cols;
    const void *kern;
    uint32_t lds;
    void (*launch)(dim3, uint32_t, hipStream_t, const GhipMxProd &, const GhipEp &, uint32_t, uint32_t);
};
template <int XT, int MT, int NT, int KS, int MODE>
static void mr_run(dim3 grid, uint32_t lds, hipStream_t st, const GhipMxProd &p, const GhipEp &ep,
                   uint32_t blk0, uint32_t tile0) {
    hipLaunchKernelGGL((k_mx_rows<XT, MT, NT, KS, MODE>), grid, dim3(MR_WAVES * 64), lds, st, p, ep, blk0, tile0);
}
template <int XT, int MT, int NT, int KS, int MODE>
static constexpr MrForm mr_form() {
    return {16 * MT, (ghip_ep_dual(MODE) ? 8u : 16u) * NT * (MR_WAVES / KS),
            (const void *)k_mx_rows<XT, MT, NT, KS, MODE>, MR_WAVES * 16u * MT * 16u * NT * 4u,
            mr_run<XT, MT, NT, KS, MODE>};
}
static const MrForm mr_linear[3] = {mr_form<GHIP_BF16, 2, 2, 2, GHIP_EP_LINEAR>(),
                                    mr_form<GHIP_MXFP8, 2, 2, 2, GHIP_EP_LINEAR>(),
                                    mr_form<GHIP_MXFP4, 2, 2, 2, GHIP_EP_LINEAR>()};
static const MrForm mr_gated[3] = {mr_form<GHIP_BF16, 2, 2, 2, GHIP_EP_GATED>(),
                                   mr_form<GHIP_MXFP8, 2, 2, 2, GHIP_EP_GATED>(),
                                   mr_form<GHIP_MXFP4, 2, 2, 2, GHIP_EP_GATED>()};

#define MR_MAX_TILES ((size_t)65535)
#define MR_MAX_BLOCKS (GHIP_MAX_THREADS / (MR_WAVES * 64))

extern "C" hipError_t ghip_launch_mx_rows(int mode, int form, const GhipMxProd *p, const GhipEp *ep, hipStream_t st) {
    if (p->M == 0 || p->N == 0 || p->K == 0 || p->K % 32 || (mode != GHIP_EP_LINEAR && mode != GHIP_EP_GATED) || form)
        return hipErrorInvalidValue;
    const MrForm *c = (mode == GHIP_EP_GATED ? mr_gated : mr_linear) + p->xt;
    const size_t blocks = ((size_t)p->N + c->cols - 1) / c->cols, tiles = ((size_t)p->M + c->mr - 1) / c->mr;
    for (size_t t0 = 0; t0 < tiles; t0 += MR_MAX_TILES)
        for (size_t b0 = 0; b0 < blocks; b0 += MR_MAX_BLOCKS) {
            const size_t nt = tiles - t0 < MR_MAX_TILES ? tiles - t0 : MR_MAX_TILES;
            const size_t nb = blocks - b0 < MR_MAX_BLOCKS ? blocks - b0 : MR_MAX_BLOCKS;
            c->launch(dim3((uint32_t)nb, (uint32_t)nt), c->lds, st, *p, *ep, (uint32_t)b0, (uint32_t)t0);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    return hipSuccess;
}

extern "C" hipError_t ghip_mx_rows_init(void) {
    for (int i = 0; i < 6; i++) {
        const MrForm *c = i < 3 ? mr_linear + i : mr_gated + i - 3;
        const hipError_t e = hipFuncSetAttribute(c->kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)c->lds);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}
