/*
 * k_ffn_rows.hip — the feed-forward products x W^T of a few rows (the forward,
 * and the sums that a backward pass computes again): the weight-streaming
 * kernel (k_rows_gemm.h) with an epilogue, for one weight matrix (linear) or
 * gate and up together (gated). Bound by HBM where the weights fill the chip
 * (operands from HBM: gated FP8 12288 x 4096, M = 1, 18.8 us, 5.4 TB/s; FP8 4096 x
 * 16384, M = 4, 12.8 us, 5.3 TB/s), by the launch, the first loads and the
 * reduction below that (under the profiler BF16 4096 x 2048, M = 1, 5.1 us; 1537 x
 * 4096, M = 37, 7.7).
 */
#include "k_rows_gemm.h"

#define FR_MAX_TILES ((size_t)65535)
#define FR_MAX_BLOCKS (GHIP_MAX_THREADS / (RW_NW * 64))

/* One launchable form: MR rows of x, NT weight groups of 16 a wave, K over KS
 * waves. chunk, over: microseconds of a wave's chunk step, and of a round's
 * first loads and reduction. */
struct FrForm {
    uint32_t mr, nt, ks;
    float chunk, over;
    const void *kern;
    uint32_t lds;
    void (*launch)(dim3, uint32_t, hipStream_t, const GhipProd &, const GhipEp &, uint32_t, uint32_t);
};

template <bool BF, int MR, int NT, int KS, int NA, int SL, int MODE>
static void fr_run(dim3 grid, uint32_t lds, hipStream_t st, const GhipProd &p, const GhipEp &ep,
                   uint32_t blk0, uint32_t tile0) {
    const RwMore more = {(const uint8_t *)p.b2, p.s2, (uint32_t)p.ars, p.exact, ep};
    hipLaunchKernelGGL((k_rows_gemm<BF, MR, NT, KS, NA, SL, MODE>), grid, dim3(RW_NW * 64), lds, st,
                       (const uint8_t *)p.b, p.s, p.a, ep.out, p.M, p.N, p.K, nullptr, blk0, tile0,
                       more);
}

#define FR_FORM(BF, MR, NT, KS, NA, SL, MODE, T, V)                                         \
    {MR, NT, KS, T, V, (const void *)k_rows_gemm<BF, MR, NT, KS, NA, SL, MODE>,               \
     rw_lds<BF, MR, NT, SL>(), fr_run<BF, MR, NT, KS, NA, SL, MODE>}

/* The times are fitted to a sweep of every form over M = 1..80, N x K from 1536
 * x 1536 to 12288 x 4096 and 4096 x 12288 on 256 CUs, operands from HBM; the
 * form picked by them took 1% longer than the best one on average, 15% at most.
 * Chunks in flight (NA) and slots (SL) are the plain linear's (k_rows.hip). */
#define FR_L(BF, MR, NT, KS, NA, SL, T, V) FR_FORM(BF, MR, NT, KS, NA, SL, GHIP_EP_LINEAR, T, V)
static const FrForm fr_linear8[] = {
    FR_L(false, 4, 1, 8, 2, 2, 0.60f, 0.11f),
    FR_L(false, 4, 1, 4, 2, 2, 0.49f, 0.29f),
    FR_L(false, 4, 1, 2, 2, 2, 0.44f, 0.37f),
    FR_L(false, 8, 1, 8, 2, 2, 0.70f, 0.60f),
    FR_L(false, 8, 1, 4, 2, 2, 0.59f, 0.69f),
    FR_L(false, 8, 1, 2, 2, 2, 0.51f, 0.72f),
    FR_L(false, 16, 1, 8, 1, 1, 0.84f, 0.10f),
    FR_L(false, 16, 2, 8, 2, 2, 1.26f, 0.62f),
    FR_L(false, 16, 2, 4, 2, 2, 1.06f, 1.36f),
    FR_L(false, 32, 1, 8, 1, 1, 1.11f, 0.57f),
    FR_L(false, 32, 2, 8, 1, 1, 1.42f, 0.81f),
    FR_L(false, 32, 2, 4, 1, 1, 1.30f, 1.35f),
    FR_L(false, 64, 2, 4, 1, 1, 1.90f, 3.13f),
};
static const FrForm fr_linear16[] = {
    FR_L(true, 8, 1, 8, 2, 2, 0.54f, 0.00f),
    FR_L(true, 8, 1, 4, 2, 2, 0.45f, 0.00f),
    FR_L(true, 16, 1, 8, 2, 2, 0.61f, 0.00f),
    FR_L(true, 16, 1, 4, 2, 2, 0.52f, 0.00f),
    FR_L(true, 16, 2, 4, 2, 2, 0.82f, 0.03f),
    FR_L(true, 32, 1, 8, 1, 1, 0.74f, 0.23f),
    FR_L(true, 32, 2, 8, 1, 1, 1.03f, 0.21f),
    FR_L(true, 32, 2, 4, 1, 1, 0.94f, 0.36f),
};
#define FR_G(BF, MR, NT, KS, NA, SL, T, V) FR_FORM(BF, MR, NT, KS, NA, SL, GHIP_EP_GATED, T, V)
static const FrForm fr_gated8[] = {
    FR_G(false, 4, 2, 8, 2, 2, 1.25f, 0.44f),
    FR_G(false, 4, 2, 4, 2, 2, 0.99f, 0.69f),
    FR_G(false, 4, 2, 2, 2, 2, 0.86f, 0.72f),
    FR_G(false, 8, 2, 8, 2, 2, 1.32f, 0.70f),
    FR_G(false, 8, 2, 4, 2, 2, 1.05f, 0.99f),
    FR_G(false, 16, 2, 8, 2, 2, 1.46f, 0.39f),
    FR_G(false, 16, 2, 4, 2, 2, 1.15f, 1.01f),
    FR_G(false, 32, 2, 8, 1, 1, 1.57f, 0.74f),
    FR_G(false, 32, 2, 4, 1, 1, 1.35f, 1.12f),
    FR_G(false, 64, 2, 4, 1, 1, 1.94f, 2.52f),
};
static const FrForm fr_gated16[] = {
    FR_G(true, 8, 2, 8, 2, 2, 0.97f, 0.00f),
    FR_G(true, 8, 2, 4, 2, 2, 0.81f, 0.00f),
    FR_G(true, 16, 2, 8, 2, 2, 1.08f, 0.00f),
    FR_G(true, 16, 2, 4, 2, 2, 0.87f, 0.00f),
    FR_G(true, 32, 2, 8, 1, 1, 1.12f, 0.00f),
    FR_G(true, 32, 2, 4, 1, 1, 0.99f, 0.00f),
};

/* dz, dg and du: the forward's sums again, at its times */
#define FR_DL(BF, MR, NT, KS, NA, SL, T, V) FR_FORM(BF, MR, NT, KS, NA, SL, GHIP_EP_DLINEAR, T, V)
static const FrForm fr_dlinear[] = {
    FR_DL(true, 8, 1, 8, 2, 2, 0.54f, 0.00f),
    FR_DL(true, 8, 1, 4, 2, 2, 0.45f, 0.00f),
    FR_DL(true, 16, 1, 8, 2, 2, 0.61f, 0.00f),
    FR_DL(true, 16, 1, 4, 2, 2, 0.52f, 0.00f),
    FR_DL(true, 16, 2, 4, 2, 2, 0.82f, 0.03f),
    FR_DL(true, 32, 1, 8, 1, 1, 0.74f, 0.23f),
    FR_DL(true, 32, 2, 8, 1, 1, 1.03f, 0.21f),
    FR_DL(true, 32, 2, 4, 1, 1, 0.94f, 0.36f),
};
#define FR_DG(BF, MR, NT, KS, NA, SL, T, V) FR_FORM(BF, MR, NT, KS, NA, SL, GHIP_EP_DGATED, T, V)
static const FrForm fr_dgated[] = {
    FR_DG(true, 8, 2, 8, 2, 2, 0.97f, 0.00f),
    FR_DG(true, 8, 2, 4, 2, 2, 0.81f, 0.00f),
    FR_DG(true, 16, 2, 8, 2, 2, 1.08f, 0.00f),
    FR_DG(true, 16, 2, 4, 2, 2, 0.87f, 0.00f),
    FR_DG(true, 32, 2, 8, 1, 1, 1.12f, 0.00f),
    FR_DG(true, 32, 2, 4, 1, 1, 0.99f, 0.00f),
};

static const FrForm *fr_forms(int mode, bool fp8, int *n) {
#define FR_TABLE(t) (*n = (int)(sizeof t / sizeof *t), t)
    if (mode == GHIP_EP_DLINEAR) return FR_TABLE(fr_dlinear);
    if (mode == GHIP_EP_DGATED) return FR_TABLE(fr_dgated);
    if (mode == GHIP_EP_GATED) return fp8 ? FR_TABLE(fr_gated8) : FR_TABLE(fr_gated16);
    return fp8 ? FR_TABLE(fr_linear8) : FR_TABLE(fr_linear16);
#undef FR_TABLE
}

/* Estimated microseconds of a form: 2.3 + the larger of its rounds of the chip
 * and the weights at 6.5 TB/s + a tenth of the other (within 10-15% rms of the
 * sweep); several row tiles of FP8 take 15% more on average for M = 64 to 300.
 * Forms of 4 and 8 rows only take as many. */
static float fr_estimate(const FrForm &c, const GhipProd *p, bool dual, uint32_t n_cu) {
    if (c.mr < 16 && p->M > c.mr) return 1e30f;
    const double cols = (dual ? 8.0 : 16.0) * c.nt * (RW_NW / c.ks);
    const double wgs = (double)(size_t)((p->N + cols - 1) / cols) * (double)((p->M + c.mr - 1) / c.mr);
    const double kb = (double)p->K * (p->s ? 1 : 2), nch = (double)(size_t)((kb + 127) / 128);
    const double rounds = (double)(size_t)((wgs + n_cu - 1) / n_cu);
    const double nc = (double)(size_t)((nch + c.ks - 1) / c.ks);
    const double hbm = (double)p->N * kb * (dual ? 2 : 1) / 6.5e6;
    const double t = rounds * (nc * c.chunk + c.over);
    const double again = p->s && p->M > c.mr ? 1.15 : 1.0;
    return (float)(2.3 + again * (t > hbm ? t + 0.1 * hbm : hbm + 0.1 * t));
}

/* Whole 16-byte pieces of x's rows (FP8 weight rows then start at 8 bytes, and
 * have 16 codes to read a half piece from), 32-bit offsets inside a wave's rows */
extern "C" int ghip_ffn_rows_fits(int mode, const GhipProd *p) {
    return mode != GHIP_EP_STORE && (!p->s || mode == GHIP_EP_LINEAR || mode == GHIP_EP_GATED) && p->aks == 1 && p->bks == 1
        && p->brs == p->K && p->K % 8 == 0 && (!p->s || p->K >= 16) && p->K <= (1u << 24) && p->ars % 8 == 0
        && p->ars <= (1u << 24) && p->M <= 0x7fffffffu && p->N <= 0x7fffffffu
        && (((uintptr_t)p->a | (uintptr_t)p->b | (uintptr_t)p->b2) & 15) == 0;
}

extern "C" int ghip_ffn_rows_pick(int mode, const GhipProd *p, uint32_t n_cu, float *us) {
    int n, best = 0;
    const FrForm *t = fr_forms(mode, p->s != nullptr, &n);
    for (int i = 0; i < n; i++) {
        const float e = fr_estimate(t[i], p, ghip_ep_dual(mode), n_cu);
        if (i == 0 || e < *us) {
            best = i;
            *us = e;
        }
    }
    return best;
}

extern "C" hipError_t ghip_launch_ffn_rows(int mode, int form, const GhipProd *p,
                                           const GhipEp *ep, hipStream_t st) {
    int n;
    const FrForm *c = fr_forms(mode, p->s != nullptr, &n);
    if (!ghip_ffn_rows_fits(mode, p) || form < 0 || form >= n || p->M == 0 || p->N == 0 || p->K == 0)
        return hipErrorInvalidValue;
    c += form;
    const size_t cols = (ghip_ep_dual(mode) ? 8u : 16u) * c->nt * (RW_NW / c->ks);
    const size_t blocks = (p->N + cols - 1) / cols, tiles = ((size_t)p->M + c->mr - 1) / c->mr;
    for (size_t t0 = 0; t0 < tiles; t0 += FR_MAX_TILES)
        for (size_t b0 = 0; b0 < blocks; b0 += FR_MAX_BLOCKS) {
            const size_t nt = tiles - t0 < FR_MAX_TILES ? tiles - t0 : FR_MAX_TILES;
            const size_t nb = blocks - b0 < FR_MAX_BLOCKS ? blocks - b0 : FR_MAX_BLOCKS;
            c->launch(dim3((uint32_t)nb, (uint32_t)nt), c->lds, st, *p, *ep, (uint32_t)b0,
                      (uint32_t)t0);
            const hipError_t e = hipGetLastError();
            if (e != hipSuccess) return e;
        }
    return hipSuccess;
}

extern "C" hipError_t ghip_ffn_rows_init(void) {
    static const int modes[6][2] = {{GHIP_EP_LINEAR, 0}, {GHIP_EP_LINEAR, 1}, {GHIP_EP_GATED, 0},
                                    {GHIP_EP_GATED, 1}, {GHIP_EP_DLINEAR, 0}, {GHIP_EP_DGATED, 0}};
    for (int i = 0; i < 6; i++) {
        int n;
        const FrForm *t = fr_forms(modes[i][0], modes[i][1], &n);
        for (int k = 0; k < n; k++) {
            const hipError_t e = hipFuncSetAttribute(
                t[k].kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)t[k].lds);
            if (e != hipSuccess) return e;
        }
    }
    return hipSuccess;
}
