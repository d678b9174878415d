/*
 * k_mx_prod.hip — which kernel a product with MXFP4 weights takes (gfx950): the one with
 * the least estimated time of all tiles (k_mx_gemm.h) and all forms that stream the
 * weights past a few rows (k_mx_rows.hip). Both estimates are fitted to one sweep that
 * timed every one of them at 16 (1) to 4096 rows, the three types of x, linear and gated,
 * eight N x K. Over it the pick is 1 to 2% behind the best one's time on average and 22%
 * at worst (gated MXFP4 32 x 4096 x 4096: 8.5 us, 6.9 best). Rows against tiles, us:
 *   gated MXFP8, 4096 x 4096      16 rows 6.7 : 10.9
 *   gated MXFP8, 12288 x 4096     16 rows 13.0 : 17.0
 *   gated BF16, 12288 x 4096      16 rows 20.1 : 22.8
 * The linear takes tiles for any number of rows (k_mx_rows.hip). Tiles against each other
 * in MXFP8: 300 x 1537 x 4096 32x64 10.0, 64x64 10.8, 128x128 16.6, 256x256 46.3; 4096 x
 * 4096 x 4096 175, 112, 69.6 (256x128), 57.8.
 */
#include <math.h>

#include "ghip_device.h"
#include "ghip_internal.h"

static uint32_t g_mx_ncu = 256;                  /* CUs: the routes' rounds */

static const GhipMxTile *tiles_of(int mode, int xt, int *n) {
    return xt == GHIP_MXFP8 ? ghip_mx_fp8_tiles(mode, n) : xt == GHIP_MXFP4 ? ghip_mx_fp4_tiles(mode, n) : ghip_mx_bf16_tiles(mode, n);
}

/* Offsets inside a tile of 256 rows are of 31 bits. */
extern "C" int ghip_mx_gemm_fits(const GhipMxProd *p) {
    return p->xld < ((size_t)1 << 23) && p->K < (1u << 23);
}

static size_t tile_grid(const GhipMxTile *t, const GhipMxProd *p) {
    const size_t n = (((size_t)p->M + t->bm - 1) / t->bm) * (((size_t)p->N + t->bn - 1) / t->bn);
    return n > GHIP_MAX_THREADS / 512 ? 0 : n;
}

extern "C" int ghip_mx_gemm_tiles(int mode, int xt) {
    int n;
    tiles_of(mode, xt, &n);
    return n;
}

extern "C" hipError_t ghip_launch_mx_gemm(int mode, int tile, const GhipMxProd *p, const GhipEp *ep, hipStream_t st) {
    int n;
    const GhipMxTile *t = tiles_of(mode, p->xt, &n);
    if (p->M == 0 || p->N == 0 || p->K == 0 || p->K % 32 || (mode != GHIP_EP_LINEAR && mode != GHIP_EP_GATED)
        || !ghip_mx_gemm_fits(p) || tile < 0 || tile >= n || !tile_grid(t + tile, p))
        return hipErrorInvalidValue;
    t += tile;
    t->launch(p, ep, (p->M + t->bm - 1) / t->bm, (p->N + t->bn - 1) / t->bn, st);
    return hipGetLastError();
}

/* Estimated microseconds of a tile: 3 for the launch, and for each round of the chip
 * its steps and what a round costs besides. A round that does not fill the chip runs at
 * a time between the empty chip's and the full one's; where a CU holds two workgroups,
 * the few that share a CU set the round's time long before all do. */
static double tile_us(const GhipMxTile *t, const GhipMxProd *p) {
    const double cap = (double)g_mx_ncu * t->occ, rounds = (double)tile_grid(t, p) / cap;
    const double whole = (double)(size_t)rounds, part = rounds - whole;
    const uint32_t k = p->xt == GHIP_BF16 ? 64 : 128;
    const double steps = (double)(((p->K + k - 1) / k + 1) & ~1u);
    double us = t->low + (t->full - t->low) * part;
    if (t->occ == 2)
        us = part <= 0.5 ? t->low + (t->mid - t->low) * 2.0 * part
                         : t->mid + (t->full - t->mid) * sqrt(2.0 * part - 1.0);
    return 3.0 + whole * (steps * t->full + t->over) + (part > 0.0 ? steps * us + t->over : 0.0);
}

extern "C" int ghip_mx_gemm_pick(int mode, const GhipMxProd *p, float *us) {
    int n, best = -1;
    const GhipMxTile *t = tiles_of(mode, p->xt, &n);
    for (int i = 0; ghip_mx_gemm_fits(p) && i < n; i++) {
        if (!tile_grid(t + i, p)) continue;
        const float e = (float)tile_us(t + i, p);
        if (best < 0 || e < *us) {
            best = i;
            *us = e;
        }
    }
    return best;
}

/* The form with the least estimated time: rows of weights streamed past a few rows of
 * x, or tiles. */
extern "C" hipError_t ghip_launch_mx(int mode, const GhipMxProd *p, const GhipEp *ep, hipStream_t st) {
    float tile_t = 0.0f, rows_t = 0.0f;
    const int tile = ghip_mx_gemm_pick(mode, p, &tile_t), form = ghip_mx_rows_pick(mode, p, &rows_t);
    if (form >= 0 && (tile < 0 || rows_t <= tile_t)) return ghip_launch_mx_rows(mode, form, p, ep, st);
    if (tile < 0) return hipErrorNotSupported;               /* ghip_internal.h */
    return ghip_launch_mx_gemm(mode, tile, p, ep, st);
}

extern "C" hipError_t ghip_mx_init(uint32_t n_cu) {
    for (int i = 0; i < 6; i++) {
        int n;
        const GhipMxTile *t = tiles_of(i & 1 ? GHIP_EP_GATED : GHIP_EP_LINEAR, i >> 1, &n);
        for (int k = 0; k < n; k++) {
            const hipError_t e = hipFuncSetAttribute(t[k].kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)t[k].lds);
            if (e != hipSuccess) return e;
        }
    }
    const hipError_t e = ghip_mx_rows_init(n_cu);
    if (e != hipSuccess) return e;
    g_mx_ncu = n_cu;
    return hipSuccess;
}
