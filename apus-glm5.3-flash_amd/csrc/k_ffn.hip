/*
 * k_ffn.hip — which kernel a dense feed-forward product takes (gfx950).
 */
#include "ghip_epilogue.h"

static uint32_t g_ffn_ncu;                       /* CUs: the routes' rounds */

static const GhipFfnTile *tiles_of(int mode, const GhipProd *p, int *n) {
    return mode == GHIP_EP_LINEAR || mode == GHIP_EP_GATED
               ? ghip_ffn_forward_tiles(mode, p->s ? p->exact ? 2 : 1 : 0, n)
               : ghip_ffn_backward_tiles(mode, p->aks != 1, n);
}

/* 16-byte loads along the fast index, from whole vectors, with offsets of 31
 * bits inside a tile (256 rows, or 64 k). */
static bool vectors(const void *q, size_t rs, size_t ks, size_t rows, size_t k, size_t per,
                    bool pad) {
    const size_t step = ks == 1 ? rs : ks, run = ks == 1 ? k : rows;
    return ((uintptr_t)q & 15) == 0 && (rs == 1 || ks == 1) && step % per == 0
           && (run % per == 0 || pad) && step < ((size_t)1 << 22);
}

extern "C" int ghip_ffn_gemm_fits(int mode, const GhipProd *p) {
    const bool fp8 = p->s != nullptr;
    const size_t per = fp8 ? 16 : 8;
    if (fp8 && mode != GHIP_EP_LINEAR && mode != GHIP_EP_GATED) return 0;
    /* the layouts that are built: k fast in both, in A alone, in neither */
    if (p->aks != 1 && p->bks == 1) return 0;
    if (mode != GHIP_EP_STORE && (p->aks != 1 || p->bks != 1)) return 0;
    if (mode == GHIP_EP_STORE && p->bks == 1) return 0;
    if (!vectors(p->a, p->ars, p->aks, p->M, p->K, 8, p->apad)
        || !vectors(p->b, p->brs, p->bks, p->N, p->K, per, false))
        return 0;
    if ((p->a2 && ((uintptr_t)p->a2 & 15)) || (p->b2 && ((uintptr_t)p->b2 & 15))) return 0;
    /* the smallest tile's grid: under 2^32 threads */
    return ((size_t)(p->M + 63) / 64) * ((size_t)(p->N + 63) / 64) * 2 * 256 <= GHIP_MAX_THREADS;
}

extern "C" int ghip_ffn_gemm_pick(int mode, const GhipProd *p, uint32_t n_cu, float *us) {
    int n, best = 0;
    const GhipFfnTile *t = tiles_of(mode, p, &n);
    const double stages = (double)((p->K + 63) / 64) * (p->a2 && !p->batch ? 2 : 1);
    for (int i = 0; i < n; i++) {
        const double wgs = (double)((p->M + t[i].bm - 1) / t[i].bm)
                           * (double)((p->N + t[i].bn - 1) / t[i].bn) * (p->batch ? 2 : 1);
        const double cap = (double)n_cu * t[i].occ, whole = (double)(size_t)(wgs / cap);
        const double part = wgs / cap - whole;           /* of the last round */
        const double e64 = 3.0 + whole * (stages * t[i].full + t[i].over)
                           + (part > 0.0 ? stages * (t[i].low + (t[i].full - t[i].low) * part) + t[i].over : 0.0);
        const float e = (float)e64;
        if (i == 0 || e < *us) {
            best = i;
            *us = e;
        }
    }
    return best;
}

extern "C" hipError_t ghip_launch_ffn_gemm(int mode, int tile, const GhipProd *p, const GhipEp *ep,
                                           hipStream_t st) {
    int n;
    const GhipFfnTile *t = tiles_of(mode, p, &n);
    if (!ghip_ffn_gemm_fits(mode, p) || tile < 0 || tile >= n) return hipErrorInvalidValue;
    t += tile;
    t->launch(p, ep, (p->M + t->bm - 1) / t->bm, (p->N + t->bn - 1) / t->bn, t->lds, st);
    return hipGetLastError();
}

extern "C" hipError_t ghip_launch_ffn(int mode, const GhipProd *p, const GhipEp *ep,
                                      hipStream_t st) {
    float us = 1e30f, rows_us = 1e30f;
    const int tile = g_ffn_ncu && ghip_ffn_gemm_fits(mode, p) ? ghip_ffn_gemm_pick(mode, p, g_ffn_ncu, &us) : -1;
    const int form = g_ffn_ncu && ghip_ffn_rows_fits(mode, p) ? ghip_ffn_rows_pick(mode, p, g_ffn_ncu, &rows_us) : -1;
    if (form >= 0 && rows_us <= us) return ghip_launch_ffn_rows(mode, form, p, ep, st);
    if (tile >= 0) return ghip_launch_ffn_gemm(mode, tile, p, ep, st);
    return ghip_launch_ffn_any(mode, p, ep, st);
}

extern "C" hipError_t ghip_ffn_init(uint32_t n_cu) {
    for (int i = 0; i < 10; i++) {
        static const int bwd[4][2] = {{GHIP_EP_DLINEAR, 0}, {GHIP_EP_DGATED, 0}, {GHIP_EP_STORE, 0}, {GHIP_EP_STORE, 1}};
        int n;
        const GhipFfnTile *t = i < 6 ? ghip_ffn_forward_tiles(i & 1 ? GHIP_EP_GATED : GHIP_EP_LINEAR, i >> 1, &n)
                                     : ghip_ffn_backward_tiles(bwd[i - 6][0], bwd[i - 6][1], &n);
        for (int k = 0; k < n; k++) {
            const hipError_t e = hipFuncSetAttribute(
                t[k].kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)t[k].lds);
            if (e != hipSuccess) return e;
        }
    }
    const hipError_t e = ghip_ffn_rows_init();
    if (e != hipSuccess) return e;
    g_ffn_ncu = n_cu;
    return hipSuccess;
}
