/*
 * k_ffn.hip — which kernel a dense feed-forward product takes (gfx950).
 */
#include <math.h>

#include "ghip_epilogue.h"

static uint32_t g_ffn_ncu;                       /* CUs: the routes' rounds */

static const GhipFfnTile *tiles_of(int mode, const GhipProd *p, int *n) {
    return mode == GHIP_EP_LINEAR || mode == GHIP_EP_GATED
               ? ghip_ffn_forward_tiles(mode, p->s ? p->exact ? 2 : 1 : 0, n)
               : ghip_ffn_backward_tiles(mode, p->aks != 1, n);
}

/* 16-byte loads along the fast index, from whole vectors (FP8: from whole 8
 * bytes), with offsets of 31
 * bits inside a tile (256 rows, or 64 k). */
static bool vectors(const void *q, size_t rs, size_t ks, size_t rows, size_t k, size_t per,
                    bool pad) {
    const size_t step = ks == 1 ? rs : ks, run = ks == 1 ? k : rows;
    return ((uintptr_t)q & 15) == 0 && (rs == 1 || ks == 1) && step % per == 0
           && (run % per == 0 || pad) && step < ((size_t)1 << 22);
}

extern "C" int ghip_ffn_gemm_fits(int mode, const GhipProd *p) {
    const bool fp8 = p->s != nullptr;
    if (fp8 && mode != GHIP_EP_LINEAR && mode != GHIP_EP_GATED) return 0;
    /* the layouts that are built: k fast in both, in A alone, in neither */
    if (p->aks != 1 && p->bks == 1) return 0;
    if (mode != GHIP_EP_STORE && (p->aks != 1 || p->bks != 1)) return 0;
    if (mode == GHIP_EP_STORE && p->bks == 1) return 0;
    if (!vectors(p->a, p->ars, p->aks, p->M, p->K, 8, p->apad)
        || !vectors(p->b, p->brs, p->bks, p->N, p->K, 8, false))
        return 0;
    if (fp8 && p->K < 16) return 0;                      /* a row's half piece needs a whole one */
    if ((p->a2 && ((uintptr_t)p->a2 & 15)) || (p->b2 && ((uintptr_t)p->b2 & 15))) return 0;
    return 1;
}

/* Workgroups of a tile; 0 where they are more than a launch takes. */
static size_t tile_grid(const GhipFfnTile *t, const GhipProd *p, uint32_t splits) {
    const size_t n = (((size_t)p->M + t->bm - 1) / t->bm) * (((size_t)p->N + t->bn - 1) / t->bn);
    return n > GHIP_MAX_THREADS / 256 / 2 / splits ? 0 : n * (p->batch ? 2 : 1) * splits;
}

/* Splits of k are for products of few tiles over a long k (dx of a wide block,
 * dW of many rows): each split's f32 sums go to memory and are added in order
 * by k_ffn_join. At most 16, of at least 8 stages, and 32 MiB of sums. */
#define FFN_MAX_SPLITS 16u
#define FFN_PART_BYTES ((size_t)32 << 20)

extern "C" size_t ghip_ffn_part_bytes(size_t M, size_t N, size_t K) {
    const size_t row = (N + 7) & ~(size_t)7, most = K / 512;
    if (M == 0 || N == 0 || row > FFN_PART_BYTES / 4 / M) return 0;
    const size_t one = M * row * 4;
    size_t n = FFN_PART_BYTES / one;
    if (n > most) n = most;
    if (n > FFN_MAX_SPLITS) n = FFN_MAX_SPLITS;
    return n < 2 ? 0 : (n * one + 255) & ~(size_t)255;
}

/* Estimated microseconds of a tile on n_cu CUs: 3 for the launch, and for each
 * round of the chip the stages and what a round costs besides. A round that
 * does not fill the chip runs at a time between the empty chip's and the full
 * one's; where a CU holds two workgroups, the few that share a CU set the
 * round's time long before all do. */
static double tile_us(const GhipFfnTile *t, const GhipProd *p, double stages, uint32_t splits,
                      uint32_t n_cu) {
    const double wgs = (double)tile_grid(t, p, splits);
    const double cap = (double)n_cu * t->occ, whole = (double)(size_t)(wgs / cap);
    const double part = wgs / cap - whole;               /* of the last round */
    double us = t->low + (t->full - t->low) * part;
    if (t->occ == 2)
        us = part <= 0.5 ? t->low + (t->mid - t->low) * 2.0 * part
                         : t->mid + (t->full - t->mid) * sqrt(2.0 * part - 1.0);
    return 3.0 + whole * (stages * t->full + t->over) + (part > 0.0 ? stages * us + t->over : 0.0);
}

static double stages_of(const GhipProd *p) {
    return (double)((p->K + 63) / 64) * (p->a2 && !p->batch ? 2 : 1);
}

/* Cells of one split's sums, and how many splits there may be. */
static size_t cells_of(const GhipProd *p) {
    return (size_t)p->M * (((size_t)p->N + 7) & ~(size_t)7) * (p->batch ? 2 : 1);
}
static uint32_t most_splits(const GhipProd *p) {
    if (!p->part) return 1;
    const size_t fit = p->part_bytes / 4 / cells_of(p), len = (size_t)(stages_of(p) / 8);
    const size_t n = fit < len ? fit : len;
    return n < 1 ? 1u : n > FFN_MAX_SPLITS ? FFN_MAX_SPLITS : (uint32_t)n;
}

extern "C" int ghip_ffn_gemm_pick(int mode, const GhipProd *p, uint32_t n_cu, float *us,
                                  uint32_t *splits) {
    int n, best = -1;
    const GhipFfnTile *t = tiles_of(mode, p, &n);
    const double stages = stages_of(p);
    const size_t cells = cells_of(p);
    const uint32_t most = mode == GHIP_EP_STORE ? most_splits(p) : 1;
    *us = 1e30f;
    for (int i = 0; i < n; i++)
        for (uint32_t s = 1; s <= most; s++) {
            if (!tile_grid(t + i, p, s)) continue;
            /* the sums' way out and back at 3 TB/s, and one more launch */
            const double join = s > 1 ? 4.0 + (double)cells * 4.0 * s * 2.0 / 3e6 : 0.0;
            const float e = (float)(tile_us(t + i, p, (double)(size_t)((stages + s - 1) / s), s, n_cu) + join);
            if (e < *us) {
                best = i;
                *us = e;
                *splits = s;
            }
        }
    return best;
}

/* out[m, n] = bf16(sum over the splits of part[s, m, n]), in order. */
__global__ __launch_bounds__(256) void k_ffn_join(const float *__restrict__ part, uint32_t splits,
                                                  uint32_t M, uint32_t N, size_t ldout,
                                                  uint16_t *out, uint16_t *out2) {
    const uint32_t per = (N + 7u) / 8u;
    const size_t one = (size_t)M * per * 8u, all = (size_t)M * per * (out2 ? 2u : 1u);
    for (size_t v = (size_t)blockIdx.x * 256u + threadIdx.x; v < all; v += (size_t)gridDim.x * 256u) {
        const bool second = v >= (size_t)M * per;
        const size_t w = second ? v - (size_t)M * per : v, m = w / per;
        const uint32_t n = (uint32_t)(w % per) * 8u;
        const float *q = part + (second ? splits * one : 0) + w * 8u;
        ghip_f32x4 a = {0.f, 0.f, 0.f, 0.f}, b = a;
#pragma unroll 4
        for (uint32_t s = 0; s < splits; s++) {
            a += *(const ghip_f32x4 *)(q + s * one);
            b += *(const ghip_f32x4 *)(q + s * one + 4);
        }
        uint16_t *o = (second ? out2 : out) + m * ldout + n, r[8];
#pragma unroll
        for (uint32_t e = 0; e < 8; e++) r[e] = (uint16_t)ghip_bf16_bits(e < 4 ? a[e & 3u] : b[e & 3u]);
        if (n + 8u <= N) {
            __builtin_memcpy(o, r, 16);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++)
                if (n + e < N) o[e] = r[e];
        }
    }
}

/* p as tile t takes it in `splits` pieces of k; false where it cannot. */
static bool split_up(int mode, const GhipFfnTile *t, uint32_t splits, const GhipProd *p, GhipProd *q) {
    if (splits < 1 || !tile_grid(t, p, splits)) return false;
    if (splits > 1
        && (mode != GHIP_EP_STORE || !p->part || splits > stages_of(p) || splits > p->part_bytes / 4 / cells_of(p)
            || ((uintptr_t)p->part & 15)))
        return false;
    *q = *p;
    q->splits = splits;
    if (splits == 1) q->part = nullptr;
    return true;
}

static hipError_t join(const GhipProd *p, const GhipEp *ep, hipStream_t st) {
    const size_t blocks = (cells_of(p) / 8 + 255) / 256;
    hipLaunchKernelGGL(k_ffn_join, dim3((uint32_t)(blocks < 8192 ? blocks : 8192)), dim3(256), 0, st,
                       p->part, p->splits, p->M, p->N, ep->ldout, ep->out, p->batch ? ep->out2 : nullptr);
    return hipGetLastError();
}

extern "C" hipError_t ghip_launch_ffn_gemm(int mode, int tile, uint32_t splits, const GhipProd *p,
                                           const GhipEp *ep, hipStream_t st) {
    int n;
    const GhipFfnTile *t = tiles_of(mode, p, &n);
    GhipProd q;
    if (!ghip_ffn_gemm_fits(mode, p) || tile < 0 || tile >= n || !split_up(mode, t + tile, splits, p, &q))
        return hipErrorInvalidValue;
    t += tile;
    t->launch(&q, ep, (p->M + t->bm - 1) / t->bm, (p->N + t->bn - 1) / t->bn, t->lds, st);
    const hipError_t e = hipGetLastError();
    return e != hipSuccess || splits == 1 ? e : join(&q, ep, st);
}

/* dx and dW in one launch take about 3 us, the larger of the longest workgroup's
 * time and the whole's share of the full chip, and 0.7 of the other (within 18%
 * rms of 150 shapes; the choice by it 2% slower than the best one on average, 24%
 * faster than two launches). At most one of the two is split, as they would share
 * the partial sums' memory. */
extern "C" int ghip_ffn_pair_pick(const GhipProd *dx, const GhipProd *dw, uint32_t n_cu, int tile[2],
                                  uint32_t splits[2]) {
    const GhipProd *const p[2] = {dx, dw};
    const GhipFfnTile *t[2];
    int nt[2], n, best = -1;
    double stages[2], join[2], us = 0.0;
    uint32_t most[2];
    for (int i = 0; i < 2; i++) {
        float one;
        uint32_t s;
        if (!n_cu || !ghip_ffn_gemm_fits(GHIP_EP_STORE, p[i])
            || ghip_ffn_gemm_pick(GHIP_EP_STORE, p[i], n_cu, &one, &s) < 0)
            return -1;
        us += one;
        t[i] = tiles_of(GHIP_EP_STORE, p[i], &nt[i]);
        stages[i] = stages_of(p[i]);
        most[i] = most_splits(p[i]);
        join[i] = (double)cells_of(p[i]) * 4.0 * 2.0 / 3e6;
    }
    const GhipFfnPair *const pairs = ghip_ffn_pairs(&n);
    for (int i = 0; i < n; i++) {
        int at[2];
        for (int k = 0; k < 2; k++) {
            const uint32_t *want = k ? pairs[i].dw : pairs[i].dx;
            for (at[k] = 0; at[k] < nt[k]; at[k]++) {
                const GhipFfnTile *c = t[k] + at[k];
                if (c->bm == want[0] && c->bn == want[1] && c->lds == want[2]) break;
            }
            if (at[k] == nt[k]) return -1;
        }
        for (uint32_t v = 1; v < most[0] + most[1]; v++) {
            const uint32_t s[2] = {v <= most[0] ? v : 1u, v <= most[0] ? 1u : v - most[0] + 1u};
            double longest = 0.0, whole = 0.0, extra = 0.0;
            bool fits = true;
            for (int k = 0; k < 2; k++) {
                const GhipFfnTile *c = t[k] + at[k];
                const size_t grid = tile_grid(c, p[k], s[k]);
                const double len = (double)(size_t)((stages[k] + s[k] - 1) / s[k]);
                const double chain = len * c->low + c->over;
                fits = fits && grid;
                whole += (double)grid / ((double)n_cu * c->occ) * (len * c->full + c->over);
                if (chain > longest) longest = chain;
                if (s[k] > 1) extra = 4.0 + join[k] * s[k];
            }
            const double e = 3.0 + (whole > longest ? whole + 0.7 * longest : longest + 0.7 * whole) + extra;
            if (fits && e < us) {
                us = e;
                best = i;
                for (int k = 0; k < 2; k++) {
                    tile[k] = at[k];
                    splits[k] = s[k];
                }
            }
        }
    }
    return best;
}

/* dbias goes with the products up to this many rows: its 256 threads a workgroup
 * take 32 of them at a time, a launch of its own 256. A pair of 12.4 us takes 12.5
 * with the sum of 1024 x 2048 (16.8 with a launch more) and 26.6 with that of 2048
 * x 2048 (19.2). */
#define FFN_SUM_ROWS 1024u
#define FFN_PAIR_LDS (80u * 1024u)                 /* two workgroups a CU */

extern "C" hipError_t ghip_launch_ffn_grads(const GhipProd *dx, const GhipEp *edx, const GhipProd *dw,
                                            const GhipEp *edw, const GhipFfnSum *sum, hipStream_t st) {
    int tile[2], n;
    uint32_t splits[2];
    hipError_t e = hipSuccess;
    const int pair = dx && dw ? ghip_ffn_pair_pick(dx, dw, g_ffn_ncu, tile, splits) : -1;
    GhipProd x, w;
    if (pair >= 0) {
        const GhipFfnTile *tx = tiles_of(GHIP_EP_STORE, dx, &n) + tile[0];
        const GhipFfnTile *tw = tiles_of(GHIP_EP_STORE, dw, &n) + tile[1];
        const bool with = sum && sum->M <= FFN_SUM_ROWS;
        if (split_up(GHIP_EP_STORE, tx, splits[0], dx, &x) && split_up(GHIP_EP_STORE, tw, splits[1], dw, &w)
            && tile_grid(tx, dx, splits[0]) + tile_grid(tw, dw, splits[1]) <= GHIP_MAX_THREADS / 256 / 2) {
            ghip_ffn_pairs(&n)[pair].launch(&x, edx, &w, edw, with ? sum : nullptr, tx, tw, st);
            e = hipGetLastError();
            if (e == hipSuccess && splits[0] > 1) e = join(&x, edx, st);
            if (e == hipSuccess && splits[1] > 1) e = join(&w, edw, st);
            return e == hipSuccess && sum && !with ? ghip_launch_ffn_colsum(sum, st) : e;
        }
    }
    if (dx) e = ghip_launch_ffn(GHIP_EP_STORE, dx, edx, st);
    if (e == hipSuccess && dw) e = ghip_launch_ffn(GHIP_EP_STORE, dw, edw, st);
    return e == hipSuccess && sum ? ghip_launch_ffn_colsum(sum, st) : e;
}

extern "C" hipError_t ghip_launch_ffn(int mode, const GhipProd *p, const GhipEp *ep,
                                      hipStream_t st) {
    float us = 1e30f, rows_us = 1e30f;
    uint32_t splits = 1;
    const int tile = g_ffn_ncu && ghip_ffn_gemm_fits(mode, p)
                         ? ghip_ffn_gemm_pick(mode, p, g_ffn_ncu, &us, &splits) : -1;
    const int form = g_ffn_ncu && ghip_ffn_rows_fits(mode, p) ? ghip_ffn_rows_pick(mode, p, g_ffn_ncu, &rows_us) : -1;
    if (form >= 0 && rows_us <= us) return ghip_launch_ffn_rows(mode, form, p, ep, st);
    if (tile >= 0) return ghip_launch_ffn_gemm(mode, tile, splits, p, ep, st);
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
    int n;
    const GhipFfnPair *pairs = ghip_ffn_pairs(&n);
    for (int i = 0; i < n; i++) {
        const hipError_t e = hipFuncSetAttribute(
            pairs[i].kern, hipFuncAttributeMaxDynamicSharedMemorySize, (int)(FFN_PAIR_LDS));
        if (e != hipSuccess) return e;
    }
    hipError_t e = ghip_ffn_rows_init();
    if (e != hipSuccess || (e = ghip_mx_init(n_cu)) != hipSuccess) return e;
    g_ffn_ncu = n_cu;
    return hipSuccess;
}
