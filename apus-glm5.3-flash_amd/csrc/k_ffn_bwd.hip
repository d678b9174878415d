/*
 * k_ffn_bwd.hip — the backward products on tiles: dz (and dg, du) from the
 * forward's sums computed again, dx = dz W (W read with k as the slow index)
 * and dW = dz^T x (both so). The kernel is k_ffn_gemm.h's.
 */
#include "k_ffn_tile.h"

static const GhipFfnTile *dlinear_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 8, 8, 2>(0.99f, 1.39f, 9.6f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 6, 8, 2>(0.87f, 1.12f, 4.2f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 8, 4, 2>(0.65f, 0.88f, 1.9f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 6, 4, 2>(0.59f, 0.76f, 0.0f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 4, 4, 4>(0.38f, 0.54f, 1.1f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 4, 4, 2>(0.47f, 0.98f, 0.0f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 2, 4, 5>(0.32f, 0.38f, 0.0f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 2, 2, 6>(0.22f, 0.25f, 0.8f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 2, 2, 3>(0.20f, 0.42f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

static const GhipFfnTile *dgated_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 8, 8, 2>(1.01f, 1.37f, 15.3f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 6, 8, 2>(1.00f, 1.15f, 8.7f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 6, 4, 2>(0.72f, 0.82f, 2.0f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 4, 4, 4>(0.41f, 0.55f, 3.2f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 4, 4, 2>(0.66f, 1.02f, 0.0f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 2, 4, 5>(0.44f, 0.43f, 0.4f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 2, 2, 6>(0.28f, 0.27f, 1.0f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 2, 2, 3>(0.28f, 0.46f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

static const GhipFfnTile *dx_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 8, 8, 2>(1.01f, 1.42f, 7.0f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 8, 4, 2>(0.56f, 0.82f, 4.0f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 4, 4, 4>(0.37f, 0.52f, 2.8f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 4, 4, 2>(0.33f, 0.92f, 2.8f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 2, 4, 5>(0.26f, 0.36f, 2.0f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 2, 2, 6>(0.19f, 0.25f, 1.6f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 2, 2, 3>(0.16f, 0.42f, 1.2f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

static const GhipFfnTile *dw_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 8, 8, 2>(1.09f, 1.51f, 7.1f),
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 4, 4, 4>(0.43f, 0.54f, 2.9f),
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 4, 4, 2>(0.34f, 0.93f, 2.9f),
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 2, 4, 5>(0.28f, 0.36f, 2.1f),
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 2, 2, 6>(0.22f, 0.27f, 1.6f),
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 2, 2, 3>(0.18f, 0.43f, 1.2f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipFfnTile *ghip_ffn_backward_tiles(int mode, int transposed, int *n) {
    if (mode == GHIP_EP_DGATED) return dgated_tiles(n);
    if (mode == GHIP_EP_DLINEAR) return dlinear_tiles(n);
    return transposed ? dw_tiles(n) : dx_tiles(n);
}
