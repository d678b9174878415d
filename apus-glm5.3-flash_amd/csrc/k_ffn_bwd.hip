/*
 * k_ffn_bwd.hip — the backward products on tiles: dz (and dg, du) from the
 * forward's sums computed again, dx = dz W (W read with k as the slow index)
 * and dW = dz^T x (both so). The kernel is k_ffn_gemm.h's.
 */
#include "k_ffn_tile.h"

static const GhipFfnTile *dlinear_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 8, 8, 2>(1.03f, 0.00f, 1.42f, 9.7f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 6, 8, 2>(0.94f, 0.00f, 1.20f, 4.7f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 8, 4, 2>(0.72f, 0.00f, 0.97f, 3.2f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 6, 4, 2>(0.66f, 0.00f, 0.84f, 1.0f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 4, 4, 4>(0.45f, 0.00f, 0.60f, 2.0f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 4, 4, 2>(0.57f, 0.76f, 1.11f, 1.0f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 2, 4, 5>(0.35f, 0.00f, 0.42f, 1.0f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 2, 2, 6>(0.23f, 0.00f, 0.27f, 1.6f),
        fg_tile<GHIP_EP_DLINEAR, 0, 0, 0, 2, 2, 2, 3>(0.24f, 0.31f, 0.46f, 1.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

static const GhipFfnTile *dgated_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 8, 8, 2>(1.03f, 0.00f, 1.40f, 16.5f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 6, 8, 2>(1.02f, 0.00f, 1.13f, 9.0f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 6, 4, 2>(0.72f, 0.00f, 0.78f, 2.2f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 4, 4, 4>(0.48f, 0.00f, 0.59f, 4.1f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 4, 4, 2>(0.66f, 0.77f, 0.97f, 1.0f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 2, 4, 5>(0.43f, 0.00f, 0.41f, 1.1f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 2, 2, 6>(0.26f, 0.00f, 0.26f, 2.2f),
        fg_tile<GHIP_EP_DGATED, 0, 0, 0, 2, 2, 2, 3>(0.26f, 0.38f, 0.45f, 1.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

static const GhipFfnTile *dx_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 8, 8, 2>(1.02f, 0.00f, 1.41f, 7.1f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 8, 4, 2>(0.58f, 0.00f, 0.81f, 4.4f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 4, 4, 2>(0.38f, 0.49f, 0.93f, 2.9f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 2, 4, 5>(0.27f, 0.00f, 0.35f, 2.2f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 2, 2, 6>(0.19f, 0.00f, 0.25f, 1.8f),
        fg_tile<GHIP_EP_STORE, 0, 0, 1, 2, 2, 2, 3>(0.17f, 0.28f, 0.42f, 1.4f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

static const GhipFfnTile *dw_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 8, 8, 2>(1.11f, 0.00f, 1.49f, 7.4f),
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 4, 4, 2>(0.40f, 0.49f, 0.93f, 3.1f),
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 2, 4, 5>(0.29f, 0.00f, 0.36f, 2.4f),
        fg_tile<GHIP_EP_STORE, 0, 1, 1, 2, 2, 2, 3>(0.24f, 0.23f, 0.44f, 1.5f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipFfnTile *ghip_ffn_backward_tiles(int mode, int transposed, int *n) {
    if (mode == GHIP_EP_DGATED) return dgated_tiles(n);
    if (mode == GHIP_EP_DLINEAR) return dlinear_tiles(n);
    return transposed ? dw_tiles(n) : dx_tiles(n);
}
