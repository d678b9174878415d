/*
 * k_ffn_nt8.hip — the forward products with FP8-block weights on tiles. The
 * kernel is k_ffn_gemm.h's.
 */
#include "k_ffn_tile.h"

template <int W8>
static const GhipFfnTile *linear_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 16, 4, 2>(1.24f, 1.54f, 10.1f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 12, 4, 2>(1.04f, 1.20f, 7.7f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 12, 2, 2>(0.72f, 0.80f, 4.2f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 8, 2, 4>(0.57f, 0.63f, 3.2f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 8, 2, 2>(0.57f, 1.02f, 1.2f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 4, 1, 6>(0.27f, 0.44f, 1.6f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 4, 1, 3>(0.28f, 0.40f, 0.8f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

template <int W8>
static const GhipFfnTile *gated_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 16, 4, 2>(1.22f, 1.51f, 6.3f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 12, 4, 2>(1.01f, 1.19f, 5.2f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 12, 2, 2>(0.70f, 0.79f, 2.3f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 8, 2, 4>(0.56f, 0.62f, 2.4f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 8, 2, 2>(0.52f, 0.99f, 1.0f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 2, 2, 2, 6>(0.32f, 0.49f, 1.6f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 2, 2, 2, 3>(0.34f, 0.45f, 0.5f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipFfnTile *ghip_ffn_fp8_tiles(int mode, int w8, int *n) {
    if (mode == GHIP_EP_GATED) return w8 == 2 ? gated_tiles<2>(n) : gated_tiles<1>(n);
    return w8 == 2 ? linear_tiles<2>(n) : linear_tiles<1>(n);
}
