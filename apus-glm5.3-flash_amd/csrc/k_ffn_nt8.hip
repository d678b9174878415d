/*
 * k_ffn_nt8.hip — the forward products with FP8-block weights on tiles. The
 * kernel is k_ffn_gemm.h's.
 */
#include "k_ffn_tile.h"

template <int W8>
static const GhipFfnTile *linear_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 16, 4, 2>(1.25f, 0.00f, 1.54f, 8.0f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 12, 4, 2>(1.04f, 0.00f, 1.20f, 6.2f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 12, 2, 2>(0.66f, 0.00f, 0.74f, 3.3f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 8, 2, 4>(0.54f, 0.00f, 0.60f, 2.6f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 8, 2, 2>(0.59f, 0.68f, 1.00f, 0.7f),
        fg_tile<GHIP_EP_LINEAR, W8, 0, 0, 1, 4, 1, 3>(0.28f, 0.35f, 0.37f, 0.8f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

template <int W8>
static const GhipFfnTile *gated_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 16, 4, 2>(1.22f, 0.00f, 1.49f, 6.7f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 12, 4, 2>(1.02f, 0.00f, 1.18f, 5.2f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 12, 2, 2>(0.67f, 0.00f, 0.74f, 2.3f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 8, 2, 4>(0.54f, 0.00f, 0.60f, 2.3f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 1, 8, 2, 2>(0.58f, 0.64f, 0.96f, 1.0f),
        fg_tile<GHIP_EP_GATED, W8, 0, 0, 2, 2, 2, 3>(0.32f, 0.45f, 0.46f, 0.6f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipFfnTile *ghip_ffn_fp8_tiles(int mode, int w8, int *n) {
    if (mode == GHIP_EP_GATED) return w8 == 2 ? gated_tiles<2>(n) : gated_tiles<1>(n);
    return w8 == 2 ? linear_tiles<2>(n) : linear_tiles<1>(n);
}
