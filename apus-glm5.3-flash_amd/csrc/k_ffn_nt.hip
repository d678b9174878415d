/*
 * k_ffn_nt.hip — the forward products (x and W both with k as the fast index)
 * on tiles: y = act(x W^T + b) + r and h = act(x Wg^T) * (x Wu^T), BF16 weights.
 * The kernel is k_ffn_gemm.h's.
 */
#include "k_ffn_tile.h"

static const GhipFfnTile *linear_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 8, 8, 2>(1.03f, 0.00f, 1.42f, 8.7f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 6, 8, 2>(0.94f, 0.00f, 1.20f, 3.7f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 6, 4, 2>(0.66f, 0.00f, 0.84f, 0.0f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 4, 4, 4>(0.45f, 0.00f, 0.60f, 1.0f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 4, 4, 2>(0.57f, 0.76f, 1.11f, 0.0f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 2, 4, 5>(0.35f, 0.00f, 0.42f, 0.0f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 2, 2, 6>(0.23f, 0.00f, 0.27f, 0.6f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 2, 2, 3>(0.24f, 0.31f, 0.46f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

static const GhipFfnTile *gated_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 8, 8, 2>(1.04f, 0.00f, 1.34f, 6.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 6, 8, 2>(1.03f, 0.00f, 1.10f, 0.4f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 6, 4, 2>(0.67f, 0.00f, 0.72f, 0.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 5, 4, 2>(0.65f, 0.00f, 0.70f, 0.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 4, 4, 4>(0.46f, 0.00f, 0.58f, 0.2f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 4, 4, 2>(0.58f, 0.70f, 0.88f, 0.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 2, 4, 5>(0.39f, 0.00f, 0.38f, 0.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 2, 2, 6>(0.25f, 0.00f, 0.25f, 0.4f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 2, 2, 3>(0.23f, 0.33f, 0.43f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipFfnTile *ghip_ffn_forward_tiles(int mode, int w8, int *n) {
    if (w8) return ghip_ffn_fp8_tiles(mode, w8, n);
    return mode == GHIP_EP_GATED ? gated_tiles(n) : linear_tiles(n);
}
