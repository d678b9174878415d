/*
 * k_ffn_nt.hip — the forward products (x and W both with k as the fast index)
 * on tiles: y = act(x W^T + b) + r and h = act(x Wg^T) * (x Wu^T), BF16 weights.
 * The kernel is k_ffn_gemm.h's.
 */
#include "k_ffn_tile.h"

static const GhipFfnTile *linear_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 8, 8, 2>(1.01f, 0.00f, 1.39f, 8.5f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 6, 8, 2>(0.88f, 0.00f, 1.12f, 3.5f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 6, 4, 2>(0.58f, 0.00f, 0.74f, 0.0f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 4, 4, 4>(0.40f, 0.00f, 0.54f, 0.9f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 4, 4, 2>(0.49f, 0.66f, 0.97f, 0.0f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 2, 4, 5>(0.32f, 0.00f, 0.38f, 0.0f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 2, 2, 6>(0.22f, 0.00f, 0.26f, 0.6f),
        fg_tile<GHIP_EP_LINEAR, 0, 0, 0, 2, 2, 2, 3>(0.22f, 0.28f, 0.42f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

static const GhipFfnTile *gated_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 8, 8, 2>(1.03f, 0.00f, 1.33f, 5.9f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 6, 8, 2>(1.03f, 0.00f, 1.11f, 0.4f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 8, 4, 2>(0.75f, 0.00f, 0.86f, 0.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 6, 4, 2>(0.69f, 0.00f, 0.74f, 0.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 5, 4, 2>(0.68f, 0.00f, 0.73f, 0.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 4, 4, 4>(0.41f, 0.00f, 0.53f, 0.2f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 4, 4, 2>(0.60f, 0.72f, 0.92f, 0.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 2, 4, 5>(0.40f, 0.00f, 0.39f, 0.0f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 2, 2, 6>(0.26f, 0.00f, 0.26f, 0.4f),
        fg_tile<GHIP_EP_GATED, 0, 0, 0, 2, 2, 2, 3>(0.24f, 0.34f, 0.43f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipFfnTile *ghip_ffn_forward_tiles(int mode, int w8, int *n) {
    if (w8) return ghip_ffn_fp8_tiles(mode, w8, n);
    return mode == GHIP_EP_GATED ? gated_tiles(n) : linear_tiles(n);
}
