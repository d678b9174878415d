/*
 * k_mx_bf16.hip — products of BF16 activations with MXFP4 weights on tiles. The
 * kernel is k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_BF16, 1, 4, 12, 4, 4>({0.85f, 0.00f, 1.03f, 6.2f}, {0.85f, 0.00f, 1.03f, 6.4f}),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 4, 3>({0.64f, 0.00f, 0.80f, 4.0f}, {0.65f, 0.00f, 0.79f, 4.2f}),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 2, 3>({0.39f, 0.50f, 0.91f, 2.1f}, {0.40f, 0.52f, 0.89f, 2.2f}),
        mg_tile<MODE, GHIP_BF16, 1, 4, 4, 2, 6>({0.27f, 0.33f, 0.56f, 2.1f}, {0.28f, 0.34f, 0.55f, 2.2f}),
        mg_tile<MODE, GHIP_BF16, 1, 4, 2, 2, 8>({0.23f, 0.25f, 0.41f, 1.8f}, {0.23f, 0.27f, 0.40f, 2.1f}),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_bf16_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
