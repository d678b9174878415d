/*
 * k_mx_fp8.hip — products of MXFP8 activations with MXFP4 weights on tiles. The kernel is
 * k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 8, 8, 3>({1.00f, 0.00f, 1.46f, 7.0f}, {1.00f, 0.00f, 1.43f, 7.8f}),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 8, 4, 3>({0.56f, 0.00f, 0.87f, 4.0f}, {0.58f, 0.00f, 0.85f, 4.2f}),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 4, 4, 3>({0.32f, 0.53f, 1.00f, 2.0f}, {0.34f, 0.57f, 0.96f, 2.0f}),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 2, 4, 4>({0.22f, 0.34f, 0.63f, 1.2f}, {0.23f, 0.38f, 0.62f, 1.5f}),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 2, 2, 6>({0.18f, 0.22f, 0.42f, 1.4f}, {0.19f, 0.25f, 0.42f, 1.7f}),
        mg_tile<MODE, GHIP_MXFP8, 1, 2, 2, 2, 8>({0.15f, 0.17f, 0.30f, 1.7f}, {0.17f, 0.22f, 0.32f, 2.2f}),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_fp8_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
