/*
 * k_mx_fp4.hip — products of MXFP4 activations with MXFP4 weights on tiles. The kernel is
 * k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 8, 8, 4>({0.62f, 0.00f, 1.09f, 6.6f}, {0.65f, 0.00f, 1.07f, 7.5f}),
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 8, 4, 6>({0.40f, 0.00f, 0.69f, 4.2f}, {0.43f, 0.00f, 0.67f, 4.7f}),
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 4, 4, 3>({0.25f, 0.43f, 0.80f, 1.7f}, {0.28f, 0.47f, 0.79f, 2.0f}),
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 2, 4, 6>({0.20f, 0.27f, 0.55f, 1.6f}, {0.23f, 0.35f, 0.54f, 1.8f}),
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 2, 2, 8>({0.15f, 0.17f, 0.35f, 1.5f}, {0.16f, 0.23f, 0.37f, 1.7f}),
        mg_tile<MODE, GHIP_MXFP4, 1, 2, 2, 2, 8>({0.14f, 0.15f, 0.23f, 1.4f}, {0.17f, 0.22f, 0.25f, 1.7f}),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_fp4_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
