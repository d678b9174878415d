/*
 * k_mx_fp4.hip — products of MXFP4 activations with MXFP4 weights on tiles. The kernel is
 * k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 8, 8, 4>(0.64f, 0.00f, 1.35f, 6.1f),
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 8, 4, 6>(0.45f, 0.00f, 0.99f, 3.1f),
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 4, 4, 3>(0.30f, 0.57f, 1.09f, 0.8f),
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 2, 4, 4>(0.28f, 0.48f, 0.88f, 0.0f),
        mg_tile<MODE, GHIP_MXFP4, 2, 2, 2, 2, 5>(0.21f, 0.36f, 0.71f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_fp4_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
