/*
 * k_mx_fp8.hip — products of MXFP8 activations with MXFP4 weights on tiles. The kernel is
 * k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 8, 8, 3>(0.97f, 0.00f, 1.61f, 6.3f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 8, 4, 3>(0.60f, 0.00f, 1.14f, 2.6f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 4, 8, 3>(0.67f, 0.00f, 1.17f, 2.5f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 4, 4, 3>(0.42f, 0.70f, 1.25f, 0.7f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 2, 4, 4>(0.36f, 0.55f, 0.96f, 0.0f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 2, 2, 5>(0.31f, 0.41f, 0.78f, 0.0f),
        mg_tile<MODE, GHIP_MXFP8, 1, 2, 2, 2, 8>(0.22f, 0.24f, 0.46f, 0.5f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_fp8_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
