/*
 * k_mx_fp8.hip — products of MXFP8 activations with MXFP4 weights on tiles. The kernel is
 * k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 8, 8, 3>(0.96f, 1.61f, 6.3f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 8, 4, 3>(0.60f, 1.14f, 2.6f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 4, 8, 3>(0.66f, 1.17f, 2.5f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 4, 4, 3>(0.40f, 1.19f, 0.7f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 4, 4, 6>(0.43f, 0.72f, 1.5f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 2, 4, 4>(0.35f, 0.93f, 0.0f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 2, 2, 5>(0.27f, 0.74f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_fp8_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
