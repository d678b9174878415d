/*
 * k_mx_fp8.hip — products of MXFP8 activations with MXFP4 weights on tiles. The kernel is
 * k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 8, 8, 3>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 8, 4, 3>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 4, 8, 3>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 4, 4, 3>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 4, 4, 6>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 2, 4, 4>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_MXFP8, 2, 2, 2, 2, 5>(1.0f, 1.0f, 1.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_fp8_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
