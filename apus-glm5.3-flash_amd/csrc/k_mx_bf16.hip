/*
 * k_mx_bf16.hip — products of BF16 activations with MXFP4 weights on tiles. The
 * kernel is k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_BF16, 1, 4, 12, 4, 4>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 4, 6>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 4, 3>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 2, 6>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 2, 3>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 4, 2, 6>(1.0f, 1.0f, 1.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 2, 2, 8>(1.0f, 1.0f, 1.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_bf16_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
