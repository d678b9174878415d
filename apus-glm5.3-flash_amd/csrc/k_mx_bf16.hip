/*
 * k_mx_bf16.hip — products of BF16 activations with MXFP4 weights on tiles. The
 * kernel is k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_BF16, 1, 4, 12, 4, 4>(0.80f, 1.09f, 5.1f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 4, 6>(0.60f, 0.91f, 4.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 4, 3>(0.57f, 1.64f, 2.8f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 2, 6>(0.42f, 0.66f, 1.4f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 2, 3>(0.41f, 1.10f, 0.4f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 4, 2, 6>(0.34f, 0.87f, 0.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 2, 2, 8>(0.29f, 0.75f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_bf16_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
