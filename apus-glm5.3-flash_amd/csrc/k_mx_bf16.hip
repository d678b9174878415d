/*
 * k_mx_bf16.hip — products of BF16 activations with MXFP4 weights on tiles. The
 * kernel is k_mx_gemm.h's.
 */
#include "k_mx_tile.h"

template <int MODE>
static const GhipMxTile *tiles(int *n) {
    static const GhipMxTile t[] = {
        mg_tile<MODE, GHIP_BF16, 1, 4, 12, 4, 4>(0.81f, 0.00f, 1.08f, 5.1f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 4, 6>(0.60f, 0.00f, 0.90f, 4.1f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 4, 3>(0.59f, 0.89f, 1.93f, 3.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 8, 2, 3>(0.43f, 0.64f, 1.18f, 0.4f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 4, 2, 6>(0.36f, 0.54f, 0.90f, 0.0f),
        mg_tile<MODE, GHIP_BF16, 1, 4, 2, 2, 8>(0.32f, 0.44f, 0.78f, 0.0f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipMxTile *ghip_mx_bf16_tiles(int mode, int *n) {
    return mode == GHIP_EP_GATED ? tiles<GHIP_EP_GATED>(n) : tiles<GHIP_EP_LINEAR>(n);
}
