/*
 * k_ffn_bwd.hip — the backward products on tiles: dz (and dg, du) from the
 * forward's sums computed again, dx = dz W (W read with k as the slow index)
 * and dW = dz^T x (both so). The kernel is k_ffn_gemm.h's.
 */
#include "k_ffn_tile.h"

template <int MODE>
static const GhipFfnTile *dz_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<MODE, 0, 0, 0, 8, 8, 2>(1.50f), fg_tile<MODE, 0, 0, 0, 8, 4, 2>(0.90f),
        fg_tile<MODE, 0, 0, 0, 4, 4, 4>(0.55f), fg_tile<MODE, 0, 0, 0, 2, 4, 5>(0.40f),
        fg_tile<MODE, 0, 0, 0, 2, 2, 6>(0.30f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

template <int AL>
static const GhipFfnTile *grad_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<GHIP_EP_STORE, 0, AL, 1, 8, 8, 2>(1.50f), fg_tile<GHIP_EP_STORE, 0, AL, 1, 8, 4, 2>(0.90f),
        fg_tile<GHIP_EP_STORE, 0, AL, 1, 4, 4, 4>(0.55f), fg_tile<GHIP_EP_STORE, 0, AL, 1, 2, 4, 5>(0.40f),
        fg_tile<GHIP_EP_STORE, 0, AL, 1, 2, 2, 6>(0.30f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipFfnTile *ghip_ffn_backward_tiles(int mode, int transposed, int *n) {
    if (mode == GHIP_EP_DGATED) return dz_tiles<GHIP_EP_DGATED>(n);
    if (mode == GHIP_EP_DLINEAR) return dz_tiles<GHIP_EP_DLINEAR>(n);
    return transposed ? grad_tiles<1>(n) : grad_tiles<0>(n);
}
