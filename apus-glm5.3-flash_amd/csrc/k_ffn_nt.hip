/*
 * k_ffn_nt.hip — the forward products (x and W both with k as the fast index)
 * on tiles: y = act(x W^T + b) + r and h = act(x Wg^T) * (x Wu^T), BF16 or
 * FP8-block weights. The kernel is k_ffn_gemm.h's.
 */
#include "k_ffn_tile.h"

template <int MODE>
static const GhipFfnTile *bf16_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<MODE, 0, 0, 0, 8, 8, 2>(1.50f), fg_tile<MODE, 0, 0, 0, 8, 4, 2>(0.90f),
        fg_tile<MODE, 0, 0, 0, 4, 4, 4>(0.55f), fg_tile<MODE, 0, 0, 0, 2, 4, 5>(0.40f),
        fg_tile<MODE, 0, 0, 0, 2, 2, 6>(0.30f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

template <int MODE, int W8>
static const GhipFfnTile *fp8_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<MODE, W8, 0, 0, 8, 8, 2>(1.60f), fg_tile<MODE, W8, 0, 0, 8, 4, 3>(1.00f),
        fg_tile<MODE, W8, 0, 0, 4, 4, 4>(0.60f), fg_tile<MODE, W8, 0, 0, 2, 4, 5>(0.45f),
        fg_tile<MODE, W8, 0, 0, 2, 2, 6>(0.32f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipFfnTile *ghip_ffn_forward_tiles(int mode, int w8, int *n) {
    if (mode == GHIP_EP_GATED)
        return w8 == 2 ? fp8_tiles<GHIP_EP_GATED, 2>(n)
               : w8    ? fp8_tiles<GHIP_EP_GATED, 1>(n) : bf16_tiles<GHIP_EP_GATED>(n);
    return w8 == 2 ? fp8_tiles<GHIP_EP_LINEAR, 2>(n)
           : w8    ? fp8_tiles<GHIP_EP_LINEAR, 1>(n) : bf16_tiles<GHIP_EP_LINEAR>(n);
}
