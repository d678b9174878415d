/*
 * k_ffn_nt.hip — the forward products (x and W both with k as the fast index)
 * on tiles: y = act(x W^T + b) + r and h = act(x Wg^T) * (x Wu^T), BF16 or
 * FP8-block weights. The kernel is k_ffn_gemm.h's.
 */
#include "k_ffn_tile.h"

template <int MODE>
static const GhipFfnTile *bf16_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<MODE, false, 0, 0, 2, 4, 4, 2>(1.60f), fg_tile<MODE, false, 0, 0, 2, 2, 4, 3>(0.90f),
        fg_tile<MODE, false, 0, 0, 2, 2, 2, 4>(0.55f), fg_tile<MODE, false, 0, 0, 2, 2, 1, 5>(0.40f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

template <int MODE>
static const GhipFfnTile *fp8_tiles(int *n) {
    static const GhipFfnTile t[] = {
        fg_tile<MODE, true, 0, 0, 2, 4, 4, 2>(1.80f), fg_tile<MODE, true, 0, 0, 2, 2, 2, 2>(0.70f),
        fg_tile<MODE, true, 0, 0, 2, 2, 1, 2>(0.60f),
    };
    *n = sizeof t / sizeof *t;
    return t;
}

extern "C" const GhipFfnTile *ghip_ffn_forward_tiles(int mode, int fp8, int *n) {
    if (mode == GHIP_EP_GATED) return fp8 ? fp8_tiles<GHIP_EP_GATED>(n) : bf16_tiles<GHIP_EP_GATED>(n);
    return fp8 ? fp8_tiles<GHIP_EP_LINEAR>(n) : bf16_tiles<GHIP_EP_LINEAR>(n);
}
