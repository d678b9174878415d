/*
 * k_ffn_tile.h — an entry of a tile table (GhipFfnTile) over k_ffn_gemm.
 */
#ifndef K_FFN_TILE_H
#define K_FFN_TILE_H

#include "k_ffn_gemm.h"

template <int MODE, int W8, int AL, int BL, int RB, int CB, int L>
static void fg_run(const GhipProd *p, const GhipEp *ep, uint32_t mt, uint32_t nt, uint32_t lds,
                   hipStream_t st) {
    hipLaunchKernelGGL((k_ffn_gemm<MODE, W8, AL, BL, RB, CB, L>),
                       dim3(mt * nt * (p->batch ? 2u : 1u)), dim3(256), lds, st, *p, *ep, mt, nt);
}

template <int MODE, int W8, int AL, int BL, int RB, int CB, int L>
static constexpr GhipFfnTile fg_tile(float us) {
    return {32u * RB, ghip_ep_dual(MODE) ? 16u * CB : 32u * CB, us,
            (L + 1u) * RB * 4096u + L * CB * (W8 ? 2048u : 4096u),
            (const void *)k_ffn_gemm<MODE, W8, AL, BL, RB, CB, L>,
            fg_run<MODE, W8, AL, BL, RB, CB, L>};
}

#endif /* K_FFN_TILE_H */
