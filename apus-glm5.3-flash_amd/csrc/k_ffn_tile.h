/*
 * k_ffn_tile.h — an entry of a tile table (GhipFfnTile) over k_ffn_gemm.
 */
#ifndef K_FFN_TILE_H
#define K_FFN_TILE_H

#include "k_ffn_gemm.h"

template <int MODE, bool FP8, int AL, int BL, int WM, int WN, int RB, int NS>
static void fg_run(const GhipProd *p, const GhipEp *ep, uint32_t mt, uint32_t nt, uint32_t lds,
                   hipStream_t st) {
    hipLaunchKernelGGL((k_ffn_gemm<MODE, FP8, AL, BL, WM, WN, RB, NS>),
                       dim3(mt * nt * (p->batch ? 2u : 1u)), dim3(WM * WN * 64), lds, st, *p, *ep, mt,
                       nt);
}

template <int MODE, bool FP8, int AL, int BL, int WM, int WN, int RB, int NS>
static constexpr GhipFfnTile fg_tile(float us) {
    return {32u * RB * WM, ghip_ep_dual(MODE) ? 32u * WN : 64u * WN, us,
            NS * (32u * RB * WM + 64u * WN) * 128u,
            (const void *)k_ffn_gemm<MODE, FP8, AL, BL, WM, WN, RB, NS>,
            fg_run<MODE, FP8, AL, BL, WM, WN, RB, NS>};
}

#endif /* K_FFN_TILE_H */
