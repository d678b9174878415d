/*
 * k_ffn_tile.h — an entry of a tile table (GhipFfnTile) over k_ffn_gemm.
 *
 * Its times lie between those of operands from HBM and of operands that other
 * calls left in the chip's cache (BF16 tiles below 256 x 256 are 1.1 to 1.4 times
 * apart). They were fitted, family by family, to a sweep of every tile over M
 * = 64..4096 and N x K from 1536 x 1536 to 12288 x 4096 and 4096 x 12288
 * (backward products: 19 shapes each) on 256 CUs; the tile picked by them took
 * 1.5-3% longer than the best one on average, 25% at most. Tiles of at most 80
 * KB of LDS run two to a CU: deeper rings against a second workgroup to hide
 * the first's waits is why some shapes are there twice. Every tile listed is
 * the pick of some shapes among 12000 drawn log-uniformly from 1 to 16384.
 */
#ifndef K_FFN_TILE_H
#define K_FFN_TILE_H

#include "k_ffn_gemm.h"

/* LDS of bm rows of A and bst bytes a stage of B, L stages ahead */
static constexpr uint32_t fg_ring(uint32_t bm, uint32_t bst, uint32_t L) {
    return (L + 1u) * bm * 128u + L * bst;
}

template <int MODE, int W8, int AL, int BL, int WM, int RB, int CB, int L>
static void fg_run(const GhipProd *p, const GhipEp *ep, uint32_t mt, uint32_t nt, uint32_t lds,
                   hipStream_t st) {
    hipLaunchKernelGGL((k_ffn_gemm<MODE, W8, AL, BL, WM, RB, CB, L>),
                       dim3(mt * nt * p->splits * (p->batch ? 2u : 1u)), dim3(256), lds, st, *p,
                       *ep, mt, nt);
}

template <int MODE, int W8, int AL, int BL, int WM, int RB, int CB, int L>
static constexpr GhipFfnTile fg_tile(float low, float mid, float full, float over) {
    constexpr uint32_t bm = 16u * RB * WM, bn = 16u * CB * (4 / WM);
    constexpr uint32_t lds = fg_ring(bm, bn * (W8 ? 64u : 128u), L);
    return {bm, ghip_ep_dual(MODE) ? bn / 2 : bn, lds <= FG_LDS_MAX / 2 ? 2u : 1u, low, mid, full, over, lds,
            (const void *)k_ffn_gemm<MODE, W8, AL, BL, WM, RB, CB, L>,
            fg_run<MODE, W8, AL, BL, WM, RB, CB, L>};
}

#endif /* K_FFN_TILE_H */
