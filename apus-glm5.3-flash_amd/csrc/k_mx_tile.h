/*
 * k_mx_tile.h — an entry of a tile table (GhipMxTile) over k_mx_gemm.
 */
#ifndef K_MX_TILE_H
#define K_MX_TILE_H

#include "k_mx_gemm.h"

template <int MODE, int XT, int WM, int WN, int RB, int CB, int R>
static void mg_run(const GhipMxProd *p, const GhipEp *ep, uint32_t mt, uint32_t nt, hipStream_t st) {
    using T = MgTile<MODE, XT, WM, WN, RB, CB, R>;
    hipLaunchKernelGGL((k_mx_gemm<MODE, XT, WM, WN, RB, CB, R>), dim3(mt * nt), dim3(64 * WM * WN), T::LDS, st,
                       *p, *ep, mt, nt);
}

/* A mode's microseconds (GhipMxTile). */
struct MgTimes {
    float low, mid, full, over;
};
template <int MODE, int XT, int WM, int WN, int RB, int CB, int R>
static constexpr GhipMxTile mg_tile(MgTimes linear, MgTimes gated) {
    using T = MgTile<MODE, XT, WM, WN, RB, CB, R>;
    const MgTimes us = MODE == GHIP_EP_GATED ? gated : linear;
    /* two fit a CU by LDS, and by registers where the sums take 64 or fewer */
    return {T::BM, T::OUTN, T::LDS <= FG_LDS_MAX / 2 && RB * CB < 32 ? 2u : 1u, T::LDS, us.low, us.mid, us.full, us.over,
            (const void *)k_mx_gemm<MODE, XT, WM, WN, RB, CB, R>, mg_run<MODE, XT, WM, WN, RB, CB, R>};
}

#endif /* K_MX_TILE_H */
