/*
 * k_ffn_grads.hip — dx, dW and dbias of one backward pass in one launch (gfx950).
 *
 * The three need dz and not each other. Where their tiles are small, each by
 * itself fills a part of the chip for as long as its k takes and costs a launch;
 * together they take the time of the longest and one launch. A workgroup does
 * one piece: 64 columns of dbias, or a tile of dx or dW as k_ffn_gemm.h computes
 * it alone. The product with the longer k comes first, so that the shorter one's
 * tiles fill its last round. Bound by that longest workgroup's chain of stages
 * below a full chip, by LDS and the loads above (linear backward 300 x 2048 x 1536
 * with GELU and dbias, dz included: 32.0 us apart, 23.4 together, 22.3 since dz takes
 * less; 138 x 1008 x 712 11.8 and 8.5, the host's time for a call).
 */
#include "k_ffn_colsum.h"
#include "k_ffn_tile.h"

typedef struct {
    uint32_t mtx, ntx, nx, mtw, ntw, nw, ns, dx_first;
} FgGrads;

template <int RB, int CB, int L, int RBX, int CBX, int LX>
__global__ __launch_bounds__(256, 2) void k_ffn_grads(GhipProd dx, GhipEp edx, GhipProd dw,
                                                      GhipEp edw, GhipFfnSum sum, FgGrads gr) {
    extern __shared__ __attribute__((aligned(1024))) uint8_t fg_lds[];
    uint32_t b = blockIdx.x;
    if (b < gr.ns) {
        fc_colsum<256, 64>(sum, b, (float (*)[65])fg_lds);
        return;
    }
    b -= gr.ns;
    const uint32_t head = gr.dx_first ? gr.nx : gr.nw;
    if ((b < head) == (gr.dx_first != 0u))
        fg_product<GHIP_EP_STORE, 0, 0, 1, 2, RBX, CBX, LX>(dx, edx, gr.mtx, gr.ntx,
                                                            gr.dx_first ? b : b - head, gr.nx);
    else
        fg_product<GHIP_EP_STORE, 0, 1, 1, 2, RB, CB, L>(dw, edw, gr.mtw, gr.ntw,
                                                         gr.dx_first ? b - head : b, gr.nw);
}

template <int RB, int CB, int L, int RBX, int CBX, int LX>
static void fg_grads(const GhipProd *dx, const GhipEp *edx, const GhipProd *dw, const GhipEp *edw,
                     const GhipFfnSum *sum, const GhipFfnTile *tx, const GhipFfnTile *tw,
                     hipStream_t st) {
    FgGrads g;
    g.mtx = (dx->M + tx->bm - 1) / tx->bm;
    g.ntx = (dx->N + tx->bn - 1) / tx->bn;
    g.nx = g.mtx * g.ntx * dx->splits;
    g.mtw = (dw->M + tw->bm - 1) / tw->bm;
    g.ntw = (dw->N + tw->bn - 1) / tw->bn;
    g.nw = g.mtw * g.ntw * dw->splits * (dw->batch ? 2u : 1u);
    g.ns = sum ? (uint32_t)((sum->N + 63) / 64) : 0u;
    g.dx_first = (uint64_t)dx->K * (dx->a2 ? 2u : 1u) / dx->splits >= dw->K / dw->splits;
    const GhipFfnSum none = {};
    hipLaunchKernelGGL((k_ffn_grads<RB, CB, L, RBX, CBX, LX>), dim3(g.nx + g.nw + g.ns), dim3(256),
                       tx->lds > tw->lds ? tx->lds : tw->lds, st, *dx, *edx, *dw, *edw,
                       sum ? *sum : none, g);
}

/* A pair of dW's tile and dx's: those that run two workgroups a CU, whose second
 * one hides what a deeper ring would. */
#define FG_PAIR(RB, CB, L, RBX, CBX, LX)                                                       \
    {{32u * RBX, 32u * CBX, fg_ring(32u * RBX, 32u * CBX * 128u, LX)},                          \
     {32u * RB, 32u * CB, fg_ring(32u * RB, 32u * CB * 128u, L)},                               \
     (const void *)k_ffn_grads<RB, CB, L, RBX, CBX, LX>, fg_grads<RB, CB, L, RBX, CBX, LX>}

extern "C" const GhipFfnPair *ghip_ffn_pairs(int *n) {
    static const GhipFfnPair t[] = {
        FG_PAIR(2, 2, 3, 2, 2, 3),
        FG_PAIR(4, 4, 2, 2, 2, 3),
        FG_PAIR(2, 2, 3, 4, 4, 2),
        FG_PAIR(4, 4, 2, 4, 4, 2),
    };
    *n = sizeof t / sizeof *t;
    return t;
}
