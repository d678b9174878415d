/*
 * k_ffn.hip — which kernel a dense feed-forward product takes (gfx950).
 */
#include "ghip_epilogue.h"

extern "C" hipError_t ghip_launch_ffn(int mode, const GhipProd *p, const GhipEp *ep,
                                      hipStream_t st) {
    return ghip_launch_ffn_any(mode, p, ep, st);
}
