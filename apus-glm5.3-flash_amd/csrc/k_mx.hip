/*
 * k_mx.hip — microscaled quantization and back (gfx950). Bound by HBM: 2 bytes a
 * value in (out) and 33/32 (MXFP8) or 17/32 (MXFP4) out (in). A lane takes 8
 * values, one 16-byte access of the BF16 side, and a quad of lanes a block, whose
 * maximum takes two DPP steps; nothing goes through LDS. Four pieces a thread, all
 * loaded before the first is used.
 *
 * Measured: 12288 x 4096 to MXFP4 26.8 us and back 19.8 (127 MB each way: 4.8 and 6.4
 * TB/s), 1111 x 2048 to MXFP8 3.9 (a launch's time).
 */
#include "ghip_mx.h"

#define MX_PER 4u                                /* 8-value pieces a thread */

/* Piece v of this launch: its row and first column. */
struct MxPlace {
    size_t row;
    uint32_t col;
};
__device__ __forceinline__ MxPlace mx_place(uint32_t v, uint32_t per) {
    const uint32_t r = v / per;
    return {r, 8u * (v - r * per)};
}

template <int TYPE>
__global__ __launch_bounds__(256) void k_mx_quantize(const uint16_t *__restrict__ x,
                                                     uint8_t *__restrict__ codes,
                                                     uint8_t *__restrict__ scales, uint32_t pieces,
                                                     uint32_t K, size_t ldx, uint32_t lds) {
    const uint32_t per = K / 8u, v0 = blockIdx.x * (256u * MX_PER) + threadIdx.x;
    ghip_u32x4 d[MX_PER];
    MxPlace at[MX_PER];
#pragma unroll
    for (uint32_t i = 0; i < MX_PER; i++) {
        const uint32_t v = v0 + 256u * i;
        if (v < pieces) {
            at[i] = mx_place(v, per);
            __builtin_memcpy(&d[i], x + at[i].row * ldx + at[i].col, 16);
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < MX_PER; i++) {
        if (v0 + 256u * i >= pieces) break;      /* whole quads: K % 32 == 0 */
        float f[8];
#pragma unroll
        for (int e = 0; e < 8; e++)
            f[e] = ghip_bf16_f32(e & 1 ? d[i][e >> 1] >> 16 : d[i][e >> 1] & 0xffffu);
        const uint32_t s = mx_scale<TYPE>(mx_quad_max(mx_amax8(f)));
        const ghip_u32x2 c = mx_codes8<TYPE>(f, s);
        uint8_t *out = codes + (at[i].row * K + at[i].col) / (TYPE == GHIP_MXFP8 ? 1u : 2u);
        if (TYPE == GHIP_MXFP8) *(ghip_u32x2 *)out = c;
        else *(uint32_t *)out = c[0];
        if ((threadIdx.x & 3u) == 0u) {
            uint8_t *row = scales + at[i].row * lds;
            const uint32_t b = at[i].col >> 5;
            row[b] = (uint8_t)s;
            if (b == K / 32u - 1u)               /* the row's last word is whole */
                for (uint32_t j = b + 1u; j < lds; j++) row[j] = 0;
        }
    }
}

template <int TYPE>
__global__ __launch_bounds__(256) void k_mx_dequant(const uint8_t *__restrict__ codes,
                                                    const uint8_t *__restrict__ scales,
                                                    uint16_t *__restrict__ out, uint32_t pieces,
                                                    uint32_t K, size_t ldo, uint32_t lds) {
    const uint32_t per = K / 8u, v0 = blockIdx.x * (256u * MX_PER) + threadIdx.x;
    ghip_u32x2 c[MX_PER];
    uint32_t s[MX_PER];
    MxPlace at[MX_PER];
#pragma unroll
    for (uint32_t i = 0; i < MX_PER; i++) {
        const uint32_t v = v0 + 256u * i;
        if (v < pieces) {
            at[i] = mx_place(v, per);
            const uint8_t *p = codes + (at[i].row * K + at[i].col) / (TYPE == GHIP_MXFP8 ? 1u : 2u);
            if (TYPE == GHIP_MXFP8) c[i] = *(const ghip_u32x2 *)p;
            else c[i][0] = *(const uint32_t *)p;
            s[i] = scales[at[i].row * lds + (at[i].col >> 5)];
        }
    }
#pragma unroll
    for (uint32_t i = 0; i < MX_PER; i++) {
        if (v0 + 256u * i >= pieces) break;
        const float f = mx_scale_f32(s[i]);
        const ghip_u32x4 o = TYPE == GHIP_MXFP8 ? mx_fp8_bf16(c[i], f) : mx_fp4_bf16(c[i][0], f);
        __builtin_memcpy(out + at[i].row * ldo + at[i].col, &o, 16);
    }
}

/* Launches of whole rows with fewer than 2^30 pieces (their numbers are of 32 bits). */
template <typename F>
static hipError_t in_rows(size_t R, size_t K, F launch) {
    const size_t per = K / 8;
    if (R == 0 || per == 0 || K % 32 || per >= ((size_t)1 << 30)) return hipErrorInvalidValue;
    const size_t most = (((size_t)1 << 30) - 1) / per;
    for (size_t r = 0; r < R; r += most) {
        const uint32_t pieces = (uint32_t)((R - r < most ? R - r : most) * per);
        launch(r, pieces, dim3((pieces + 256u * MX_PER - 1u) / (256u * MX_PER)));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

extern "C" size_t ghip_mx_scale_ld(size_t K) { return (K + 127) / 128 * 4; }

extern "C" hipError_t ghip_launch_mx_quantize(int type, const uint16_t *x, uint8_t *codes,
                                              uint8_t *scales, size_t R, size_t K, size_t ldx,
                                              hipStream_t st) {
    const size_t lds = ghip_mx_scale_ld(K);
    return in_rows(R, K, [&](size_t r, uint32_t pieces, dim3 grid) {
        if (type == GHIP_MXFP8)
            hipLaunchKernelGGL((k_mx_quantize<GHIP_MXFP8>), grid, dim3(256), 0, st, x + r * ldx,
                               codes + r * K, scales + r * lds, pieces, (uint32_t)K, ldx, (uint32_t)lds);
        else
            hipLaunchKernelGGL((k_mx_quantize<GHIP_MXFP4>), grid, dim3(256), 0, st, x + r * ldx,
                               codes + r * K / 2, scales + r * lds, pieces, (uint32_t)K, ldx, (uint32_t)lds);
    });
}

extern "C" hipError_t ghip_launch_mx_dequant(int type, const uint8_t *codes, const uint8_t *scales,
                                             uint16_t *out, size_t R, size_t K, size_t ldo,
                                             hipStream_t st) {
    const size_t lds = ghip_mx_scale_ld(K);
    return in_rows(R, K, [&](size_t r, uint32_t pieces, dim3 grid) {
        if (type == GHIP_MXFP8)
            hipLaunchKernelGGL((k_mx_dequant<GHIP_MXFP8>), grid, dim3(256), 0, st, codes + r * K,
                               scales + r * lds, out + r * ldo, pieces, (uint32_t)K, ldo, (uint32_t)lds);
        else
            hipLaunchKernelGGL((k_mx_dequant<GHIP_MXFP4>), grid, dim3(256), 0, st, codes + r * K / 2,
                               scales + r * lds, out + r * ldo, pieces, (uint32_t)K, ldo, (uint32_t)lds);
    });
}
