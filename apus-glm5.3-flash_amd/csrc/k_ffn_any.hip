/*
 * k_ffn_any.hip — the dense feed-forward products of any shape, stride and
 * alignment on MFMA (gfx950):
 *
 *   out[m, n] = epilogue(sum_p sum_k A_p(m, k) * B_p(n, k))
 *
 * with A_p(m, k) at a[m * ars + k * aks] and B_p(n, k) at b[n * brs + k * bks]
 * (bf16, or FP8 codes with an F32 scale a 128x128 block of (n, k)), one of the
 * two steps 1. That covers the forward (A = x, B = W: k the fast index of
 * both), dx = dz W (k the slow index of B; two pairs for the gated block) and
 * dW = dz^T x (k the slow index of both). In the dual modes the second B gives
 * a second sum of the same A.
 *
 * A workgroup of 4 waves owns 64 x 64 outputs, each wave 32 x 32 as four
 * v_mfma_f32_16x16x32_bf16 a step of k = 32; tiles reach LDS through registers
 * by loads of 8 elements at any alignment (8 of one element at the matrix's
 * edges), the next step's in flight during the products, elements past M, N or
 * k as zeros. It is bound by the two barriers of a step and its load's latency,
 * 0.8 us a step: the route for what the kernels with direct loads cannot take
 * (linear with SiLU, BF16, odd K: 1 x 4096 x 4095 106 us, 64 x 2000 x 2001 40, 1111
 * x 2048 x 4095 116, 4096 x 4096 x 4095 453, 300 TFLOP/s; FP8 97 to 130% of
 * that).
 */
#include "ghip_epilogue.h"
#include "k_ffn_colsum.h"

#define FA_LD 40u                                /* LDS row: 32 values, 80 bytes */

typedef unsigned short fa_u16x8 __attribute__((ext_vector_type(8)));

template <int MODE, bool FP8>
__global__ __launch_bounds__(256) void k_ffn_any(GhipProd p, GhipEp ep, uint32_t blk0) {
    constexpr int NB = ghip_ep_dual(MODE) ? 2 : 1;
    __shared__ __attribute__((aligned(16))) uint16_t as[64 * FA_LD], bs[NB][64 * FA_LD];
    const uint32_t tid = threadIdx.x, lane = tid & 63u, wv = tid >> 6;
    const uint32_t n16 = lane & 15u, g = lane >> 4;
    const uint32_t mt = (p.M + 63u) / 64u, t = blk0 + blockIdx.x;
    const uint32_t row0 = (t % mt) * 64u, col0 = (t / mt) * 64u;
    const uint32_t rw = (wv >> 1) * 32u, cw = (wv & 1u) * 32u;
    ghip_f32x4 acc[NB][2][2] = {};
    const uint32_t nkb = (p.K + 127u) >> 7;

    /* A thread loads 8 elements along the operand's fast index: k 8 (tid % 4) ..
     * of row tid / 4, or rows 8 (tid % 8) .. of k tid / 8. Where all 8 exist that
     * is one load at whatever alignment the row has, else one each */
    auto spot = [&](bool kfast, uint32_t &r, uint32_t &k) {
        r = kfast ? tid >> 2 : 8u * (tid & 7u);
        k = kfast ? 8u * (tid & 3u) : tid >> 3;
    };
    auto load8 = [&](const uint16_t *q, bool whole, uint32_t live, fa_u16x8 &v) {
        if (whole) {
            __builtin_memcpy(&v, q, 16);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) v[e] = e < live ? q[e] : (uint16_t)0;
        }
    };
    fa_u16x8 ra, rb[NB];
    auto fetch = [&](int pr, uint32_t k0) {
        uint32_t r, k;
        spot(p.aks == 1, r, k);
        {
            const uint32_t m = row0 + r, kk = k0 + k;
            const uint32_t left = p.aks == 1 ? (kk < p.K ? p.K - kk : 0u) : (m < p.M ? p.M - m : 0u);
            const bool in = m < p.M && kk < p.K;
            const uint16_t *q = (pr ? p.a2 : p.a) + (in ? (size_t)m * p.ars + (size_t)kk * p.aks : 0);
            load8(q, in && left >= 8u, in ? left : 0u, ra);
        }
        spot(p.bks == 1, r, k);
        const uint32_t n = col0 + r, kk = k0 + k;
        const uint32_t left = p.bks == 1 ? (kk < p.K ? p.K - kk : 0u) : (n < p.N ? p.N - n : 0u);
        const bool in = n < p.N && kk < p.K;
        const size_t o = in ? (size_t)n * p.brs + (size_t)kk * p.bks : 0;
#pragma unroll
        for (int d = 0; d < NB; d++) {
            const void *b = d || pr ? p.b2 : p.b;
            if constexpr (FP8) {
                uint64_t c = 0;
                const uint8_t *q = (const uint8_t *)b + o;
                if (in && left >= 8u) {
                    __builtin_memcpy(&c, q, 8);
                } else if (in) {
                    for (uint32_t e = 0; e < left; e++) c |= (uint64_t)q[e] << (8u * e);
                }
                const float sc = in ? (d ? p.s2 : p.s)[(size_t)(n >> 7) * nkb + (kk >> 7)] : 0.0f;
                const ghip_u32x2 lo = ghip_deq4<true>((uint32_t)c, sc), hi = ghip_deq4<true>((uint32_t)(c >> 32), sc);
                const ghip_u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
                rb[d] = __builtin_bit_cast(fa_u16x8, v);
                if (in && left < 8u) {                   /* codes past K: 0, not 0 * scale */
#pragma unroll
                    for (uint32_t e = 0; e < 8; e++) rb[d][e] = e < left ? rb[d][e] : (uint16_t)0;
                }
            } else {
                load8((const uint16_t *)b + o, in && left >= 8u, in ? left : 0u, rb[d]);
            }
        }
    };
    auto put = [&](uint16_t *to, bool kfast, const fa_u16x8 &v) {
        uint32_t r, k;
        spot(kfast, r, k);
        if (kfast) {
            *(fa_u16x8 *)(to + r * FA_LD + k) = v;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) to[(r + e) * FA_LD + k] = v[e];
        }
    };
    const int pairs = p.a2 ? 2 : 1;
    const uint32_t steps = (p.K + 31u) / 32u, total = steps * (uint32_t)pairs;
    fetch(0, 0);
    for (uint32_t j = 0; j < total; j++) {
        __syncthreads();
        put(as, p.aks == 1, ra);
#pragma unroll
        for (int d = 0; d < NB; d++) put(bs[d], p.bks == 1, rb[d]);
        __syncthreads();
        if (j + 1u < total) fetch((int)((j + 1u) / steps), ((j + 1u) % steps) * 32u);
        ghip_bf16x8 av[2];
#pragma unroll
        for (uint32_t i = 0; i < 2; i++)
            av[i] = *(const ghip_bf16x8 *)(as + (rw + 16u * i + n16) * FA_LD + 8u * g);
#pragma unroll
        for (int d = 0; d < NB; d++)
#pragma unroll
            for (uint32_t c = 0; c < 2; c++) {
                const ghip_bf16x8 bv =
                    *(const ghip_bf16x8 *)(bs[d] + (cw + 16u * c + n16) * FA_LD + 8u * g);
#pragma unroll
                for (uint32_t i = 0; i < 2; i++)
                    acc[d][i][c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(av[i], bv, acc[d][i][c],
                                                                          0, 0, 0);
            }
    }
    /* register q of block (i, c): row 16 i + 4 g + q, column 16 c + n16 */
    ghip_with_act(ep.act, [&](auto act) {
#pragma unroll
        for (uint32_t i = 0; i < 2; i++)
#pragma unroll
            for (uint32_t c = 0; c < 2; c++)
#pragma unroll
                for (uint32_t q = 0; q < 4; q++) {
                    const uint32_t m = row0 + rw + 16u * i + 4u * g + q, n = col0 + cw + 16u * c + n16;
                    if (ep.pad && m < p.M && n >= p.N && n < ((p.N + 7u) & ~7u)) {
                        ep.out[(size_t)m * ep.ldout + n] = 0;
                        if (MODE == GHIP_EP_DGATED) ep.out2[(size_t)m * ep.ldout + n] = 0;
                    }
                    if (m < p.M && n < p.N)
                        ghip_ep_store<MODE, decltype(act)::value>(ep, ep.out, m, n, acc[0][i][c][q],
                                                                  acc[NB - 1][i][c][q]);
                }
    });
}

/* dbias. Bound by latency: with the launch, 300 x 2048 2.8 us, 4096 x 2048 10.9 (64
 * columns a workgroup: 14; 16: 13.8). */
#define FA_SUM 32u                               /* columns of a workgroup */
__global__ __launch_bounds__(1024) void k_ffn_colsum(GhipFfnSum p) {
    __shared__ float sum[8 * 1024 / FA_SUM][FA_SUM + 1];
    fc_colsum<1024, FA_SUM>(p, blockIdx.x, sum);
}

/* dst[m, 0 .. N up to a multiple of 8) = src[m, 0 .. N), zeros behind: rows of any
 * alignment as whole vectors. */
__global__ __launch_bounds__(256) void k_ffn_pack(const uint16_t *__restrict__ src, size_t ld,
                                                  uint32_t M, uint32_t N, uint32_t per,
                                                  uint16_t *__restrict__ dst) {
    for (size_t v = (size_t)blockIdx.x * 256u + threadIdx.x; v < (size_t)M * per;
         v += (size_t)gridDim.x * 256u) {
        const size_t m = v / per;
        const uint32_t n = (uint32_t)(v % per) * 8u;
        const uint16_t *q = src + m * ld + n;
        fa_u16x8 d;
        if (n + 8u <= N) {
            __builtin_memcpy(&d, q, 16);
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 8; e++) d[e] = n + e < N ? q[e] : (uint16_t)0;
        }
        *(fa_u16x8 *)(dst + v * 8u) = d;
    }
}

template <int MODE, bool FP8>
static hipError_t fa_run(const GhipProd *p, const GhipEp *ep, hipStream_t st) {
    const size_t tiles = (((size_t)p->M + 63) / 64) * (((size_t)p->N + 63) / 64);
    const size_t most = GHIP_MAX_THREADS / 256u;
    if (tiles > 0xffffffffu) return hipErrorInvalidValue;
    for (size_t b = 0; b < tiles; b += most) {
        const size_t n = tiles - b < most ? tiles - b : most;
        hipLaunchKernelGGL((k_ffn_any<MODE, FP8>), dim3((uint32_t)n), dim3(256), 0, st, *p, *ep,
                           (uint32_t)b);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

extern "C" hipError_t ghip_launch_ffn_any(int mode, const GhipProd *p, const GhipEp *ep,
                                          hipStream_t st) {
    if (p->M == 0 || p->N == 0 || p->K == 0) return hipErrorInvalidValue;
    if (p->batch) {
        GhipProd one = *p, two = *p;
        GhipEp to = *ep;
        one.batch = two.batch = 0;
        two.a = p->a2;
        two.b = p->b2;
        one.a2 = two.a2 = nullptr;
        one.b2 = two.b2 = nullptr;
        to.out = ep->out2;
        const hipError_t e = ghip_launch_ffn_any(mode, &one, ep, st);
        return e == hipSuccess ? ghip_launch_ffn_any(mode, &two, &to, st) : e;
    }
    const bool fp8 = p->s != nullptr;
    switch (mode) {
    case GHIP_EP_STORE: return fp8 ? hipErrorInvalidValue : fa_run<GHIP_EP_STORE, false>(p, ep, st);
    case GHIP_EP_LINEAR:
        return fp8 ? fa_run<GHIP_EP_LINEAR, true>(p, ep, st) : fa_run<GHIP_EP_LINEAR, false>(p, ep, st);
    case GHIP_EP_GATED:
        return fp8 ? fa_run<GHIP_EP_GATED, true>(p, ep, st) : fa_run<GHIP_EP_GATED, false>(p, ep, st);
    case GHIP_EP_DLINEAR: return fp8 ? hipErrorInvalidValue : fa_run<GHIP_EP_DLINEAR, false>(p, ep, st);
    case GHIP_EP_DGATED: return fp8 ? hipErrorInvalidValue : fa_run<GHIP_EP_DGATED, false>(p, ep, st);
    default: return hipErrorInvalidValue;
    }
}

extern "C" hipError_t ghip_launch_ffn_colsum(const GhipFfnSum *p, hipStream_t st) {
    if (p->M == 0 || p->N == 0 || p->M > 0x7fffffffu || p->N > 0x7fffffffu) return hipErrorInvalidValue;
    const size_t most = GHIP_MAX_THREADS / 1024u * FA_SUM;   /* columns of a launch */
    for (size_t n0 = 0; n0 < p->N; n0 += most) {
        GhipFfnSum q = *p;
        q.dz += n0;
        q.out += n0;
        q.N = p->N - n0 < most ? p->N - n0 : most;
        hipLaunchKernelGGL(k_ffn_colsum, dim3((uint32_t)((q.N + FA_SUM - 1) / FA_SUM)), dim3(1024), 0, st, q);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

extern "C" hipError_t ghip_launch_ffn_pack(const uint16_t *src, size_t ld, size_t M, size_t N,
                                           uint16_t *dst, hipStream_t st) {
    if (M == 0 || N == 0 || M > 0x7fffffffu || N > 0x7fffffffu || ((uintptr_t)dst & 15u))
        return hipErrorInvalidValue;
    const size_t per = (N + 7) / 8, blocks = (M * per + 255) / 256;
    hipLaunchKernelGGL(k_ffn_pack, dim3((uint32_t)(blocks < 16384 ? blocks : 16384)), dim3(256), 0, st,
                       src, ld, (uint32_t)M, (uint32_t)N, (uint32_t)per, dst);
    return hipGetLastError();
}
