/*
 * ghip_epilogue.h — what the dense feed-forward kernels do with a finished
 * f32 sum before it leaves the registers (k_ffn*.hip):
 *
 *   GHIP_EP_STORE   y = z                                     (gradients)
 *   GHIP_EP_LINEAR  y = act(z + b) + r
 *   GHIP_EP_GATED   h = act(min(g, limit)) * clamp(u, -limit, limit)
 *   GHIP_EP_DLINEAR dz = dy * act'(z + b)
 *   GHIP_EP_DGATED  dg = dh * clamp(u) * act'(min(g, limit)), 0 where g > limit
 *                   du = dh * act(min(g, limit)), 0 where |u| > limit
 *
 * All of it in f32, with one rounding to bf16 (nearest even) at the store: the
 * sums are f32, so bias, activation, clamp, product and residual cost no
 * precision. dz, dg and du are rounded because the products that read them
 * take bf16 operands.
 *
 * exp comes from the hardware exp2 and 1/x from the hardware reciprocal, each
 * about 1 ulp of f32; an argument v of exp is itself rounded a few times, which
 * adds up to 8 |v| 2^-24 relative (|v| is under 88 where the result is not 0):
 * at most 2^-14 against the output's half step of 2^-8, for values far left of 0
 * as for all others. An argument whose exp is above 2^126 makes the sigmoid 0,
 * so values of 1 + |z| times 2^-126 and less are lost.
 */
#ifndef GHIP_EPILOGUE_H
#define GHIP_EPILOGUE_H

#include <type_traits>

#include "ghip_device.h"
#include "ghip_internal.h"

#define GHIP_GELU_C 0.7978845608028654f          /* sqrt(2 / pi) */
#define GHIP_GELU_A 0.044715f

__device__ __forceinline__ float ghip_sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __expf(-z));
}

/* Phi(z) = (1 + erf(z / sqrt 2)) / 2, and e = exp(-z^2 / 2). The sum cancels left
 * of 0 (4% off at z = -5, 0 below -5.6); so Phi(-|z|) = e R(|z|), where R (the
 * Mills ratio over sqrt(2 pi)) falls like 1 / |z| and is t times a polynomial of
 * t = 1 / (1 + 0.326 |z|): the minimax one of degree 7, 2^-20 relative for every
 * z. Its exp serves the slope too, and it takes no branch: 4096 x 4096 x 1024
 * with GELU 42 us, 56 with the library's erfc (53 with its erf). */
__device__ __forceinline__ float ghip_phi(float z, float &e) {
    const float u = __builtin_fabsf(z);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(0.326f, u, 1.0f));
    float q = 0.0337685977f;
    q = __builtin_fmaf(q, t, -0.112105614f);
    q = __builtin_fmaf(q, t, 0.0818245333f);
    q = __builtin_fmaf(q, t, 0.0275429578f);
    q = __builtin_fmaf(q, t, 0.0929912787f);
    q = __builtin_fmaf(q, t, 0.115857593f);
    q = __builtin_fmaf(q, t, 0.130065828f);
    q = __builtin_fmaf(q, t, 0.130055185f);
    e = __expf(-0.5f * z * z);
    const float low = e * t * q;
    return z < 0.0f ? low : 1.0f - low;
}

template <int ACT>
__device__ __forceinline__ float ghip_act(float z) {
    [[maybe_unused]] float e;
    if constexpr (ACT == GHIP_ACT_RELU) return z < 0.0f ? 0.0f : z;      /* keeps a NaN */
    else if constexpr (ACT == GHIP_ACT_SILU) return z * ghip_sigmoid(z);
    else if constexpr (ACT == GHIP_ACT_GELU) return z * ghip_phi(z, e);
    else if constexpr (ACT == GHIP_ACT_GELU_TANH)
        /* (1 + tanh v) / 2 = sigmoid(2 v) */
        return z * ghip_sigmoid(2.0f * GHIP_GELU_C * (z + GHIP_GELU_A * z * z * z));
    else return z;
}

/* The derivative (ReLU's: ghip_pull). The smooth ones are 0 or 1 to the last bit
 * well inside +-100 (+-20), and the clamp keeps an infinite z from making 0 * inf
 * of that. */
template <int ACT>
__device__ __forceinline__ float ghip_slope(float z) {
    if constexpr (ACT == GHIP_ACT_SILU) {
        z = z > 100.0f ? 100.0f : z < -100.0f ? -100.0f : z;
        const float s = ghip_sigmoid(z);
        return s * (1.0f + z * (1.0f - s));
    } else if constexpr (ACT == GHIP_ACT_GELU) {
        z = z > 20.0f ? 20.0f : z < -20.0f ? -20.0f : z;
        float e;
        const float phi = ghip_phi(z, e);
        return phi + z * e * 0.3989422804014327f;
    } else if constexpr (ACT == GHIP_ACT_GELU_TANH) {
        z = z > 20.0f ? 20.0f : z < -20.0f ? -20.0f : z;
        const float s = ghip_sigmoid(2.0f * GHIP_GELU_C * (z + GHIP_GELU_A * z * z * z));
        return s + z * s * (1.0f - s) * 2.0f * GHIP_GELU_C * (1.0f + 3.0f * GHIP_GELU_A * z * z);
    } else {
        return 1.0f;
    }
}

/* d * act'(z). ReLU selects, as the clamps do: nothing passes where z <= 0, not
 * 0 * inf either, and a NaN z stays one. */
template <int ACT>
__device__ __forceinline__ float ghip_pull(float z, float d) {
    if constexpr (ACT == GHIP_ACT_RELU) return z > 0.0f ? d : z <= 0.0f ? 0.0f : z;
    else return d * ghip_slope<ACT>(z);
}

/* The value(s) that leave the registers: s0 the sum (g), s1 the second one (u),
 * b the bias, in the residual or the incoming gradient. */
template <int MODE, int ACT>
__device__ __forceinline__ void ghip_ep_value(float s0, float s1, float b, float in, float limit,
                                              float &o0, float &o1) {
    o1 = 0.0f;
    if constexpr (MODE == GHIP_EP_STORE) {
        o0 = s0;
    } else if constexpr (MODE == GHIP_EP_LINEAR) {
        o0 = ghip_act<ACT>(s0 + b) + in;
    } else if constexpr (MODE == GHIP_EP_DLINEAR) {
        o0 = ghip_pull<ACT>(s0 + b, in);
    } else {
        const float g = s0 > limit ? limit : s0;             /* keep a NaN */
        const float u = s1 > limit ? limit : s1 < -limit ? -limit : s1;
        if constexpr (MODE == GHIP_EP_GATED) {
            o0 = ghip_act<ACT>(g) * u;
        } else {
            o0 = s0 > limit ? 0.0f : ghip_pull<ACT>(g, in * u);
            o1 = s1 > limit || s1 < -limit ? 0.0f : in * ghip_act<ACT>(g);
        }
    }
}

/* Run f with the activation as a constant (wave-uniform branch). */
template <typename F>
__device__ __forceinline__ void ghip_with_act(int act, F f) {
    switch (act) {
    case GHIP_ACT_RELU: f(std::integral_constant<int, GHIP_ACT_RELU>{}); break;
    case GHIP_ACT_SILU: f(std::integral_constant<int, GHIP_ACT_SILU>{}); break;
    case GHIP_ACT_GELU: f(std::integral_constant<int, GHIP_ACT_GELU>{}); break;
    case GHIP_ACT_GELU_TANH: f(std::integral_constant<int, GHIP_ACT_GELU_TANH>{}); break;
    default: f(std::integral_constant<int, GHIP_ACT_NONE>{}); break;
    }
}

/* Modes with two sums a column (the gate's and the up projection's). */
constexpr bool ghip_ep_dual(int mode) { return mode == GHIP_EP_GATED || mode == GHIP_EP_DGATED; }

/* One output, row m, column n, from its sums, bias and incoming value. */
template <int MODE, int ACT>
__device__ __forceinline__ void ghip_ep_put(const GhipEp &ep, uint16_t *out, uint32_t m, uint32_t n,
                                            float s0, float s1, float b, float in) {
    float o0, o1;
    ghip_ep_value<MODE, ACT>(s0, s1, b, in, ep.limit, o0, o1);
    out[(size_t)m * ep.ldout + n] = (uint16_t)ghip_bf16_bits(o0);
    if constexpr (MODE == GHIP_EP_DGATED)
        ep.out2[(size_t)m * ep.ldout + n] = (uint16_t)ghip_bf16_bits(o1);
}

template <int MODE, int ACT>
__device__ __forceinline__ void ghip_ep_store(const GhipEp &ep, uint16_t *out, uint32_t m,
                                              uint32_t n, float s0, float s1) {
    const float b = ep.bias ? ghip_bf16_f32(ep.bias[n]) : 0.0f;
    const float in = ep.in ? ghip_bf16_f32(ep.in[(size_t)m * ep.ldin + n]) : 0.0f;
    ghip_ep_put<MODE, ACT>(ep, out, m, n, s0, s1, b, in);
}

#endif /* GHIP_EPILOGUE_H */
