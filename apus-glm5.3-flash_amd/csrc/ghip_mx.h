/*
 * ghip_mx.h — microscaled values on gfx950: 32 values along k share an E8M0 scale
 * (the byte b stands for 2^(b - 127), 255 for NaN), the values are E4M3 (MXFP8, a
 * byte each, 0x7F and 0xFF NaN) or E2M1 (MXFP4, two a byte, the lower nibble
 * first). A row of scales is ceil(K / 128) words.
 *
 * The scale of a block is the smallest power of two at which its largest value is
 * not past the type's largest (448 = 1.75 * 2^8, 6 = 1.5 * 2^2): nothing
 * saturates, and where rounding moves a block's maximum across a step the values
 * stay the same up to the type's subnormals. Truncating the exponent instead
 * clips up to a quarter of a block's largest value.
 */
#ifndef GHIP_MX_H
#define GHIP_MX_H

#include "ghip_device.h"
#include "ghip_internal.h"

typedef __bf16 mx_bf16x2 __attribute__((ext_vector_type(2)));

/* The scale byte of a block whose largest |value| has these f32 bits. */
template <int TYPE>
__device__ __forceinline__ uint32_t mx_scale(uint32_t amax) {
    constexpr uint32_t BIAS = TYPE == GHIP_MXFP8 ? 8u : 2u, TOP = TYPE == GHIP_MXFP8 ? 0x600000u : 0x400000u;
    const uint32_t e = (amax >> 23) + ((amax & 0x7fffffu) > TOP ? 1u : 0u);
    return amax >= 0x7f800000u ? 255u : e > BIAS ? e - BIAS : 0u;
}

/* 1 / scale; a NaN block's values become 0. */
__device__ __forceinline__ float mx_inverse(uint32_t scale) {
    return scale == 255u ? 0.0f : __uint_as_float((254u - scale) << 23);
}

/* The largest of the |value| bits of a quad of lanes (a block of 32: 8 values a
 * lane). */
__device__ __forceinline__ uint32_t mx_quad_max(uint32_t a) {
    a = max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0xB1, 0xF, 0xF, true));
    return max(a, (uint32_t)__builtin_amdgcn_update_dpp(0, (int)a, 0x4E, 0xF, 0xF, true));
}

__device__ __forceinline__ uint32_t mx_amax8(const float (&v)[8]) {
    uint32_t a = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) a = max(a, __float_as_uint(v[e]) & 0x7fffffffu);
    return a;
}

/* Eight values as codes, in the low 32 (MXFP4) or all 64 bits: round to nearest,
 * ties to even. A NaN block's codes are 0. */
template <int TYPE>
__device__ __forceinline__ ghip_u32x2 mx_codes8(const float (&v)[8], uint32_t scale) {
    const float inv = mx_inverse(scale);
    float q[8];
#pragma unroll
    for (int e = 0; e < 8; e++) q[e] = scale == 255u ? 0.0f : v[e] * inv;
    if constexpr (TYPE == GHIP_MXFP8) {
        int lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[0], q[1], 0, false);
        lo = __builtin_amdgcn_cvt_pk_fp8_f32(q[2], q[3], lo, true);
        int hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[4], q[5], 0, false);
        hi = __builtin_amdgcn_cvt_pk_fp8_f32(q[6], q[7], hi, true);
        return (ghip_u32x2){(uint32_t)lo, (uint32_t)hi};
    } else {
        uint32_t c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(0u, q[0], q[1], 1.0f, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[2], q[3], 1.0f, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[4], q[5], 1.0f, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, q[6], q[7], 1.0f, 3);
        return (ghip_u32x2){c, 0u};
    }
}

/* A scale byte as f32. */
__device__ __forceinline__ float mx_scale_f32(uint32_t b) {
    return __uint_as_float(b == 255u ? 0x7fc00000u : b ? b << 23 : 0x400000u);
}

/* Eight MXFP4 codes (the nibbles of c) -> bf16, exact but for what bf16 cannot hold. */
__device__ __forceinline__ ghip_u32x4 mx_fp4_bf16(uint32_t c, float scale) {
    const mx_bf16x2 a = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 0);
    const mx_bf16x2 b = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 1);
    const mx_bf16x2 d = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 2);
    const mx_bf16x2 e = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(c, scale, 3);
    return (ghip_u32x4){__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b),
                        __builtin_bit_cast(uint32_t, d), __builtin_bit_cast(uint32_t, e)};
}

/* Eight MXFP8 codes -> bf16. */
__device__ __forceinline__ ghip_u32x4 mx_fp8_bf16(ghip_u32x2 c, float scale) {
    ghip_u32x4 o;
#pragma unroll
    for (int h = 0; h < 2; h++) {
        const ghip_f32x2 a = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], false);
        const ghip_f32x2 b = __builtin_amdgcn_cvt_pk_f32_fp8((int)c[h], true);
        mx_bf16x2 p, q;
        p[0] = (__bf16)(a[0] * scale);
        p[1] = (__bf16)(a[1] * scale);
        q[0] = (__bf16)(b[0] * scale);
        q[1] = (__bf16)(b[1] * scale);
        o[2 * h] = __builtin_bit_cast(uint32_t, p);
        o[2 * h + 1] = __builtin_bit_cast(uint32_t, q);
    }
    return o;
}

#endif /* GHIP_MX_H */
