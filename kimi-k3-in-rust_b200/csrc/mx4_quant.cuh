// mx4_quant.cuh -- 32 values to one MXFP4 group: E2M1 codes under one E8M0 scale byte.
//     s = floor(log2 max|v|) - 2,  byte = clamp(s + 127, 0, 254),  code = E2M1(v * 2^(127-byte))
// rounded to nearest, ties to even, saturating at +-6. floor(log2) is the fp32 exponent field of
// the largest magnitude; the product with a power of two is exact wherever the code is not 0
// (a result below the normal range is far below the smallest code's border). An infinity gives
// byte 253 and the code 6, which reads back as infinity, beside finite elements rounded under that byte; a
// NaN gives byte 255 (the format's NaN) and zero codes.
#pragma once

#include "common.cuh"

namespace k3c {

// n <= 32 valid elements at p (the others read as 0); vec: p is 16-byte aligned.
__device__ __forceinline__ void mx4_load32(float (&v)[32], const uint16_t *p, int n, int vec) {
    if (vec && n == 32) {
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint4 u = ldg_nc_v4(p + 8 * q);
            const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
            for (int i = 0; i < 4; i++) {
                v[8 * q + 2 * i] = __uint_as_float(w[i] << 16);
                v[8 * q + 2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] = i < n ? bf16_bits_to_f32(p[i]) : 0.0f;
    }
}
__device__ __forceinline__ void mx4_load32(float (&v)[32], const float *p, int n, int vec) {
    if (vec && n == 32) {
#pragma unroll
        for (int q = 0; q < 8; q++) {
            const uint4 u = ldg_nc_v4(p + 4 * q);
            v[4 * q] = __uint_as_float(u.x);
            v[4 * q + 1] = __uint_as_float(u.y);
            v[4 * q + 2] = __uint_as_float(u.z);
            v[4 * q + 3] = __uint_as_float(u.w);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 32; i++) v[i] = i < n ? p[i] : 0.0f;
    }
}

// Eight floats (already scaled) to eight E2M1 codes, element k in bits 4k..4k+3.
__device__ __forceinline__ uint32_t f32x8_to_e2m1(const float *f) {
    uint32_t d;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b0, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b1, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b2, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b3, %8, %7;\n\t"
        "mov.b32 %0, {b0, b1, b2, b3};\n\t}"
        : "=r"(d)
        : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
    return d;
}

// The scale byte of a group whose largest magnitude has these bits (magnitudes order as their bits,
// NaN above infinity), and 2^(127-byte); byte 255, a NaN, has no multiplier and zero codes.
__device__ __forceinline__ uint32_t mx4_scale_byte(uint32_t top) {
    if (top > 0x7F800000u) return 255;
    const uint32_t e = top >> 23;
    return e > 2 ? e - 2 : 0;
}
__device__ __forceinline__ float mx4_multiplier(uint32_t byte) { return __uint_as_float((254u - min(byte, 253u)) << 23); }

// Quantises v, returns the scale byte.
__device__ __forceinline__ uint8_t mx4_quant32(const float (&v)[32], uint4 &codes) {
    uint32_t top = 0;
#pragma unroll
    for (int i = 0; i < 32; i++) top = max(top, __float_as_uint(v[i]) & 0x7FFFFFFFu);
    const uint32_t byte = mx4_scale_byte(top);
    const float m = mx4_multiplier(byte);
    float f[32];
#pragma unroll
    for (int i = 0; i < 32; i++) f[i] = v[i] * m;
    codes = make_uint4(f32x8_to_e2m1(f), f32x8_to_e2m1(f + 8), f32x8_to_e2m1(f + 16), f32x8_to_e2m1(f + 24));
    if (byte == 255) codes = make_uint4(0, 0, 0, 0);
    return (uint8_t)byte;
}

}  // namespace k3c
