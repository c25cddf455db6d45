// Device side of the MXFP4 kernels: scales and conversions.
#pragma once

#include "matmul_device.h"
#include "mx_kernels.h"

namespace s2 {

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));

constexpr uint32_t kMxNan = 255;   // the scale of a block without values

// Byte b of four scales as what the conversions of codes take: they read the exponent field
// alone, 2^-127 for 0 and a NaN for 255.
__device__ __forceinline__ float mx_scale_of(uint32_t scales, int b) {
    return __uint_as_float(b == 3 ? scales >> 1 : scales << (23 - 8 * b));
}

// 2^(scale - 127); a NaN for 255
__device__ __forceinline__ float mx_scale(uint32_t scale) {
    return __uint_as_float(scale == 0 ? 0x00400000u : scale == kMxNan ? 0x7fc00000u : scale << 23);
}

typedef int i32x8 __attribute__((ext_vector_type(8)));

// 16x16x128 of two operands in e2m1: lane (row l16, group g) holds a block of 32 k of its
// row and the block's scale in byte ABYTE or BBYTE of sa or sb.
template <int ABYTE, int BBYTE>
__device__ __forceinline__ f32x4 mx_mfma(uint4 a, uint4 b, f32x4 c, uint32_t sa, uint32_t sb) {
    const i32x8 x = {(int)a.x, (int)a.y, (int)a.z, (int)a.w, 0, 0, 0, 0};
    const i32x8 y = {(int)b.x, (int)b.y, (int)b.z, (int)b.w, 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(x, y, c, 4, 4, ABYTE, (int)sa, BBYTE, (int)sb);
}

// Eight codes as bf16, which holds every code times a scale up to its largest number.
__device__ __forceinline__ uint4 mx_bf16(uint32_t codes, float scale) {
    return make_uint4(
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, 3)));
}

// Eight codes as fp16.
__device__ __forceinline__ uint4 mx_f16(uint32_t codes) {
    return make_uint4(
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 0)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 1)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 2)),
        __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(codes, 1.f, 3)));
}

// Eight fp16 values as two bf16 terms each, whose sum is exact: 11 bits, by truncation the
// first eight and the rest.
__device__ __forceinline__ void mx_terms16(uint4 v, uint4 (&t)[2]) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float v0 = (float)__builtin_bit_cast(_Float16, (uint16_t)w[e]);
        const float v1 = (float)__builtin_bit_cast(_Float16, (uint16_t)(w[e] >> 16));
        const uint32_t b0 = __float_as_uint(v0) & 0xffff0000u, b1 = __float_as_uint(v1) & 0xffff0000u;
        hi[e] = (b0 >> 16) | b1;
        // an infinity stays in the first term, a NaN's payload lies in its upper bits
        lo[e] = pack2_bf16_rne(fabsf(v0) == __builtin_inff() ? 0.f : v0 - __uint_as_float(b0),
                               fabsf(v1) == __builtin_inff() ? 0.f : v1 - __uint_as_float(b1));
    }
    t[0] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    t[1] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
}

}  // namespace s2
