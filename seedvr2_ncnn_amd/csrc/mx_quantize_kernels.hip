// Rows to MXFP4 and back.
//
// A block's scale is X = 2^(floor(log2 max|x|) - 2): the largest magnitude lies in
// [4, 8) X and e2m1's largest number is 6.  It is the exponent field of the largest bit
// pattern less two, so no logarithm is taken; x / X is exact and v_cvt_scalef32_pk_fp4_f32
// rounds it once, to the nearest code, ties to the even one, saturating at 6.  Both
// kernels move their rows once: memory bounds them, 21664 x 10240 in bf16 110 and 106 us,
// 5.1 and 5.3 TB/s of rows and codes (a copy reaches 4.9).  16 or 32 bytes a thread, so that
// a block is four neighbours and its maximum two lane moves.
#include "mx_device.h"

namespace s2 {

namespace {

// Eight values a thread, four threads a block, blocks of a row beside each other.
template <int XK, bool ODD>
__global__ __launch_bounds__(256) void mx_quantize_kernel(const void* x, long x_stride, long pieces,
                                                          int k, int row_pieces, uint8_t* codes,
                                                          long code_stride, uint8_t* scales,
                                                          long scale_stride) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (long)gridDim.x * 256) {
        const long row = i / row_pieces;
        const int p = (int)(i - row * row_pieces);
        const int left = k - 8 * p;
        float v[8];
        if constexpr (XK == 0) {
            piece32<false>((const float*)x + row * x_stride + 8 * p, left, v);
        } else {
            const uint4 q = piece16<false, ODD>((const uint16_t*)x + row * x_stride + 8 * p, left);
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint16_t h = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                v[e] = XK == 1 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
            }
        }
        uint32_t high = 0;   // of magnitudes, whose order is that of their bit patterns
#pragma unroll
        for (int e = 0; e < 8; ++e) high = max(high, __float_as_uint(v[e]) & 0x7fffffffu);
        // rows begin at multiples of four pieces, so a block's threads are neighbours
        high = max(high, (uint32_t)__shfl_xor((int)high, 1));
        high = max(high, (uint32_t)__shfl_xor((int)high, 2));
        const bool nan = high >= 0x7f800000u;
        const uint32_t scale = nan ? kMxNan : max((int)(high >> 23) - 2, 0);
        const float s = mx_scale(scale);
        uint32_t c = 0;
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[0], v[1], s, 0);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[2], v[3], s, 1);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[4], v[5], s, 2);
        c = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(c, v[6], v[7], s, 3);
        *reinterpret_cast<uint32_t*>(codes + row * code_stride + 4 * p) = nan ? 0u : c;
        if ((p & 3) == 0) scales[row * scale_stride + (p >> 2)] = (uint8_t)scale;
    }
}

template <int YK>
__global__ __launch_bounds__(256) void mx_dequantize_kernel(MxRows q, long pieces, int k,
                                                            int row_pieces, void* y,
                                                            long y_stride) {
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < pieces; i += (long)gridDim.x * 256) {
        const long row = i / row_pieces;
        const int p = (int)(i - row * row_pieces);
        const int left = k - 8 * p;
        if (left <= 0) continue;
        const uint32_t c = *reinterpret_cast<const uint32_t*>(q.codes + row * q.code_stride + 4 * p);
        const float s = mx_scale(q.scales[row * q.scale_stride + (p >> 2)]);
        f32x2 v[4];
        v[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 0);
        v[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 1);
        v[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 2);
        v[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c, s, 3);
        const long at = row * y_stride + 8 * p;
        if (left >= 8) {
            store4_any<YK>(y, at, f32x4{v[0][0], v[0][1], v[1][0], v[1][1]});
            store4_any<YK>(y, at + 4, f32x4{v[2][0], v[2][1], v[3][0], v[3][1]});
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (e < left) store1(y, at + e, v[e >> 1][e & 1], YK);
        }
    }
}

unsigned grid_of(long pieces) { return (unsigned)std::min<long>((pieces + 255) / 256, 1L << 20); }

}  // namespace

hipError_t launch_mx_quantize(const void* x, int x_kind, long x_stride, int m, int k, uint8_t* codes,
                              long code_stride, uint8_t* scales, long scale_stride, hipStream_t stream) {
    if (m <= 0) return hipSuccess;
    const int row_pieces = mx_blocks(k) * 4;
    const long pieces = (long)m * row_pieces;
    const unsigned nb = grid_of(pieces);
    const bool odd = (uintptr_t)x % 4 || (m > 1 && x_stride % 2);
    if (x_kind == 0)
        mx_quantize_kernel<0, false><<<nb, 256, 0, stream>>>(x, x_stride, pieces, k, row_pieces, codes,
                                                             code_stride, scales, scale_stride);
    else if (x_kind == 1 && odd)
        mx_quantize_kernel<1, true><<<nb, 256, 0, stream>>>(x, x_stride, pieces, k, row_pieces, codes,
                                                            code_stride, scales, scale_stride);
    else if (x_kind == 1)
        mx_quantize_kernel<1, false><<<nb, 256, 0, stream>>>(x, x_stride, pieces, k, row_pieces, codes,
                                                             code_stride, scales, scale_stride);
    else if (odd)
        mx_quantize_kernel<2, true><<<nb, 256, 0, stream>>>(x, x_stride, pieces, k, row_pieces, codes,
                                                            code_stride, scales, scale_stride);
    else
        mx_quantize_kernel<2, false><<<nb, 256, 0, stream>>>(x, x_stride, pieces, k, row_pieces, codes,
                                                             code_stride, scales, scale_stride);
    return hipGetLastError();
}

hipError_t launch_mx_dequantize(const MxRows& rows, int m, int k, void* y, int y_kind, long y_stride,
                                hipStream_t stream) {
    if (m <= 0) return hipSuccess;
    const int row_pieces = mx_blocks(k) * 4;
    const long pieces = (long)m * row_pieces;
    const unsigned nb = grid_of(pieces);
    if (y_kind == 0)
        mx_dequantize_kernel<0><<<nb, 256, 0, stream>>>(rows, pieces, k, row_pieces, y, y_stride);
    else if (y_kind == 1)
        mx_dequantize_kernel<1><<<nb, 256, 0, stream>>>(rows, pieces, k, row_pieces, y, y_stride);
    else
        mx_dequantize_kernel<2><<<nb, 256, 0, stream>>>(rows, pieces, k, row_pieces, y, y_stride);
    return hipGetLastError();
}

}  // namespace s2
