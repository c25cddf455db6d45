// The MXFP4 operators' launchers: quantisation of rows and products with weights in
// MXFP4.  A row of k values is blocks of 32, the last one padded: 16 bytes of e2m1 codes
// a block (two a byte, the first in the low half) and one e8m0 scale, 2^(byte - 127).
// Element kinds are the s2_dtype codes; strides are in elements, of codes and scales in
// bytes.
//
//   mx_quantize_kernels.hip  rows to MXFP4 and back
//   mx_linear_kernels.hip    which kernel takes a product; few rows
//   mx_tile_kernels.hip      block tiles of codes
//   mx_weight_kernels.hip    block tiles of 16-bit rows and a weight's codes
#pragma once

#include "matmul_kernels.h"

namespace s2 {

__host__ __device__ inline int mx_blocks(int k) { return (k + 31) / 32; }

struct MxRows {
    const uint8_t* codes;    // 16-byte rows
    long code_stride;
    const uint8_t* scales;
    long scale_stride;
};

// y = residual + act(x W^T + bias): x in MXFP4 (`mx`) or as x_kind says.
struct MxLinearArgs {
    bool mx;
    MxRows xq;
    const void* x;
    int x_kind;
    long x_stride;
    int m;
    MxRows w;                // code_stride 16 mx_blocks(k)
    const float* bias;
    int n, k;
    int act;
    const void* res;
    long res_stride;
    void* y;
    int y_kind;
    long y_stride;
};

hipError_t launch_mx_quantize(const void* x, int x_kind, long x_stride, int m, int k, uint8_t* codes,
                              long code_stride, uint8_t* scales, long scale_stride, hipStream_t stream);
hipError_t launch_mx_dequantize(const MxRows& rows, int m, int k, void* y, int y_kind, long y_stride,
                                hipStream_t stream);

// What a 256 x 256 tile's workspace holds: scales as its kernel reads them.
struct DealtBytes {
    size_t x, w;
};
inline DealtBytes mx_dealt_bytes(int m, int n, int blocks) {
    const size_t steps = (blocks + 7) / 8;
    return {((size_t)m + 255) / 256 * 2 * steps * 1024, ((size_t)n + 255) / 256 * 4 * steps * 512};
}

// Scales of a product on tiles: rows that begin at 16 bytes, but for 256 x 256.
struct MxTileScales {
    const uint8_t* x;
    long x_stride;
    const uint8_t* w;
    long w_stride;
    int blocks;
};

// a: the product with rows of codes as 16-bit elements, k of them eight a block.
// workspace: mx_dealt_bytes for a 256 x 256 tile.
hipError_t launch_mx_tiles(const MatmulArgs& a, const MxTileScales& scales, const TileChoice& tile,
                           float* sums, void* workspace, hipStream_t stream);

// a: the product with x as bf16 rows, or planes of them; its weight the codes.
hipError_t launch_mx_weight_tiles(const MatmulArgs& a, const MxTileScales& scales, const TileChoice& tile,
                                  float* sums, hipStream_t stream);

size_t mx_linear_workspace(const MxLinearArgs& a);
hipError_t launch_mx_linear(const MxLinearArgs& a, void* workspace, size_t workspace_bytes,
                            hipStream_t stream);

}  // namespace s2
