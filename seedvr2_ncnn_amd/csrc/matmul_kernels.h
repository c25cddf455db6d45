// The linear and grouped linear kernels' launchers.  Element kinds are the s2_dtype
// codes (0 fp32, 1 bf16, 2 fp16); strides are in elements.
//
//   matmul_kernels.hip       which kernel takes a call; packing; any shape and alignment
//   matmul_tile_kernels.hip  block tiles fed by DMA, and the sum of split k ranges
//   matmul_rows_kernels.hip  few rows
//   matmul_short_kernels.hip many fp32 rows of a short k
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>

#include <algorithm>

namespace s2 {

// y = residual + act(x W^T + bias).  offsets == null: all m rows with one
// weight; else rows offsets[g] .. offsets[g + 1] - 1 with weight and bias g.
struct MatmulArgs {
    const void* x;
    int x_kind;
    long x_stride;
    int m;
    const int* offsets;   // device [groups + 1] or null
    int groups;           // 1 without offsets
    const void* w;        // [groups][n][k]
    int w_kind;           // 1 or 2
    const float* bias;    // [groups][n] or null
    int n, k;
    int act;              // s2_activation
    const void* res;      // of y's kind, or null
    long res_stride;
    void* y;
    int y_kind;
    long y_stride;
    // packed fp32 rows: `planes` bf16 terms of a row, plane q at q * plane elements,
    // zeros from k to plane (a multiple of 64).  Else planes is 1, plane 0.
    int planes;
    long plane;
};

// Tiles of tm rows that the m rows of a call's groups can make.
inline long row_tiles(const MatmulArgs& a, int tm) {
    if (!a.offsets) return ((long)a.m + tm - 1) / tm;
    return ((long)a.m + (long)std::min(a.groups, a.m) * (tm - 1)) / tm;
}

// A call's kernel and what it keeps in the workspace.
struct MatmulPlan {
    enum Kernel { kRows, kTiles, kShort, kAny } kernel;
    int rows, cols;        // kRows: of a tile, 16, 32 or 64 each
    int bm, bn;            // kTiles: the tile
    int parts;             // kTiles: ranges of k; kShort: of rows
    bool whole;            // kTiles, kShort: y and residual in pieces of four columns
    bool pack_x, pack_w;
    size_t x_bytes, w_bytes, sum_bytes;   // 256-byte multiples, in this order
    size_t bytes() const { return x_bytes + w_bytes + sum_bytes; }
};

// The tile and the ranges of k that take the least time over `steps` steps of 128 bytes of
// a row, of tiles of `largest` rows at most and with room for `most` ranges' sums.
struct TileChoice {
    double us;
    int bm, bn, parts;
};
TileChoice choose_tiles(const MatmulArgs& a, long steps, long most, int largest = 256);
// Four neighbours of a row of y, the residual or the bias move as one piece.
bool whole_pieces(const MatmulArgs& a);

// The plan for a call with that much workspace.
MatmulPlan plan_matmul(const MatmulArgs& a, size_t workspace_bytes);
hipError_t launch_matmul(const MatmulArgs& a, void* workspace, size_t workspace_bytes,
                         hipStream_t stream);

// The kernels' own launchers, for calls that plan_matmul gives them.
hipError_t launch_matmul_tiles(const MatmulArgs& a, const MatmulPlan& plan, float* sums,
                               hipStream_t stream);
// parts > 1: a tile's k steps are dealt to `parts` workgroups, whose fp32 accumulators
// go to partial[part][m][n]; matmul_sum_kernel adds them and does the epilogue.  For
// few tiles and long k.
struct TileSplit {
    int ntiles, mtiles;
    int parts;
    bool whole;       // y, residual and n in pieces of four columns
    int pitch;        // of partial's rows: n rounded up to four
    float* partial;
};
hipError_t launch_matmul_sum(const MatmulArgs& a, const TileSplit& split, hipStream_t stream);
constexpr int kShortMost = 160;   // k of the kernel for short k
hipError_t launch_matmul_short(const MatmulArgs& a, const MatmulPlan& plan, hipStream_t stream);
hipError_t launch_matmul_rows(const MatmulArgs& a, const MatmulPlan& plan, hipStream_t stream);

}  // namespace s2
