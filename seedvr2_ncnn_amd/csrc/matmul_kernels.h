// Launcher of the linear and grouped linear kernels (matmul_kernels.hip).
// Element kinds are the s2_dtype codes (0 fp32, 1 bf16, 2 fp16); strides are in
// elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>

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
};

size_t matmul_workspace(int m, int n, int k, int x_kind);
hipError_t launch_matmul(const MatmulArgs& a, void* workspace, size_t workspace_bytes,
                         hipStream_t stream);

}  // namespace s2
