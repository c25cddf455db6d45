// Launcher of the channels-last group norm (group_norm_kernels.hip).  Element
// kinds are the s2_dtype codes (0 fp32, 1 bf16, 2 fp16); strides are in elements.
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>

namespace s2 {

struct GroupNormArgs {
    const void* x;
    int x_kind;
    long x_frame, x_pixel;   // strides
    int frames, pixels, channels, groups;
    const float* gamma;      // [channels] or null
    const float* beta;       // [channels] or null
    float eps;
    int act;                 // s2_activation
    void* y;
    int y_kind;
    long y_frame, y_pixel;
};

// Partial statistics of a call (0: it needs none).
size_t group_norm_workspace(int frames, int pixels, int channels, int groups);
hipError_t launch_group_norm(const GroupNormArgs& p, void* workspace, hipStream_t stream);

}  // namespace s2
