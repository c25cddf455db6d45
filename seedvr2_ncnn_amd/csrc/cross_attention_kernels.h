// Cross attention's launchers.  Element kinds are the s2_dtype codes, strides are in
// elements.
//
//   cross_attention_kernels.hip  which kernel takes a call; the joining of ranges of keys
//   cross_tile_kernels.hip       16-bit operands
//   cross_f32_kernels.hip        fp32 operands
#pragma once

#include <hip/hip_runtime.h>
#include <stddef.h>
#include <stdint.h>

#include <algorithm>

namespace s2 {

// Rows [.. heads][d] of an operand: sample b's row i of head h begins at b * batch + i *
// row + h * head.  With offsets, row offsets[b] + i of the whole operand and batch 0.
struct CrossRows {
    long batch, row, head;
};

struct CrossArgs {
    const void* q;
    const void* k;
    const void* v;
    void* out;
    int kind, out_kind;
    CrossRows qs, ks, vs, os;
    int batch;
    int lq, lk;               // rows of a sample; with offsets of all samples
    const int* q_offsets;     // device [batch + 1], both or none
    const int* k_offsets;
    const int* key_lengths;   // device [batch] or null
    const uint8_t* key_mask;  // device [batch][lk] (offsets: [lk]), zero for keys left out, or null
    long mask_batch;
    int heads, kv_heads, d;
    float scale;
    int first;                // workgroups of the launches before
};

constexpr int kTileRows = 128, kTileRows32 = 64;   // of 16-bit operands' tiles, of fp32 ones'
constexpr int kTileKeys = 32;
constexpr long kLaunchBlocks = 1 << 23;   // workgroups of a launch
// samples whose offsets a wave holds
constexpr int kScanSamples = 64;
// keys of a head that LDS holds in the kernel for many rows on few of them, and its workgroups
// on a compute unit
constexpr int kShortKeys = 128, kShortEach = 2;

// A call's kernel.  Rows: queries times the heads that share a kv head.
struct CrossPlan {
    int run;      // of 128 rows each that a tile has; 1 but for many rows on few keys
    int tiles;    // of rows of a kv head, at most
    int parts;    // ranges of keys
};

// Sums of a range of keys: [row of q][head][part], d floats each, then the maximum and the
// sum of the weights of each.
struct CrossParts {
    int parts;
    float* sums;
    float2* weights;
};

// `blocks` workgroups of 256 threads, by launches whose threads 32 bits count.
template <typename F>
hipError_t launch_in_turn(const CrossArgs& args, long blocks, F&& launch) {
    CrossArgs a = args;
    for (long at = 0; at < blocks; at += kLaunchBlocks) {
        a.first = (int)at;
        launch(a, (unsigned)std::min(kLaunchBlocks, blocks - at));
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

CrossParts cross_parts(const CrossArgs& a, const CrossPlan& plan, void* workspace);
hipError_t launch_cross_tiles(const CrossArgs& a, const CrossPlan& plan, void* workspace, hipStream_t stream);
hipError_t launch_cross_f32(const CrossArgs& a, const CrossPlan& plan, void* workspace, hipStream_t stream);

size_t cross_attention_workspace(const CrossArgs& a);
hipError_t launch_cross_attention(const CrossArgs& a, void* workspace, size_t workspace_bytes,
                                  hipStream_t stream);

}  // namespace s2
