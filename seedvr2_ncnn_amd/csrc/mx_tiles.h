// Device side of the MXFP4 products on block tiles: scales of rows to LDS by DMA.
#pragma once

#include "matmul_tiles.h"
#include "mx_device.h"

namespace s2 {

constexpr int kScaleRow = 16;   // bytes of a row's scales in LDS: 512 k

// DMA of the scales of 64 rows, a row a lane.
struct ScaleLoad {
    i32x4 rsrc;
    uint32_t vo;
};

// LDS row r of x is row r.  Of each 64 weight rows, LDS row 16 j + c is row 4 c + j.
// rows: from base on; block: of 64 rows.
template <bool WEIGHT>
__device__ __forceinline__ ScaleLoad scale_load(const uint8_t* base, int rows, long ld, int blocks,
                                                int block) {
    const int lane = threadIdx.x & 63;
    const int row = 64 * block + (WEIGHT ? 4 * (lane & 15) + (lane >> 4) : lane);
    // whole dwords: rows begin at 16 bytes, so the last one's is no one else's
    const long bytes = rows > 0 ? (long)(rows - 1) * ld + (blocks + 3) / 4 * 4 : 0;
    return ScaleLoad{wave_uniform(buffer_rsrc(base, (uint32_t)bytes)), (uint32_t)(row * ld)};
}

}  // namespace s2
