// Device side of the block-tile kernels: operand rows to LDS by DMA, the workgroups' tiles,
// partial sums of split k ranges.
#pragma once

#include "matmul_device.h"

namespace s2 {

constexpr int kBK = 64;

// DMA of LDS rows of 128 bytes, eight rows an instruction, into 64-row blocks whose
// even and odd instructions differ in the swizzle.
struct TileLoad {
    i32x4 rsrc;
    uint32_t vo[2];     // byte offsets of the lane's chunk in even and odd instructions
    uint32_t past[2];   // set in a plane's last k step where the lane's chunk lies past k
};

// A lane's part of a load through rsrc; ld: elements between rows.
template <bool WEIGHT>
__device__ __forceinline__ TileLoad tile_lanes(i32x4 rsrc, long ld, int k, int lane) {
    const int l8 = lane >> 3;
    TileLoad t;
    t.rsrc = rsrc;
    const int sw = lds_swizzle(l8);   // rows 8 apart differ in bit 2
    const int rem = k % kBK;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
        const int c = (lane & 7) ^ sw ^ (4 * o);
        const int row = WEIGHT ? 4 * l8 + 32 * o : l8 + 8 * o;
        t.vo[o] = (uint32_t)((long)row * ld * 2) + c * 16;
        t.past[o] = rem && c * 8 >= rem ? 0x80000000u : 0u;
    }
    return t;
}

// LDS row r of x is row r.  Of each 64 weight rows, LDS row 16 j + c is row 4 c + j.
// extent: elements of a row.
template <bool WEIGHT>
__device__ __forceinline__ TileLoad tile_load(const uint16_t* base, int rows, long ld, long extent,
                                              int k) {
    const long bytes = rows > 0 ? ((long)(rows - 1) * ld + extent) * 2 : 0;
    return tile_lanes<WEIGHT>(wave_uniform(buffer_rsrc(base, (uint32_t)bytes)), ld, k, threadIdx.x & 63);
}

// Instructions first .. first + COUNT - 1 (first even) of a tile, at k byte offset soff.
template <bool WEIGHT, int COUNT>
__device__ __forceinline__ void tile_issue(const TileLoad& t, uint32_t lds_addr, int first,
                                           uint32_t soff, bool last, long ld) {
    soff = __builtin_amdgcn_readfirstlane(soff);
#pragma unroll
    for (int j = 0; j < COUNT; ++j) {
        const int q = first + j;
        const uint32_t rows = (WEIGHT ? (q & ~7) * 8 + ((q & 7) >> 1) : 8 * (q & ~1)) * (uint32_t)(ld * 2);
        uint32_t vo = t.vo[j & 1] + rows;
        if (last) vo |= t.past[j & 1];
        lds_dma16(t.rsrc, __builtin_amdgcn_readfirstlane(lds_addr + q * 1024), vo, soff);
    }
}

__device__ __forceinline__ void block_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The workgroup's tile and k steps (over the planes of x, one after the other).
struct TilePlace {
    RowTile rt;
    int rows, col0, part, kb, ke, nk;
};

__device__ __forceinline__ TilePlace tile_place(const MatmulArgs& a, const TileSplit& sp, int bm,
                                                int bn) {
    // consecutive tiles share an XCD's L2; four row tiles sweep the columns together.
    // Dealt out over the tiles that there are: a grid is as large as the groups' sizes can
    // make it, and workgroups without a tile come last (dealt out over the grid, 238 of
    // 301 tiles were two rounds on six of the eight XCDs, 72 us; 41 so).
    constexpr int GROUP = 4;
    RowTiles rts(a, bm, sp.mtiles);
    const int mtiles = rts.count;
    const int blocks = mtiles * sp.ntiles * sp.parts;
    TilePlace p;
    if ((int)blockIdx.x >= blocks) {
        p.rows = 0;
        return p;
    }
    const int lid = xcd_remap(blockIdx.x, blocks);
    p.part = lid % sp.parts;
    const int t = lid / sp.parts;
    const int first = t / (GROUP * sp.ntiles) * GROUP;
    const int gm = min(mtiles - first, GROUP);
    const int in = t % (GROUP * sp.ntiles);
    p.rt = rts.at(first + in % gm);
    p.rows = min(p.rt.end - p.rt.row0, bm);
    p.col0 = in / gm * bn;
    p.nk = (a.k + kBK - 1) / kBK;
    const long all = (long)p.nk * a.planes;
    p.kb = (int)(all * p.part / sp.parts);
    p.ke = (int)(all * (p.part + 1) / sp.parts);
    return p;
}

// Byte offsets of a k step in a row of x and of the weight.
struct StepAt {
    uint32_t x, w;
    bool last;   // of its plane
};

__device__ __forceinline__ StepAt step_at(const MatmulArgs& a, const TilePlace& p, int s) {
    int plane = 0;
    while (s >= p.nk) {   // at most twice
        s -= p.nk;
        ++plane;
    }
    StepAt at;
    at.w = (uint32_t)(s * kBK * 2);
    at.x = at.w + (uint32_t)(plane * a.plane * 2);
    at.last = s + 1 == p.nk;
    return at;
}

__device__ __forceinline__ TileLoad x_load(const MatmulArgs& a, const TilePlace& p) {
    const bool packed = a.plane != 0;
    return tile_load<false>((const uint16_t*)a.x + p.rt.row0 * a.x_stride, p.rows, a.x_stride,
                            packed ? a.planes * a.plane : (long)a.k, packed ? kBK : a.k);
}

__device__ __forceinline__ TileLoad w_load(const MatmulArgs& a, const TilePlace& p, int bn) {
    return tile_load<true>((const uint16_t*)a.w + ((long)p.rt.group * a.n + p.col0) * a.k,
                           min(a.n - p.col0, bn), a.k, a.k, a.k);
}

// A wave's accumulators to its part's sums, rows of pitch n rounded up to four.
template <int NI>
__device__ __forceinline__ void store_part(const MatmulArgs& a, const TileSplit& sp, const TilePlace& p,
                                           int row_w, int col, const f32x4 (&acc)[NI][4]) {
    if (col >= a.n) return;
    const int g = (threadIdx.x & 63) >> 4;
    float* out = sp.partial + ((long)p.part * a.m + p.rt.row0) * sp.pitch + col;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row_w + 16 * i + 4 * g + r;
            if (row < p.rows)
                *reinterpret_cast<f32x4*>(out + (long)row * sp.pitch) =
                    f32x4{acc[i][0][r], acc[i][1][r], acc[i][2][r], acc[i][3][r]};
        }
}

// Waits until all but the loads of the last `later` steps (at most MOST), EACH a step,
// have landed.
template <int EACH, int MOST>
__device__ __forceinline__ void wait_loads(int later) {
    if constexpr (MOST == 0) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
        if (later >= MOST)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"(MOST * EACH) : "memory");
        else
            wait_loads<EACH, MOST - 1>(later);
    }
}

}  // namespace s2
