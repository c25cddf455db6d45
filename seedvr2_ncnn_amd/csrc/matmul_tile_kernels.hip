// Linear and grouped linear on block tiles: 16-bit operands in 16-byte rows (k % 8 == 0
// or packed).
//
// Both operands go to LDS by buffer_load ... lds (no VGPR staging) in stages of 64 k.
// Descriptors end with the tile's rows and the weight's, and a lane whose 16 bytes lie
// past k reads past the descriptor's end, so ragged m, n and k read zeros.
#include "matmul_device.h"

namespace s2 {

namespace {

constexpr int kBK = 64;

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

// DMA of LDS rows of 128 bytes, eight rows an instruction, into 64-row blocks whose
// even and odd instructions differ in the swizzle.
struct TileLoad {
    i32x4 rsrc;
    uint32_t vo[2];     // byte offsets of the lane's chunk in even and odd instructions
    uint32_t past[2];   // set in a plane's last k step where the lane's chunk lies past k
};

// LDS row r of x is row r.  Of each 64 weight rows, LDS row 16 j + c is row 4 c + j.
// extent: elements of a row.
template <bool WEIGHT>
__device__ __forceinline__ TileLoad tile_load(const uint16_t* base, int rows, long ld, long extent,
                                              int k) {
    const int lane = threadIdx.x & 63;
    const int l8 = lane >> 3;
    TileLoad t;
    const long bytes = rows > 0 ? ((long)(rows - 1) * ld + extent) * 2 : 0;
    t.rsrc = wave_uniform(buffer_rsrc(base, (uint32_t)bytes));
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

// 256x256 tile, eight waves (2 x 4) of 128x64, one workgroup per compute unit.
//
// The two waves of each SIMD (group 0: rows 0-127, group 1: rows 128-255) take turns:
// one issues the 64 MFMAs of a 64-k step from fragment registers while the other reads
// its fragments of the next step, so the matrix core never waits for LDS.  Every phase
// ends at a barrier; group 1 runs one phase behind.  Group 1 loads the weight rows into
// the stage that it has just read (as its last reader), group 0 the x rows a phase
// later; each waits for its loads two phases after issuing them, before the barrier
// that opens the stage.
template <int T, int YK>
__global__ __launch_bounds__(512, 1) void matmul_256_kernel(MatmulArgs a, TileSplit sp) {
    constexpr int TB = 256 * kBK * 2, SB = 2 * TB, RB = kBK * 2;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * SB];
    const TilePlace p = tile_place(a, sp, 256, 256);
    if (p.rows <= 0) return;   // the whole workgroup
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int grp = wave >> 2, wq = wave & 3;
    const int sw = lds_swizzle(l16);
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    const long ldw = a.k;
    // group 0 loads x, group 1 the weight
    TileLoad t;
    if (grp == 0)
        t = x_load(a, p);
    else
        t = w_load(a, p, 256);
    t.rsrc = wave_uniform(t.rsrc);
    auto issue = [&](int stage, int s) {
        const StepAt at = step_at(a, p, s);
        if (grp == 0)
            tile_issue<false, 8>(t, base + stage * SB, wq * 8, at.x, at.last, a.x_stride);
        else
            tile_issue<true, 8>(t, base + stage * SB + TB, wq * 8, at.w, at.last, ldw);
    };
    uint4 fx[2][8], fw[2][4];
    auto read_step = [&](int stage) {
        const uint8_t* st = lds + stage * SB;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int pc = ((4 * kk + g) ^ sw) * 16;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                fx[kk][i] = *(const uint4*)(st + (grp * 128 + 16 * i + l16) * RB + pc);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                fw[kk][j] = *(const uint4*)(st + TB + (wq * 64 + 16 * j + l16) * RB + pc);
        }
    };
    f32x4 acc[8][4];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = p.ke - p.kb;
    issue(0, p.kb);
    if (steps > 1) {
        issue(1, p.kb + 1);
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    } else {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
    block_barrier();
    if (grp == 1) block_barrier();
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        if (grp == 0 && s >= 1 && s + 1 < steps) issue((s + 1) & 1, p.kb + s + 1);
        read_step(s & 1);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        if (grp == 1) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the weight rows of step s + 1
            if (s + 2 < steps) issue(s & 1, p.kb + s + 2);
        }
        block_barrier();
        __builtin_amdgcn_s_setprio(1);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < 8; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = mfma<T>(fx[kk][i], fw[kk][j], acc[i][j]);
        __builtin_amdgcn_s_setprio(0);
        if (grp == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // the x rows of step s + 1
        // group 1's last phase has no one to meet; group 0's barrier here meets the one
        // after group 1's last read
        if (!(grp == 1 && s + 1 == steps)) block_barrier();
    }
    const int col = p.col0 + wq * 64 + 4 * l16;
    if (sp.parts > 1) {
        store_part<8>(a, sp, p, grp * 128, col, acc);
    } else {
        TileEnd<YK, 8> end(a, p.rt, p.rows, grp * 128, col, sp.whole);
        end.finish(a, acc);
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

// BM x BN tile, four waves of 16 NI x 64 (WN of them side by side), two workgroups a
// compute unit.  The loads of STAGES - 1 steps are in flight under the MFMAs of one.
// (Twice the stages with one workgroup a unit, for few tiles, gained nothing: 77 x 2560
// by 15360 x 2560 on 64 x 64 tiles 21 us against 20.)
template <int T, int YK, int NI, int WN, int STAGES>
__global__ __launch_bounds__(256, 1) void matmul_tile_kernel(MatmulArgs a, TileSplit sp) {
    constexpr int BM = 16 * NI * (4 / WN), BN = 64 * WN;
    constexpr int XB = BM * kBK * 2, SB = XB + BN * kBK * 2, RB = kBK * 2;
    constexpr int XI = BM / 32, WI = BN / 32;   // DMA instructions of a wave
    __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * SB];
    const TilePlace p = tile_place(a, sp, BM, BN);
    if (p.rows <= 0) return;   // the whole workgroup
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    const int sw = lds_swizzle(l16);
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    const TileLoad tx = x_load(a, p), tw = w_load(a, p, BN);
    const int col = p.col0 + wn * 64 + 4 * l16;
    // bias and residual come under the main loop
    TileEnd<YK, NI> end(a, p.rt, p.rows, wm * 16 * NI, col, sp.whole);
    auto issue = [&](int s) {
        const StepAt at = step_at(a, p, p.kb + s);
        const uint32_t st = base + s % STAGES * SB;
        tile_issue<false, XI>(tx, st, wave * XI, at.x, at.last, a.x_stride);
        tile_issue<true, WI>(tw, st + XB, wave * WI, at.w, at.last, a.k);
    };
    f32x4 acc[NI][4];
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = p.ke - p.kb;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
        if (s < steps) issue(s);
    int stage = 0;
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        // step s: the loads of later ones may still be in flight
        wait_loads<XI + WI, STAGES - 2>(steps - 1 - s);
        block_barrier();   // and no one reads step s - 1
        // where two stages are read and filled in turn the loads go first; else they follow
        // the LDS reads, which the MFMAs wait for (1 to 8%)
        constexpr bool FIRST = STAGES == 2;
        if (FIRST && s + STAGES - 1 < steps) issue(s + STAGES - 1);
        const uint8_t* st = lds + stage * SB;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        uint4 fx[2][NI], fw[2][4];
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int pc = ((4 * kk + g) ^ sw) * 16;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                fw[kk][j] = *(const uint4*)(st + XB + (wn * 64 + 16 * j + l16) * RB + pc);
#pragma unroll
            for (int i = 0; i < NI; ++i)
                fx[kk][i] = *(const uint4*)(st + (wm * 16 * NI + 16 * i + l16) * RB + pc);
        }
        if (!FIRST) {
            asm volatile("" ::: "memory");
            if (s + STAGES - 1 < steps) issue(s + STAGES - 1);
        }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
            for (int i = 0; i < NI; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = mfma<T>(fx[kk][i], fw[kk][j], acc[i][j]);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if (sp.parts > 1)
        store_part<NI>(a, sp, p, wm * 16 * NI, col, acc);
    else
        end.finish(a, acc);
}

// y = residual + act(sum of the parts + bias), four columns a thread, parts in order.
template <int YK>
__global__ __launch_bounds__(256) void matmul_sum_kernel(MatmulArgs a, TileSplit sp) {
    const int quads = sp.pitch / 4;
    const long all = (long)a.m * quads;
    for (long q = (long)blockIdx.x * 256 + threadIdx.x; q < all; q += (long)gridDim.x * 256) {
        const long row = q / quads;
        const int col = (int)(q - row * quads) * 4;
        const float* src = sp.partial + row * sp.pitch + col;
        f32x4 v = *reinterpret_cast<const f32x4*>(src);
#pragma unroll 4
        for (int i = 1; i < sp.parts; ++i)
            v += *reinterpret_cast<const f32x4*>(src + (long)i * a.m * sp.pitch);
        const int cols = min(4, a.n - col);
        if (a.bias)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) v[j] += a.bias[col + j];
        with_activation(a.act, [&](auto act) {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = activate<YK == 0>(v[j], decltype(act)::value);
        });
        if (a.res)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) v[j] += load1(a.res, row * a.res_stride + col + j, YK);
        const long at = row * a.y_stride + col;
        if (sp.whole) {
            store4(a.y, at, v[0], v[1], v[2], v[3], YK);
        } else if (cols == 4) {
            store4_any<YK>(a.y, at, v);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (j < cols) store1(a.y, at + j, v[j], YK);
        }
    }
}

template <int T, int YK>
hipError_t launch(const MatmulArgs& a, const MatmulPlan& plan, float* sums, hipStream_t stream) {
    const long mtiles = row_tiles(a, plan.bm), ntiles = (a.n + plan.bn - 1) / plan.bn;
    const long blocks = mtiles * ntiles * plan.parts;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    const int pitch = (a.n + 3) / 4 * 4;
    const TileSplit sp{(int)ntiles, (int)mtiles, plan.parts, plan.whole, pitch, sums};
    const unsigned nb = (unsigned)blocks;
    if (plan.bm == 256)
        matmul_256_kernel<T, YK><<<nb, 512, 0, stream>>>(a, sp);
    else if (plan.bn == 128)
        matmul_tile_kernel<T, YK, 4, 2, 2><<<nb, 256, 0, stream>>>(a, sp);
    else if (plan.bm == 128)
        matmul_tile_kernel<T, YK, 2, 1, 3><<<nb, 256, 0, stream>>>(a, sp);
    else
        matmul_tile_kernel<T, YK, 1, 1, 4><<<nb, 256, 0, stream>>>(a, sp);
    if (plan.parts > 1) {
        const long quads = (long)a.m * (pitch / 4);
        matmul_sum_kernel<YK><<<(unsigned)std::min<long>((quads + 255) / 256, 4096), 256, 0, stream>>>(
            a, sp);
    }
    return hipGetLastError();
}

template <int T>
hipError_t launch_y(const MatmulArgs& a, const MatmulPlan& plan, float* sums, hipStream_t stream) {
    return a.y_kind == 0   ? launch<T, 0>(a, plan, sums, stream)
           : a.y_kind == 1 ? launch<T, 1>(a, plan, sums, stream)
                           : launch<T, 2>(a, plan, sums, stream);
}

}  // namespace

hipError_t launch_matmul_tiles(const MatmulArgs& a, const MatmulPlan& plan, float* sums,
                               hipStream_t stream) {
    return a.w_kind == 2 ? launch_y<2>(a, plan, sums, stream) : launch_y<1>(a, plan, sums, stream);
}

}  // namespace s2
