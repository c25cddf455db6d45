// Products of two MXFP4 operands on block tiles.
//
// 32 codes and eight 16-bit elements are 16 bytes alike, and one 16x16x128 product of codes
// takes as long as one 16x16x32 product of 16-bit elements.  So the tiles, their LDS rows
// of 128 bytes (256 k here), the DMA and its swizzle are those of the 16-bit products
// (matmul_tiles.h, with a row's codes as 16-bit elements, four values each); every step
// does four times the k.  What comes with it are the scales: 16 bytes of a row (two
// steps) are one lane's DMA, and a lane takes those of its blocks g and 4 + g out of the
// eight of a step.
#include "mx_tiles.h"

namespace s2 {

namespace {

// The scales of a lane's blocks g and 4 + g of step s, in the lowest bytes.
__device__ __forceinline__ uint2 scale_pair(const uint8_t* row, int s) {
    const int g = (threadIdx.x & 63) >> 4;
    const uint2 v = *(const uint2*)(row + 8 * (s & 1));
    return make_uint2(v.x >> (8 * g), v.y >> (8 * g));
}

// Past the last block the codes are zeros; a scale of 1 there, whatever lies behind the
// row.  left: blocks of the step.
__device__ __forceinline__ uint2 scales_past(uint2 pair, int left) {
    const int g = (threadIdx.x & 63) >> 4;
    return make_uint2(g >= left ? 127u : pair.x, 4 + g >= left ? 127u : pair.y);
}

// The step after which a tile's scales are past the row, and how many blocks it has.
struct LastStep {
    int step, left;
    __device__ __forceinline__ LastStep(const MxTileScales& sc)
        : step(sc.blocks % 8 ? sc.blocks / 8 : -1), left(sc.blocks % 8) {}
};

// Scales dealt out to the lanes of mx_256_kernel: of 128 rows of x and a step, lane (g,
// l16) has 16 bytes, blocks g and 4 + g of rows l16, 16 + l16, ..; of 64 weight rows
// 8 bytes, of rows 4 l16, 4 l16 + 1, ..  So a wave's scales of a step are one LDS read of x's
// and one of the weight's, in six registers (a read for each row and a register for each
// spilled: 1045 us for 21664 x 2560 by 10240 x 2560 with tanh-GELU, 551 so), and DMA moves them as
// they lie.  1 past the last block, and past the last row.
struct DealJob {
    const uint8_t* src;
    long stride;
    int rows;        // of src
    long dwords;     // of dst
    uint32_t* dst;
};

template <bool WEIGHT>
__device__ __forceinline__ uint32_t dealt(const DealJob& job, long i, int blocks, int steps) {
    constexpr int D = WEIGHT ? 2 : 4;   // dwords of a lane
    const int d = (int)(i % D), lane = (int)(i / D % 64);
    const long t = i / (D * 64);
    const int step = (int)(t % steps);
    const long group = t / steps;
    const int l16 = lane & 15, b = step * 8 + (lane >> 4);
    uint32_t v = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const int r = 2 * d + (e >> 1);
        const long row = WEIGHT ? group * 64 + 4 * l16 + r : group * 128 + 16 * r + l16;
        const int at = b + 4 * (e & 1);
        const uint32_t s = row < job.rows && at < blocks ? job.src[row * job.stride + at] : 127u;
        v |= s << (8 * e);
    }
    return v;
}

__global__ __launch_bounds__(256) void mx_deal_kernel(DealJob x, DealJob w, int blocks, int steps) {
    const long all = x.dwords + w.dwords;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) {
        if (i < x.dwords)
            x.dst[i] = dealt<false>(x, i, blocks, steps);
        else
            w.dst[i - x.dwords] = dealt<true>(w, i - x.dwords, blocks, steps);
    }
}

// 256x256 tile, eight waves (2 x 4) of 128x64, one workgroup per compute unit; the two
// groups of waves take turns at the matrix cores as in the 16-bit products.  21664 x 2560 by
// 10240 x 2560 with tanh-GELU 360 to 395 us by the card, 3.0 PFLOP/s: ten steps of 2 us and 7 us of first loads
// and epilogue a tile; 8192^3 3.9 to 4.3, of 6.5 that products of random codes reach without
// memory at the clocks that their power leaves.
template <int YK>
__global__ __launch_bounds__(512, 1) void mx_256_kernel(MatmulArgs a, TileSplit sp, const uint32_t* x_scales,
                                                        const uint32_t* w_scales) {
    constexpr int TB = 256 * kBK * 2, SB = 2 * TB, RB = kBK * 2, CB = 4096;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * (SB + CB)];
    const TilePlace p = tile_place(a, sp, 256, 256);
    if (p.rows <= 0) return;   // the whole workgroup
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int grp = wave >> 2, wq = wave & 3;
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    // Group 0 loads x and all scales, its first two waves x's 1 KB a step each, the others the
    // weight's; group 1 loads the weight.  Group 1 fills a stage while its waves still read it,
    // which is right for what a wave reads alone, the 64 weight rows that it loads, and for
    // nothing else; group 0 fills one that no wave reads any more.
    i32x4 rt;
    if (grp == 0)
        rt = x_load(a, p).rsrc;
    else
        rt = w_load(a, p, 256).rsrc;
    rt = wave_uniform(rt);
    const bool of_x = wq < 2;
    const uint32_t* scales = of_x ? x_scales + ((long)p.rt.row0 / 128 + wq) * p.nk * 256
                                  : w_scales + ((long)p.col0 / 64 + 2 * (wq & 1)) * p.nk * 128;
    // 64 rows of the weight are 512 bytes a step: lanes 32 .. 63 take the next 64
    const uint32_t half = (uint32_t)p.nk * 512;
    const i32x4 rc = wave_uniform(buffer_rsrc(scales, 2 * half));
    // Lane numbers that the compiler takes as new: what follows from them is computed anew in
    // every step, since kept in registers it would be spilled, and a reload waits for the DMA
    // before it (551 us, 458 so).
    auto this_lane = [] {
        int l = threadIdx.x & 63;
        asm volatile("" : "+v"(l));
        return l;
    };
    auto issue = [&](int stage, int s) {
        const StepAt at = step_at(a, p, s);
        const int l = this_lane();
        if (grp == 0) {
            lds_dma16(rc, __builtin_amdgcn_readfirstlane(base + 2 * SB + stage * CB + wq * 1024),
                      of_x ? l * 16 : (l & 31) * 16 + (l >> 5) * half,
                      __builtin_amdgcn_readfirstlane((uint32_t)s * (of_x ? 1024 : 512)));
            tile_issue<false, 8>(tile_lanes<false>(rt, a.x_stride, a.k, l), base + stage * SB, wq * 8, at.x, at.last,
                                 a.x_stride);
        } else
            tile_issue<true, 8>(tile_lanes<true>(rt, a.k, a.k, l), base + stage * SB + TB, wq * 8, at.w, at.last, a.k);
    };
    uint4 fx[2][8], fw[2][4];
    uint4 sx;
    uint2 sw2;
    auto read_step = [&](int stage) {
        const int l = this_lane();
        const int l16 = l & 15;
        const uint8_t* st = lds + stage * SB + l16 * RB;
        const uint8_t* cs = lds + 2 * SB + stage * CB;
        sx = *(const uint4*)(cs + grp * 1024 + l * 16);
        sw2 = *(const uint2*)(cs + 2048 + wq * 512 + l * 8);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int pc = ((4 * kk + (l >> 4)) ^ lds_swizzle(l16)) * 16;
#pragma unroll
            for (int i = 0; i < 8; ++i) fx[kk][i] = *(const uint4*)(st + pc + (grp * 128 + 16 * i) * RB);
#pragma unroll
            for (int j = 0; j < 4; ++j) fw[kk][j] = *(const uint4*)(st + pc + TB + (wq * 64 + 16 * j) * RB);
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
        asm volatile("s_waitcnt vmcnt(8)" ::: "memory");   // a step is nine loads, or group 1's eight
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
        auto products = [&](auto half_k) {
            constexpr int KK = decltype(half_k)::value;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t a4 = i == 0 ? sx.x : i == 1 ? sx.y : i == 2 ? sx.z : sx.w;
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    const uint32_t b4 = j ? sw2.y : sw2.x;
                    f32x4* c0 = &acc[2 * i][2 * j];
                    f32x4* c1 = &acc[2 * i + 1][2 * j];
                    c0[0] = mx_mfma<KK, KK>(fx[KK][2 * i], fw[KK][2 * j], c0[0], a4, b4);
                    c0[1] = mx_mfma<KK, 2 + KK>(fx[KK][2 * i], fw[KK][2 * j + 1], c0[1], a4, b4);
                    c1[0] = mx_mfma<2 + KK, KK>(fx[KK][2 * i + 1], fw[KK][2 * j], c1[0], a4, b4);
                    c1[1] = mx_mfma<2 + KK, 2 + KK>(fx[KK][2 * i + 1], fw[KK][2 * j + 1], c1[1], a4, b4);
                }
            }
        };
        products(std::integral_constant<int, 0>{});
        products(std::integral_constant<int, 1>{});
        // the compiler would move them behind the barrier, out of this group's turn (423 us,
        // 378 so)
#pragma unroll
        for (int i = 0; i < 8; ++i)
            asm volatile("" : "+v"(acc[i][0]), "+v"(acc[i][1]), "+v"(acc[i][2]), "+v"(acc[i][3]));
        __builtin_amdgcn_s_setprio(0);
        if (grp == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // x and scales of step s + 1
        // group 1's last phase has no one to meet; group 0's barrier here meets the one
        // after group 1's last read
        if (!(grp == 1 && s + 1 == steps)) block_barrier();
    }
    const int col = p.col0 + wq * 64 + 4 * (threadIdx.x & 15);
    if (sp.parts > 1) {
        store_part<8>(a, sp, p, grp * 128, col, acc);
    } else {
        TileEnd<YK, 8> end(a, p.rt, p.rows, grp * 128, col, sp.whole);
        end.finish(a, acc);
    }
}

// BM x BN tile, four waves of 16 NI x 64 (WN of them side by side).  The loads of STAGES -
// 1 steps are in flight under the products of one.
template <int YK, int NI, int WN, int STAGES>
__global__ __launch_bounds__(256, 1) void mx_tile_kernel(MatmulArgs a, TileSplit sp, MxTileScales sc) {
    constexpr int BM = 16 * NI * (4 / WN), BN = 64 * WN;
    constexpr int XB = BM * kBK * 2, SB = XB + BN * kBK * 2, RB = kBK * 2;
    constexpr int XI = BM / 32, WI = BN / 32;   // DMA instructions of a wave
    constexpr int PAIRS = STAGES / 2 + 1;       // pairs of steps that STAGES steps lie in
    constexpr int CB = (BM + BN) * kScaleRow, CI = (BM + BN) / 64;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * SB + PAIRS * CB];
    const TilePlace p = tile_place(a, sp, BM, BN);
    if (p.rows <= 0) return;   // the whole workgroup
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int wm = wave / WN, wn = wave % WN;
    const int sw = lds_swizzle(l16);
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    const TileLoad tx = x_load(a, p), tw = w_load(a, p, BN);
    // 64 rows' scales a wave, x's first; with fewer such than waves, some load the same
    const int cb = wave % CI;
    ScaleLoad c;
    if (cb < BM / 64)
        c = scale_load<false>(sc.x + p.rt.row0 * sc.x_stride, p.rows, sc.x_stride, sc.blocks, cb);
    else
        c = scale_load<true>(sc.w + p.col0 * sc.w_stride, min(a.n - p.col0, BN), sc.w_stride, sc.blocks,
                             cb - BM / 64);
    c.rsrc = wave_uniform(c.rsrc);
    const int col = p.col0 + wn * 64 + 4 * l16;
    // bias and residual come under the main loop
    TileEnd<YK, NI> end(a, p.rt, p.rows, wm * 16 * NI, col, sp.whole);
    auto issue = [&](int s) {
        const StepAt at = step_at(a, p, p.kb + s);
        const int pair = (p.kb + s) >> 1;
        if (s == 0 || !((p.kb + s) & 1))
            lds_dma16(c.rsrc,
                      __builtin_amdgcn_readfirstlane(base + STAGES * SB + pair % PAIRS * CB + cb * 64 * kScaleRow),
                      c.vo, __builtin_amdgcn_readfirstlane(pair * kScaleRow));
        const uint32_t st = base + s % STAGES * SB;
        tile_issue<false, XI>(tx, st, wave * XI, at.x, at.last, a.x_stride);
        tile_issue<true, WI>(tw, st + XB, wave * WI, at.w, at.last, a.k);
    };
    const LastStep last(sc);
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
        // step s: the loads of later ones may still be in flight, but for as many of the
        // first of them as those steps have loads of scales
        wait_loads<XI + WI, STAGES - 2>(steps - 1 - s);
        block_barrier();   // and no one reads step s - 1
        // where two stages are read and filled in turn the loads go first; else they follow
        // the LDS reads, which the MFMAs wait for
        constexpr bool FIRST = STAGES == 2;
        if (FIRST && s + STAGES - 1 < steps) issue(s + STAGES - 1);
        const uint8_t* st = lds + stage * SB;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        const uint8_t* cs = lds + STAGES * SB + ((p.kb + s) >> 1) % PAIRS * CB;
        uint2 sx[NI], sw4[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) sw4[j] = scale_pair(cs + (BM + wn * 64 + 16 * j + l16) * kScaleRow, p.kb + s);
#pragma unroll
        for (int i = 0; i < NI; ++i) sx[i] = scale_pair(cs + (wm * 16 * NI + 16 * i + l16) * kScaleRow, p.kb + s);
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
        if (p.kb + s == last.step) {
#pragma unroll
            for (int i = 0; i < NI; ++i) sx[i] = scales_past(sx[i], last.left);
#pragma unroll
            for (int j = 0; j < 4; ++j) sw4[j] = scales_past(sw4[j], last.left);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = mx_mfma<0, 0>(fx[0][i], fw[0][j], acc[i][j], sx[i].x, sw4[j].x);
#pragma unroll
        for (int i = 0; i < NI; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = mx_mfma<0, 0>(fx[1][i], fw[1][j], acc[i][j], sx[i].y, sw4[j].y);
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    if (sp.parts > 1)
        store_part<NI>(a, sp, p, wm * 16 * NI, col, acc);
    else
        end.finish(a, acc);
}

template <int YK>
hipError_t launch(const MatmulArgs& a, const MxTileScales& sc, const TileChoice& t, float* sums,
                  void* workspace, hipStream_t stream) {
    const long mtiles = row_tiles(a, t.bm), ntiles = (a.n + t.bn - 1) / t.bn;
    const long blocks = mtiles * ntiles * t.parts;
    const TileSplit sp{(int)ntiles, (int)mtiles, t.parts, whole_pieces(a), (a.n + 3) / 4 * 4, sums};
    const unsigned nb = (unsigned)blocks;
    if (t.bm == 256) {
        const int steps = (a.k + kBK - 1) / kBK;
        const DealtBytes size = mx_dealt_bytes(a.m, a.n, a.k / 8);
        uint32_t* dealt = (uint32_t*)workspace;
        const DealJob x{sc.x, sc.x_stride, a.m, (long)size.x / 4, dealt};
        const DealJob w{sc.w, sc.w_stride, a.n, (long)size.w / 4, dealt + size.x / 4};
        const long all = x.dwords + w.dwords;
        mx_deal_kernel<<<(unsigned)std::min<long>((all + 255) / 256, 4096), 256, 0, stream>>>(x, w, sc.blocks,
                                                                                              steps);
        mx_256_kernel<YK><<<nb, 512, 0, stream>>>(a, sp, x.dst, w.dst);
    } else if (t.bn == 128)
        mx_tile_kernel<YK, 4, 2, 2><<<nb, 256, 0, stream>>>(a, sp, sc);
    else if (t.bm == 128)
        mx_tile_kernel<YK, 2, 1, 3><<<nb, 256, 0, stream>>>(a, sp, sc);
    else
        mx_tile_kernel<YK, 1, 1, 4><<<nb, 256, 0, stream>>>(a, sp, sc);
    if (t.parts > 1) return launch_matmul_sum(a, sp, stream);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_mx_tiles(const MatmulArgs& a, const MxTileScales& scales, const TileChoice& tile,
                           float* sums, void* workspace, hipStream_t stream) {
    return a.y_kind == 0   ? launch<0>(a, scales, tile, sums, workspace, stream)
           : a.y_kind == 1 ? launch<1>(a, scales, tile, sums, workspace, stream)
                           : launch<2>(a, scales, tile, sums, workspace, stream);
}

}  // namespace s2
