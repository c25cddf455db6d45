// Products of 16-bit rows with weights in MXFP4 on block tiles.
//
// y = x W^T as W's values in bf16, which hold a code times its scale exactly, on 16x16x32
// products; by fp16 rows the codes alone in fp16 and the scale on each block's sums, a
// product's 32 k being one block, for fp16 does not reach as far.  x goes to LDS as in the
// 16-bit products (matmul_tiles.h; fp32 rows, and fp16 ones that begin at no 16 bytes, as
// planes of bf16 terms); the weight as its codes, a quarter of the bytes,
// 256 k (128 bytes of a row) at a time, and becomes bf16 in operand registers: four
// conversions make an operand of a lane's eight codes, which 16 NI rows share.
//
// A compute unit takes in about 40 KB a microsecond so, with two steps in flight; its caches
// deliver several times that, and what it waits for has not been taken apart: 128 x 2560 by
// 15360 x 2560 17 us, 0.6 PFLOP/s, its bytes once 6.  (In steps of 64 k 30 us, of 256 k with one wave a SIMD 18.4; 41 with the weight's values written
// for the 16-bit tiles.  By fp16 rows 23, where the scales' products add up, 48 as two planes
// and 16-bit tiles.)
#include "mx_tiles.h"

namespace s2 {

namespace {

// BM x BN tile, two groups of four waves of 16 NI x 64 (WN of them side by side), 256 k a
// step, of which each group takes half; their sums meet in LDS at the end.  Wider tiles do
// not leave LDS for two steps in flight under the products of a third.  a.w: codes.
template <int T, int YK, int NI, int WN, int STAGES>
__global__ __launch_bounds__(512, 1) void mx_weight_kernel(MatmulArgs a, TileSplit sp, MxTileScales sc) {
    constexpr int BM = 16 * NI * (4 / WN), BN = 64 * WN;
    constexpr int RB = kBK * 2, XB = BM * RB, WB = BN * RB;   // of x a quarter of a step
    constexpr int SB = 4 * XB + WB + BN * kScaleRow;
    constexpr int XI = BM / 16, WI = 2;   // DMA instructions of a wave; BN / 16 waves load codes
    __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * SB];
    TilePlace p = tile_place(a, sp, BM, BN);
    if (p.rows <= 0) return;   // the whole workgroup
    const int quarters = p.nk;
    p.nk = (quarters + 3) / 4;
    p.kb = (int)((long)p.nk * a.planes * p.part / sp.parts);
    p.ke = (int)((long)p.nk * a.planes * (p.part + 1) / sp.parts);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int grp = wave >> 2, wm = wave % 4 / WN, wn = wave % WN;
    const bool loads_w = wave < BN / 16;
    const int sw = lds_swizzle(l16);
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    const int ck = 8 * sc.blocks;   // of codes, as 16-bit elements
    const TileLoad tx = x_load(a, p);
    const TileLoad tw = tile_load<true>((const uint16_t*)a.w + (long)p.col0 * ck, min(a.n - p.col0, BN), ck, ck, ck);
    const ScaleLoad c = scale_load<true>(sc.w + p.col0 * sc.w_stride, min(a.n - p.col0, BN), sc.w_stride, sc.blocks,
                                         wave % WN);
    const int col = p.col0 + wn * 64 + 4 * l16;
    // bias and residual come under the main loop
    TileEnd<YK, NI> end(a, p.rt, p.rows, wm * 16 * NI, col, sp.whole);
    // Two waves load a quarter of x's 256 k; one past the row is zeros.
    auto issue = [&](int s) {
        int step = p.kb + s, plane = 0;
        while (step >= p.nk) {   // at most twice
            step -= p.nk;
            ++plane;
        }
        const uint32_t st = base + s % STAGES * SB;
        if (loads_w) tile_issue<true, WI>(tw, st + 4 * XB, wave * WI, step * RB, step + 1 == p.nk, ck);
        if (wave < WN)
            lds_dma16(c.rsrc, __builtin_amdgcn_readfirstlane(st + 4 * XB + WB + wave * 64 * kScaleRow), c.vo,
                      __builtin_amdgcn_readfirstlane(step / 2 * kScaleRow));
        const int q = 4 * step + (wave >> 1);
        TileLoad t = tx;
        if (q >= quarters) t.past[0] = t.past[1] = kOutside;
        tile_issue<false, XI>(t, st + (wave >> 1) * XB, (wave & 1) * XI, (uint32_t)(q * RB + plane * a.plane * 2), q + 1 >= quarters,
                              a.x_stride);
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
    int stage = 0, step = p.kb % p.nk;
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        // step s: the loads of later ones may still be in flight
        if (loads_w)
            wait_loads<XI + WI, STAGES - 2>(steps - 1 - s);
        else
            wait_loads<XI, STAGES - 2>(steps - 1 - s);
        block_barrier();   // and no one reads step s - 1
        if (s + STAGES - 1 < steps) issue(s + STAGES - 1);
        const uint8_t* st = lds + stage * SB;
        stage = stage + 1 == STAGES ? 0 : stage + 1;
        const uint8_t* xs = st + 2 * grp * XB + (wm * 16 * NI + l16) * RB;
        const uint8_t* ws = st + 4 * XB + (wn * 64 + l16) * RB + 4 * g;
        const uint8_t* cs = st + 4 * XB + WB + (wn * 64 + l16) * kScaleRow + (step & 1) * 8 + grp * 4;
        uint32_t scales[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) scales[j] = *(const uint32_t*)(cs + 16 * j * kScaleRow);
        const int left = sc.blocks - 8 * step - 4 * grp;
        if (left < 4) {   // past the last block x is zeros, whatever is behind the scales
            const uint32_t keep = left > 0 ? ~(~0u << (8 * left)) : 0u;
#pragma unroll
            for (int j = 0; j < 4; ++j) scales[j] &= keep;
        }
        step = step + 1 == p.nk ? 0 : step + 1;
#pragma unroll
        for (int b = 0; b < 4; ++b) {   // blocks of 32 k
            uint4 fx[NI];
#pragma unroll
            for (int i = 0; i < NI; ++i)
                fx[i] = *(const uint4*)(xs + b / 2 * XB + 16 * i * RB + ((b % 2 * 4 + g) ^ sw) * 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t codes = *(const uint32_t*)(ws + 16 * j * RB + ((4 * grp + b) ^ sw) * 16);
                const uint4 w = T == 1 ? mx_bf16(codes, mx_scale_of(scales[j], b)) : mx_f16(codes);
                const float scale = mx_scale(scales[j] >> (8 * b) & 255u);
#pragma unroll
                for (int i = 0; i < NI; ++i) {
                    if constexpr (T == 1) {
                        acc[i][j] = mfma<1>(fx[i], w, acc[i][j]);
                    } else {
                        const f32x4 v = mfma<2>(fx[i], w, f32x4{0.f, 0.f, 0.f, 0.f});
#pragma unroll
                        for (int r = 0; r < 4; ++r) acc[i][j][r] = fmaf(v[r], scale, acc[i][j][r]);
                    }
                }
            }
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    block_barrier();   // the last stage is no longer read
    f32x4* sums = (f32x4*)lds + (wave & 3) * NI * 4 * 64 + lane;
    if (grp == 1)
#pragma unroll
        for (int i = 0; i < NI * 4; ++i) sums[i * 64] = acc[i / 4][i % 4];
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    block_barrier();
    if (grp == 1) return;
#pragma unroll
    for (int i = 0; i < NI * 4; ++i) acc[i / 4][i % 4] += sums[i * 64];
    if (sp.parts > 1)
        store_part<NI>(a, sp, p, wm * 16 * NI, col, acc);
    else
        end.finish(a, acc);
}

template <int T, int YK>
hipError_t launch(const MatmulArgs& a, const MxTileScales& sc, const TileChoice& t, float* sums, hipStream_t stream) {
    const long mtiles = row_tiles(a, t.bm), ntiles = (a.n + t.bn - 1) / t.bn;
    const long blocks = mtiles * ntiles * t.parts;
    const TileSplit sp{(int)ntiles, (int)mtiles, t.parts, whole_pieces(a), (a.n + 3) / 4 * 4, sums};
    const unsigned nb = (unsigned)blocks;
    if (t.bn == 128)
        mx_weight_kernel<T, YK, 2, 2, 3><<<nb, 512, 0, stream>>>(a, sp, sc);
    else
        mx_weight_kernel<T, YK, 1, 1, 3><<<nb, 512, 0, stream>>>(a, sp, sc);
    if (t.parts > 1) return launch_matmul_sum(a, sp, stream);
    return hipGetLastError();
}

template <int T>
hipError_t launch_y(const MatmulArgs& a, const MxTileScales& sc, const TileChoice& t, float* sums, hipStream_t stream) {
    return a.y_kind == 0   ? launch<T, 0>(a, sc, t, sums, stream)
           : a.y_kind == 1 ? launch<T, 1>(a, sc, t, sums, stream)
                           : launch<T, 2>(a, sc, t, sums, stream);
}

}  // namespace

hipError_t launch_mx_weight_tiles(const MatmulArgs& a, const MxTileScales& scales, const TileChoice& tile, float* sums,
                                  hipStream_t stream) {
    return a.x_kind == 2 ? launch_y<2>(a, scales, tile, sums, stream) : launch_y<1>(a, scales, tile, sums, stream);
}

}  // namespace s2
