// Matrix products with bias, activation and residual in the epilogue, over all
// rows (s2_linear) or over ragged row groups with a weight each
// (s2_grouped_linear):  y = residual + act(x W^T + bias).
//
// x [m][k] and W [n][k] are both k-contiguous, the operand layout of the 16-bit
// MFMAs.  Row 16 j + c of the 64 weight rows of a wave stands in LDS for column
// 4 c + j, so that accumulators j = 0 .. 3 of a lane are four neighbours of a row
// of y, and 16 lanes hold 64: the epilogue adds bias and residual and stores whole
// 128-byte row pieces straight from the registers, with one rounding at the end.
#include "matmul_kernels.h"

#include <algorithm>
#include <type_traits>

#include "activations.h"
#include "s2_device.h"

namespace s2 {

namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// T: 1 bf16, 2 fp16
template <int T>
__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
    if constexpr (T == 1)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Rows [row0, end) of group `group` that tile t of tm rows starts at; end == row0
// when there is no such tile.
struct RowTile {
    int row0, end, group;
};

__device__ __forceinline__ RowTile row_tile(const MatmulArgs& a, int t, int tm) {
    if (!a.offsets) return RowTile{t * tm, a.m, 0};
    // every wave counts the groups' tiles, 64 groups at a time; offsets are kept
    // to [0, m], whatever they hold
    const int lane = threadIdx.x & 63;
    for (int g0 = 0; g0 < a.groups; g0 += 64) {
        const int g = g0 + lane;
        int start = 0, end = 0;
        if (g < a.groups) {
            start = max(a.offsets[g], 0);
            end = min(a.offsets[g + 1], a.m);
        }
        const int tiles = end > start ? (end - start + tm - 1) / tm : 0;
        int upto = tiles;   // tiles of the groups up to this one
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int other = __shfl_up(upto, o);
            if (lane >= o) upto += other;
        }
        const uint64_t past = __ballot(upto > t);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            const int first = __shfl(start, l) + (t - __shfl(upto - tiles, l)) * tm;
            return RowTile{__builtin_amdgcn_readfirstlane(first),
                           __builtin_amdgcn_readfirstlane(__shfl(end, l)),
                           __builtin_amdgcn_readfirstlane(g0 + l)};
        }
        t -= __builtin_amdgcn_readfirstlane(__shfl(upto, 63));
    }
    return RowTile{0, 0, 0};
}

// Tiles of tm rows that m rows in a call's groups can make.
long row_tiles(const MatmulArgs& a, int tm) {
    if (!a.offsets) return ((long)a.m + tm - 1) / tm;
    return ((long)a.m + (long)std::min(a.groups, a.m) * (tm - 1)) / tm;
}

__device__ __forceinline__ float load1(const void* p, long idx, int kind) {
    if (kind == 1) return bf16_to_f32(((const uint16_t*)p)[idx]);
    if (kind == 2) return (float)((const _Float16*)p)[idx];
    return ((const float*)p)[idx];
}

__device__ __forceinline__ void store1(void* p, long idx, float v, int kind) {
    if (kind == 1)
        ((uint16_t*)p)[idx] = f32_to_bf16(v);
    else if (kind == 2)
        ((_Float16*)p)[idx] = f32_to_f16(v);
    else
        ((float*)p)[idx] = v;
}

// Four neighbours of a row of y, the residual or the bias move as one piece.
bool whole_pieces(const MatmulArgs& a) {
    const size_t e = a.y_kind ? 8 : 16;
    return a.n % 4 == 0 && a.y_stride % 4 == 0 && (uintptr_t)a.y % e == 0 &&
           (uintptr_t)a.bias % 16 == 0 &&
           (!a.res || (a.res_stride % 4 == 0 && (uintptr_t)a.res % e == 0));
}

template <int ACT>
__device__ __forceinline__ float act_of(float v) {
    return activate(v, ACT);
}

// Epilogue of a wave's tile of NI x 16 rows and 64 columns: accumulator [i][j][r] is
// row row_w + 16 i + 4 g + r of the block tile's `rows`, column col + j.  WHOLE: pieces
// of four; else single elements.
template <int YK, int NI, bool WHOLE>
__device__ __forceinline__ void epilogue(const MatmulArgs& a, const RowTile& rt, int rows, int row_w,
                                         int col, const f32x4 (&acc)[NI][4]) {
    const int g = (threadIdx.x & 63) >> 4;
    if (col >= a.n) return;
    f32x4 b = {0.f, 0.f, 0.f, 0.f};
    if (a.bias) {
        const float* bias = a.bias + (long)rt.group * a.n + col;
        if (WHOLE) {
            b = *reinterpret_cast<const f32x4*>(bias);
        } else {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (col + j < a.n) b[j] = bias[j];
        }
    }
    auto emit = [&](auto act_tag) {
        constexpr int ACT = decltype(act_tag)::value;
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const int r0 = row_w + 16 * i + 4 * g;
            const long row = rt.row0 + r0;
            f32x4 res[4];
            if (a.res) {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    if (r0 + r >= rows) continue;
                    const long at = (row + r) * a.res_stride + col;
                    if (!WHOLE) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            if (col + j < a.n) res[r][j] = load1(a.res, at + j, YK);
                    } else if (YK == 0) {
                        res[r] = *reinterpret_cast<const f32x4*>((const float*)a.res + at);
                    } else {
                        const uint2 q = *reinterpret_cast<const uint2*>((const uint16_t*)a.res + at);
                        const uint32_t w[2] = {q.x, q.y};
#pragma unroll
                        for (int j = 0; j < 4; ++j) {
                            const uint16_t h = (uint16_t)(w[j >> 1] >> (16 * (j & 1)));
                            res[r][j] = YK == 1 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
                        }
                    }
                }
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                if (r0 + r >= rows) continue;
                float v[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    v[j] = act_of<ACT>(acc[i][j][r] + b[j]);
                    if (a.res) v[j] += res[r][j];
                }
                const long at = (row + r) * a.y_stride + col;
                if (WHOLE) {
                    store4(a.y, at, v[0], v[1], v[2], v[3], YK);
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (col + j < a.n) store1(a.y, at + j, v[j], YK);
                }
            }
        }
    };
    if (a.act == S2_ACT_NONE)
        emit(std::integral_constant<int, S2_ACT_NONE>{});
    else if (a.act == S2_ACT_GELU)
        emit(std::integral_constant<int, S2_ACT_GELU>{});
    else if (a.act == S2_ACT_SILU)
        emit(std::integral_constant<int, S2_ACT_SILU>{});
    else
        emit(std::integral_constant<int, S2_ACT_GELU_TANH>{});
}

// fp32 as a sum of bf16 values: each takes the top 8 bits of what the ones before
// leave, by truncation, which cannot overflow and leaves an exact rest.  The last
// of two rounds instead (to 2^-15 of x); three are exact.  Infinities and NaNs
// stay in the first.
template <int XP>
__device__ __forceinline__ void split_bf16(float x, uint16_t (&h)[XP]) {
    const bool finite = (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u;
    if (!finite) {
        h[0] = f32_to_bf16(x);
#pragma unroll
        for (int i = 1; i < XP; ++i) h[i] = 0;
        return;
    }
#pragma unroll
    for (int i = 0; i < XP; ++i) {
        h[i] = i + 1 == XP ? f32_to_bf16(x) : (uint16_t)(__float_as_uint(x) >> 16);
        x -= bf16_to_f32(h[i]);
    }
}

// Eight consecutive k of a row as an MFMA operand piece.  GRAN elements lie together
// (8: 16 bytes of 16-bit elements, 4, or 1); FULL: all eight are before k.
template <int GRAN, bool FULL>
__device__ __forceinline__ uint4 piece16(const uint16_t* p, int left) {
    if constexpr (GRAN == 8) {
        if (FULL || left > 0) return *reinterpret_cast<const uint4*>(p);
        return make_uint4(0, 0, 0, 0);
    } else {
        alignas(16) uint16_t h[8];
#pragma unroll
        for (int e = 0; e < 8; e += GRAN) {
            if constexpr (GRAN == 4) {
                uint2 q = make_uint2(0, 0);
                if (FULL || left > e) q = *reinterpret_cast<const uint2*>(p + e);
                *reinterpret_cast<uint2*>(h + e) = q;
            } else {
                h[e] = FULL || left > e ? p[e] : (uint16_t)0;
            }
        }
        return pack8_bf16(h);
    }
}

template <int GRAN, bool FULL>
__device__ __forceinline__ void piece32(const float* p, int left, float (&v)[8]) {
#pragma unroll
    for (int e = 0; e < 8; e += 4) {
        if constexpr (GRAN >= 4) {
            f32x4 q = {0.f, 0.f, 0.f, 0.f};
            if (FULL || left > e) q = *reinterpret_cast<const f32x4*>(p + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[e + i] = q[i];
        } else {
#pragma unroll
            for (int i = 0; i < 4; ++i) v[e + i] = FULL || left > e + i ? p[e + i] : 0.f;
        }
    }
}

// Few rows: up to 16 * MT of them by 16 columns a workgroup.  What costs is reading
// the weight, once, straight into the MFMAs' operand registers; the waves take every
// other 64 k (128 bytes of each weight row), x comes from the caches, and the waves'
// sums meet in LDS.  Rows and columns past the end repeat the last one, and are
// dropped.
template <int T, int XP, int MT, int GRAN>
__global__ __launch_bounds__(512) void matmul_rows_kernel(MatmulArgs a, int ntiles) {
    constexpr int U = MT * (XP ? 2 : 1) >= 4 ? 2 : 4;   // 64-k chunks in flight
    constexpr int PL = XP ? XP : 1;
    __shared__ float sums[8][MT * 256];
    const RowTile rt = row_tile(a, blockIdx.x / ntiles, 16 * MT);
    const int col0 = blockIdx.x % ntiles * 16;
    const int rows = min(rt.end - rt.row0, 16 * MT);
    if (rows <= 0) return;   // the whole workgroup
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int l16 = lane & 15, g = lane >> 4;
    const uint16_t* w = (const uint16_t*)a.w +
                        ((long)rt.group * a.n + min(col0 + l16, a.n - 1)) * a.k + 8 * g;
    long xo[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xo[i] = (long)(rt.row0 + min(16 * i + l16, rows - 1)) * a.x_stride + 8 * g;
    f32x4 acc[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};

    // C chunks from k0, waves * 64 apart
    auto chunks = [&](int k0, auto count, auto full) {
        constexpr int C = decltype(count)::value;
        constexpr bool FULL = decltype(full)::value;
        uint4 fw[2 * C], fx[XP ? 1 : 2 * C][XP ? 1 : MT];
        float ff[XP ? 2 * C : 1][XP ? MT : 1][8];
#pragma unroll
        for (int c = 0; c < 2 * C; ++c) {
            const int kc = k0 + (c >> 1) * waves * 64 + (c & 1) * 32;
            fw[c] = piece16<GRAN, FULL>(w + kc, a.k - kc - 8 * g);
        }
#pragma unroll
        for (int c = 0; c < 2 * C; ++c) {
            const int kc = k0 + (c >> 1) * waves * 64 + (c & 1) * 32;
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if constexpr (XP)
                    piece32<GRAN, FULL>((const float*)a.x + xo[i] + kc, a.k - kc - 8 * g, ff[c][i]);
                else
                    fx[c][i] = piece16<GRAN, FULL>((const uint16_t*)a.x + xo[i] + kc, a.k - kc - 8 * g);
            }
        }
#pragma unroll
        for (int c = 0; c < 2 * C; ++c)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if constexpr (XP) {
                    alignas(16) uint16_t h[PL][8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        uint16_t one[PL];
                        split_bf16<PL>(ff[c][i][e], one);
#pragma unroll
                        for (int q = 0; q < PL; ++q) h[q][e] = one[q];
                    }
#pragma unroll
                    for (int q = 0; q < PL; ++q) acc[i] = mfma<T>(fw[c], pack8_bf16(h[q]), acc[i]);
                } else {
                    acc[i] = mfma<T>(fw[c], fx[c][i], acc[i]);
                }
            }
    };
    int k0 = wave * 64;
    const int step = waves * 64;
    for (; k0 + (U - 1) * step + 64 <= a.k; k0 += U * step)
        chunks(k0, std::integral_constant<int, U>{}, std::true_type{});
    for (; k0 + 64 <= a.k; k0 += step) chunks(k0, std::integral_constant<int, 1>{}, std::true_type{});
    if (k0 < a.k) chunks(k0, std::integral_constant<int, 1>{}, std::false_type{});

    // accumulator register r: column 4 g + r of row l16
#pragma unroll
    for (int i = 0; i < MT; ++i)
        *reinterpret_cast<f32x4*>(&sums[wave][(i * 16 + l16) * 16 + 4 * g]) = acc[i];
    __syncthreads();
    for (int o = threadIdx.x; o < rows * 16; o += blockDim.x) {
        const int col = col0 + (o & 15);
        if (col >= a.n) continue;
        const long row = rt.row0 + (o >> 4);
        float v = sums[0][o];
        for (int s = 1; s < waves; ++s) v += sums[s][o];
        if (a.bias) v += a.bias[(long)rt.group * a.n + col];
        v = activate(v, a.act);
        if (a.res) v += load1(a.res, row * a.res_stride + col, a.y_kind);
        store1(a.y, row * a.y_stride + col, v, a.y_kind);
    }
}

// Any strides, alignment, n and k; fp32 activations.  Block tile 128x128,
// k-step 32, four waves in a 2x2 grid of 64x64, both operands through registers
// into double-buffered LDS.  XP: bf16 planes that stand for an fp32 x (0: x is of
// the weight's type).  GRAN: elements loaded at once, 4 where rows allow it, or 1.
template <int T, int XP, int GRAN, int YK, bool WHOLE>
__global__ __launch_bounds__(256, 2) void matmul_any_kernel(MatmulArgs a, int ntiles) {
    constexpr int BM = 128, BN = 128, BK = 32, P = BK + 8, PL = XP ? XP : 1;
    __shared__ __attribute__((aligned(16))) uint16_t x_lds[2][PL][BM * P];
    __shared__ __attribute__((aligned(16))) uint16_t w_lds[2][BN * P];
    const int lid = xcd_remap(blockIdx.x, gridDim.x);
    const RowTile rt = row_tile(a, lid / ntiles, BM);
    const int col0 = lid % ntiles * BN;
    const int rows = min(rt.end - rt.row0, BM);
    if (rows <= 0) return;   // the whole workgroup
    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int l16 = lane & 15;
    const int g = lane >> 4;
    const int wm = tid >> 7;
    const int wn = (tid >> 6) & 1;
    const uint16_t* w = (const uint16_t*)a.w + (long)rt.group * a.n * a.k;

    // thread -> (LDS row, quarter of 8 k) twice per operand
    float xf[XP ? 2 : 1][8];
    alignas(16) uint16_t xr[2][8], wr[2][8];
    auto load = [&](int k0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = (tid >> 2) + 64 * c;
            const int kc = k0 + (tid & 3) * 8;
            const int col = col0 + (r & ~63) + 4 * (r & 15) + ((r >> 4) & 3);
            const bool xin = r < rows, win = col < a.n;
            const long xo = (long)(rt.row0 + r) * a.x_stride + kc;
            const long wo = (long)col * a.k + kc;
#pragma unroll
            for (int e = 0; e < 8; e += GRAN) {
                const bool kin = kc + e < a.k;
                if constexpr (GRAN == 4) {
                    uint2 q = make_uint2(0, 0);
                    if (win && kin) q = *reinterpret_cast<const uint2*>(w + wo + e);
                    *reinterpret_cast<uint2*>(&wr[c][e]) = q;
                    if constexpr (XP) {
                        f32x4 q4 = {0.f, 0.f, 0.f, 0.f};
                        if (xin && kin) q4 = *reinterpret_cast<const f32x4*>((const float*)a.x + xo + e);
#pragma unroll
                        for (int i = 0; i < 4; ++i) xf[c][e + i] = q4[i];
                    } else {
                        q = make_uint2(0, 0);
                        if (xin && kin) q = *reinterpret_cast<const uint2*>((const uint16_t*)a.x + xo + e);
                        *reinterpret_cast<uint2*>(&xr[c][e]) = q;
                    }
                } else {
                    wr[c][e] = win && kin ? w[wo + e] : (uint16_t)0;
                    if constexpr (XP)
                        xf[c][e] = xin && kin ? ((const float*)a.x)[xo + e] : 0.f;
                    else
                        xr[c][e] = xin && kin ? ((const uint16_t*)a.x)[xo + e] : (uint16_t)0;
                }
            }
        }
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = (tid >> 2) + 64 * c;
            const int at = r * P + (tid & 3) * 8;
            *reinterpret_cast<uint4*>(&w_lds[buf][at]) = pack8_bf16(wr[c]);
            if constexpr (XP) {
                uint16_t h[PL][8];
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    uint16_t one[PL];
                    split_bf16<PL>(xf[c][e], one);
#pragma unroll
                    for (int i = 0; i < PL; ++i) h[i][e] = one[i];
                }
#pragma unroll
                for (int i = 0; i < PL; ++i)
                    *reinterpret_cast<uint4*>(&x_lds[buf][i][at]) = pack8_bf16(h[i]);
            } else {
                *reinterpret_cast<uint4*>(&x_lds[buf][0][at]) = pack8_bf16(xr[c]);
            }
        }
    };

    f32x4 acc[4][4];   // [row tile][column tile]
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int nk = (a.k + BK - 1) / BK;
    load(0);
    put(0);
    __syncthreads();
#pragma unroll 1
    for (int kt = 0; kt < nk; ++kt) {
        const int buf = kt & 1;
        if (kt + 1 < nk) load((kt + 1) * BK);
        uint4 fw[4];
#pragma unroll
        for (int j = 0; j < 4; ++j)
            fw[j] = *reinterpret_cast<const uint4*>(&w_lds[buf][(wn * 64 + 16 * j + l16) * P + 8 * g]);
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int q = 0; q < PL; ++q) {
                const uint4 fx = *reinterpret_cast<const uint4*>(
                    &x_lds[buf][q][(wm * 64 + 16 * i + l16) * P + 8 * g]);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = mfma<T>(fx, fw[j], acc[i][j]);
            }
        if (kt + 1 < nk) put(buf ^ 1);
        __syncthreads();
    }
    epilogue<YK, 4, WHOLE>(a, rt, rows, wm * 64, col0 + wn * 64 + 4 * l16, acc);
}

// 16-bit operands in 16-byte rows (k % 8 == 0), outputs in whole pieces.
//
// Block tile (128 * GROUPS) x (64 * WN): waves of 128x64 (SUB = 8 row tiles) or
// 64x64 (SUB = 4), fed from two LDS stages of 64 k that buffer_load ... lds fills
// (no VGPR staging); descriptors end with the tile's rows and the weight's, and a
// lane whose 16 bytes lie past k reads past the descriptor's end, so ragged m, n and
// k read zeros.
//
// parts > 1: a tile's k steps are dealt to `parts` workgroups, whose fp32
// accumulators go to partial[part][m][n]; matmul_sum_kernel adds them and does the
// epilogue.  For few tiles and long k.
struct TileSplit {
    int ntiles, mtiles;
    int parts;
    float* partial;
};

constexpr int kBK = 64;

// One operand's DMA: 64 LDS rows of 128 bytes in eight instructions of eight rows.
struct TileLoad {
    i32x4 rsrc;
    uint32_t vo[2];     // byte offsets of the lane's chunk in even and odd instructions
    uint32_t past[2];   // set in the last k step where the lane's chunk lies past k
};

// x: LDS row r is row r.  weight: LDS row 16 j + c is row 4 c + j.
template <bool WEIGHT>
__device__ __forceinline__ TileLoad tile_load(const uint16_t* base, int rows, long ld, int k,
                                              int row0) {
    const int lane = threadIdx.x & 63;
    const int l8 = lane >> 3;
    TileLoad t;
    const long bytes = rows > 0 ? ((long)(rows - 1) * ld + k) * 2 : 0;
    t.rsrc = wave_uniform(buffer_rsrc(base, (uint32_t)bytes));
    const int sw = lds_swizzle(l8);   // rows 8 apart differ in bit 2
    const int rem = k % kBK;
#pragma unroll
    for (int o = 0; o < 2; ++o) {
        const int c = (lane & 7) ^ sw ^ (4 * o);
        const int row = WEIGHT ? row0 + 4 * l8 + 32 * o : row0 + l8 + 8 * o;
        t.vo[o] = (uint32_t)((long)row * ld * 2) + c * 16;
        t.past[o] = rem && c * 8 >= rem ? 0x80000000u : 0u;
    }
    return t;
}

template <bool WEIGHT>
__device__ __forceinline__ void tile_issue(const TileLoad& t, uint32_t lds_addr, int kt, bool last,
                                           long ld) {
    const uint32_t soff = __builtin_amdgcn_readfirstlane((uint32_t)(kt * kBK * 2));
#pragma unroll
    for (int j = 0; j < 8; ++j) {
        const uint32_t rows = (WEIGHT ? j >> 1 : 16 * (j >> 1)) * (uint32_t)(ld * 2);
        uint32_t vo = t.vo[j & 1] + rows;
        if (last) vo |= t.past[j & 1];
        lds_dma16(t.rsrc, __builtin_amdgcn_readfirstlane(lds_addr + j * 1024), vo, soff);
    }
}

__device__ __forceinline__ void block_barrier() {
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_barrier" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
}

// The workgroup's tile and k steps.
struct TilePlace {
    RowTile rt;
    int rows, col0, part, kb, ke;
};

__device__ __forceinline__ TilePlace tile_place(const MatmulArgs& a, const TileSplit& sp, int bm,
                                                int bn) {
    // consecutive tiles share an XCD's L2; four row tiles sweep the columns together
    constexpr int GROUP = 4;
    const int lid = xcd_remap(blockIdx.x, gridDim.x);
    TilePlace p;
    p.part = lid % sp.parts;
    const int t = lid / sp.parts;
    const int first = t / (GROUP * sp.ntiles) * GROUP;
    const int gm = min(sp.mtiles - first, GROUP);
    const int in = t % (GROUP * sp.ntiles);
    p.rt = row_tile(a, first + in % gm, bm);
    p.rows = min(p.rt.end - p.rt.row0, bm);
    p.col0 = in / gm * bn;
    const int nk = (a.k + kBK - 1) / kBK;
    p.kb = (int)((long)nk * p.part / sp.parts);
    p.ke = (int)((long)nk * (p.part + 1) / sp.parts);
    return p;
}

// A wave's accumulators to the epilogue, or to its part's sums.
template <int YK, int NI>
__device__ __forceinline__ void tile_end(const MatmulArgs& a, const TileSplit& sp, const TilePlace& p,
                                         int row_w, int col, const f32x4 (&acc)[NI][4]) {
    if (sp.parts == 1) {
        epilogue<YK, NI, true>(a, p.rt, p.rows, row_w, col, acc);
        return;
    }
    if (col >= a.n) return;
    const int g = (threadIdx.x & 63) >> 4;
    float* out = sp.partial + ((long)p.part * a.m + p.rt.row0) * a.n + col;
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int row = row_w + 16 * i + 4 * g + r;
            if (row < p.rows)
                *reinterpret_cast<f32x4*>(out + (long)row * a.n) =
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
    const int nk = (a.k + kBK - 1) / kBK;
    const bool ragged = a.k % kBK != 0;
    const long ldw = a.k;
    // group 0 loads x, group 1 the weight
    TileLoad t;
    if (grp == 0)
        t = tile_load<false>((const uint16_t*)a.x + p.rt.row0 * a.x_stride, p.rows, a.x_stride, a.k,
                             wq * 64);
    else
        t = tile_load<true>((const uint16_t*)a.w + ((long)p.rt.group * a.n + p.col0) * ldw,
                            min(a.n - p.col0, 256), ldw, a.k, wq * 64);
    t.rsrc = wave_uniform(t.rsrc);
    const uint32_t mine = base + grp * TB + wq * 8 * 1024;
    auto issue = [&](int stage, int kt) {
        const bool last = ragged && kt + 1 == nk;
        if (grp == 0)
            tile_issue<false>(t, mine + stage * SB, kt, last, a.x_stride);
        else
            tile_issue<true>(t, mine + stage * SB, kt, last, ldw);
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
    tile_end<YK, 8>(a, sp, p, grp * 128, p.col0 + wq * 64 + 4 * l16, acc);
}

// 128x128 tile, four waves (2 x 2) of 64x64, two workgroups per compute unit: each
// one's loads and barriers pass under the other's MFMAs.
template <int T, int YK>
__global__ __launch_bounds__(256, 2) void matmul_128_kernel(MatmulArgs a, TileSplit sp) {
    constexpr int TB = 128 * kBK * 2, SB = 2 * TB, RB = kBK * 2;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[2 * SB];
    const TilePlace p = tile_place(a, sp, 128, 128);
    if (p.rows <= 0) return;   // the whole workgroup
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int wm = wave >> 1, wn = wave & 1;
    const int sw = lds_swizzle(l16);
    const uint32_t base = (uint32_t)(uintptr_t)lds;
    const int nk = (a.k + kBK - 1) / kBK;
    const bool ragged = a.k % kBK != 0;
    const long ldw = a.k;
    // waves 0 and 1 load x, 2 and 3 the weight, 64 rows each
    TileLoad t;
    if (wave < 2)
        t = tile_load<false>((const uint16_t*)a.x + p.rt.row0 * a.x_stride, p.rows, a.x_stride, a.k,
                             wave * 64);
    else
        t = tile_load<true>((const uint16_t*)a.w + ((long)p.rt.group * a.n + p.col0) * ldw,
                            min(a.n - p.col0, 128), ldw, a.k, (wave & 1) * 64);
    t.rsrc = wave_uniform(t.rsrc);
    const uint32_t mine = base + wave * 8 * 1024;
    auto issue = [&](int stage, int kt) {
        const bool last = ragged && kt + 1 == nk;
        if (wave < 2)
            tile_issue<false>(t, mine + stage * SB, kt, last, a.x_stride);
        else
            tile_issue<true>(t, mine + stage * SB, kt, last, ldw);
    };
    f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    const int steps = p.ke - p.kb;
    issue(0, p.kb);
#pragma unroll 1
    for (int s = 0; s < steps; ++s) {
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");   // step s
        block_barrier();                                   // and no one reads step s - 1
        if (s + 1 < steps) issue((s + 1) & 1, p.kb + s + 1);
        const uint8_t* st = lds + (s & 1) * SB;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const int pc = ((4 * kk + g) ^ sw) * 16;
            uint4 fx[4], fw[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
                fx[i] = *(const uint4*)(st + (wm * 64 + 16 * i + l16) * RB + pc);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                fw[j] = *(const uint4*)(st + TB + (wn * 64 + 16 * j + l16) * RB + pc);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = mfma<T>(fx[i], fw[j], acc[i][j]);
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    }
    tile_end<YK, 4>(a, sp, p, wm * 64, p.col0 + wn * 64 + 4 * l16, acc);
}

// y = residual + act(sum of the parts + bias), four columns a thread, parts in order.
template <int YK>
__global__ __launch_bounds__(256) void matmul_sum_kernel(MatmulArgs a, TileSplit sp) {
    const int quads = a.n / 4;
    const long all = (long)a.m * quads;
    for (long q = (long)blockIdx.x * 256 + threadIdx.x; q < all; q += (long)gridDim.x * 256) {
        const long row = q / quads;
        const int col = (int)(q - row * quads) * 4;
        const float* src = sp.partial + row * a.n + col;
        f32x4 v = *reinterpret_cast<const f32x4*>(src);
#pragma unroll 4
        for (int i = 1; i < sp.parts; ++i)
            v += *reinterpret_cast<const f32x4*>(src + (long)i * a.m * a.n);
        if (a.bias) v += *reinterpret_cast<const f32x4*>(a.bias + col);
#pragma unroll
        for (int j = 0; j < 4; ++j) v[j] = activate(v[j], a.act);
        if (a.res)
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] += load1(a.res, row * a.res_stride + col + j, YK);
        store4(a.y, row * a.y_stride + col, v[0], v[1], v[2], v[3], YK);
    }
}

template <int T, int XP, int YK>
hipError_t launch_any(const MatmulArgs& a, hipStream_t stream) {
    const int ntiles = (a.n + 127) / 128;
    const long blocks = row_tiles(a, 128) * ntiles;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    const bool four = a.k % 4 == 0 && a.x_stride % 4 == 0 && (uintptr_t)a.x % (XP ? 16 : 8) == 0 &&
                      (uintptr_t)a.w % 8 == 0;
    const bool whole = whole_pieces(a);
    const unsigned nb = (unsigned)blocks;
    if (four && whole)
        matmul_any_kernel<T, XP, 4, YK, true><<<nb, 256, 0, stream>>>(a, ntiles);
    else if (four)
        matmul_any_kernel<T, XP, 4, YK, false><<<nb, 256, 0, stream>>>(a, ntiles);
    else if (whole)
        matmul_any_kernel<T, XP, 1, YK, true><<<nb, 256, 0, stream>>>(a, ntiles);
    else
        matmul_any_kernel<T, XP, 1, YK, false><<<nb, 256, 0, stream>>>(a, ntiles);
    return hipGetLastError();
}

// Whether the tile kernels take a call: 16-byte rows of 16-bit x and weight, whole
// pieces of y, and tiles within the descriptors' 32-bit offsets.
bool tiles_take(const MatmulArgs& a) {
    return a.x_kind == a.w_kind && a.k % 8 == 0 && a.x_stride % 8 == 0 && (uintptr_t)a.x % 16 == 0 &&
           (uintptr_t)a.w % 16 == 0 && whole_pieces(a) && 256 * a.x_stride * 2 < 0x7fffffffL &&
           256L * a.k * 2 < 0x7fffffffL;
}

constexpr int kUnits = 256;   // compute units of an MI355X

struct TilePlan {
    int bm;      // 256 or 128, rows and columns of a tile
    int parts;
};

// The 256 tile where its tiles keep at least three quarters of the compute units busy.
// Else 128 tiles, split along k where they fill under half of the places (two a compute
// unit) and the workspace holds the parts' sums, into parts of 256 k or more.
TilePlan plan_tiles(const MatmulArgs& a, size_t workspace_bytes) {
    const long big = row_tiles(a, 256) * ((a.n + 255) / 256);
    if (big >= kUnits * 3 / 4) return TilePlan{256, 1};
    const long tiles = row_tiles(a, 128) * ((a.n + 127) / 128);
    long parts = 1;
    if (!a.offsets && tiles * 2 <= 2 * kUnits) {
        parts = std::min<long>({2 * kUnits / tiles, a.k / 256, 16});
        const size_t each = (size_t)a.m * a.n * sizeof(float);
        parts = std::min<long>(parts, (long)(workspace_bytes / each));
    }
    return TilePlan{128, parts < 2 ? 1 : (int)parts};
}

template <int T, int YK>
hipError_t launch_tiles(const MatmulArgs& a, void* workspace, size_t workspace_bytes,
                        hipStream_t stream) {
    const TilePlan plan = plan_tiles(a, workspace_bytes);
    const long mtiles = row_tiles(a, plan.bm), ntiles = (a.n + plan.bm - 1) / plan.bm;
    const long blocks = mtiles * ntiles * plan.parts;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    const TileSplit sp{(int)ntiles, (int)mtiles, plan.parts, (float*)workspace};
    if (plan.bm == 256)
        matmul_256_kernel<T, YK><<<(unsigned)blocks, 512, 0, stream>>>(a, sp);
    else
        matmul_128_kernel<T, YK><<<(unsigned)blocks, 256, 0, stream>>>(a, sp);
    if (plan.parts > 1) {
        const long quads = (long)a.m * (a.n / 4);
        matmul_sum_kernel<YK><<<(unsigned)std::min<long>((quads + 255) / 256, 4096), 256, 0, stream>>>(
            a, sp);
    }
    return hipGetLastError();
}

// Elements that lie together in every row of x and of the weight.
int row_gran(const MatmulArgs& a) {
    for (int e : {8, 4})
        if (a.k % e == 0 && a.x_stride % e == 0 && (uintptr_t)a.w % (2 * e) == 0 &&
            (uintptr_t)a.x % (a.x_kind ? 2 * e : 16) == 0)
            return e;
    return 1;
}

template <int T, int XP, int MT>
hipError_t launch_rows_mt(const MatmulArgs& a, hipStream_t stream) {
    const int ntiles = (a.n + 15) / 16;
    const long blocks = row_tiles(a, 16 * MT) * ntiles;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    const int chunks = (a.k + 63) / 64;
    const int waves = std::min(8, std::max(1, chunks));
    const unsigned nb = (unsigned)blocks, nt = 64 * waves;
    const int gran = row_gran(a);
    if (gran == 8)
        matmul_rows_kernel<T, XP, MT, 8><<<nb, nt, 0, stream>>>(a, ntiles);
    else if (gran == 4)
        matmul_rows_kernel<T, XP, MT, 4><<<nb, nt, 0, stream>>>(a, ntiles);
    else
        matmul_rows_kernel<T, XP, MT, 1><<<nb, nt, 0, stream>>>(a, ntiles);
    return hipGetLastError();
}

template <int T, int XP>
hipError_t launch_rows(const MatmulArgs& a, int rows, hipStream_t stream) {
    if (rows <= 16) return launch_rows_mt<T, XP, 1>(a, stream);
    if (rows <= 32) return launch_rows_mt<T, XP, 2>(a, stream);
    return launch_rows_mt<T, XP, 4>(a, stream);
}

template <int YK>
hipError_t launch_y(const MatmulArgs& a, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    const int rows = a.offsets ? (a.m + a.groups - 1) / a.groups : a.m;   // of a group
    if (rows <= 64) {
        if (a.w_kind == 2) return launch_rows<2, 0>(a, rows, stream);
        if (a.x_kind == 1) return launch_rows<1, 0>(a, rows, stream);
        return launch_rows<1, YK == 0 ? 3 : 2>(a, rows, stream);
    }
    if (tiles_take(a))
        return a.w_kind == 2 ? launch_tiles<2, YK>(a, workspace, workspace_bytes, stream)
                             : launch_tiles<1, YK>(a, workspace, workspace_bytes, stream);
    if (a.w_kind == 2) return launch_any<2, 0, YK>(a, stream);
    if (a.x_kind == 0) return launch_any<1, YK == 0 ? 3 : 2, YK>(a, stream);
    return launch_any<1, 0, YK>(a, stream);
}

}  // namespace

size_t matmul_workspace(int m, int n, int k, int x_kind) {
    if (m <= 0 || x_kind == 0) return 0;
    MatmulArgs a{};
    a.m = m;
    a.n = n;
    a.k = k;
    a.groups = 1;
    if (m <= 64) return 0;
    const int parts = plan_tiles(a, ~(size_t)0).parts;
    return parts > 1 ? (size_t)parts * m * n * sizeof(float) : 0;
}

hipError_t launch_matmul(const MatmulArgs& args, void* workspace, size_t workspace_bytes,
                         hipStream_t stream) {
    if (args.m <= 0) return hipSuccess;
    MatmulArgs a = args;
    if (a.m == 1) {   // the strides of a single row say nothing
        a.x_stride = a.k;
        a.res_stride = a.y_stride = a.n;
    }
    return a.y_kind == 0   ? launch_y<0>(a, workspace, workspace_bytes, stream)
           : a.y_kind == 1 ? launch_y<1>(a, workspace, workspace_bytes, stream)
                           : launch_y<2>(a, workspace, workspace_bytes, stream);
}

}  // namespace s2
