// Matrix products with bias, activation and residual in the epilogue, over all
// rows (s2_linear) or over ragged row groups with a weight each
// (s2_grouped_linear):  y = residual + act(x W^T + bias).
//
// x [m][k] and W [n][k] are both k-contiguous, the operand layout of the 16-bit
// MFMAs.  W is the MFMA's first operand, x its second, so that a lane's
// accumulators are columns of one row of y; and row 4 g + r of the accumulator of
// column tile j stands for column 16 g + 4 j + r of a wave's 64, so that they
// are 16 neighbours: the epilogue works on whole 16-byte pieces of y and of the
// residual straight from the registers, with one rounding at the end.
#include "matmul_kernels.h"

#include <algorithm>

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

// Whether 16-byte pieces of y, the residual and the bias can be moved whole.
__device__ __forceinline__ bool vector_ends(const MatmulArgs& a) {
    const int e = a.y_kind ? 8 : 4;
    return ((uintptr_t)a.y | (uintptr_t)a.res | (uintptr_t)a.bias) % 16 == 0 &&
           a.y_stride % e == 0 && (!a.res || a.res_stride % e == 0) && a.n % 4 == 0;
}

// 16 columns of one row, from column col: bias, activation, residual, rounding.
__device__ __forceinline__ void finish16(const MatmulArgs& a, int group, long row, int col,
                                         float (&v)[16], bool whole) {
    const float* bias = a.bias ? a.bias + (long)group * a.n + col : nullptr;
    if (whole && col + 16 <= a.n) {
        if (bias) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const f32x4 b = *reinterpret_cast<const f32x4*>(bias + 4 * j);
#pragma unroll
                for (int r = 0; r < 4; ++r) v[4 * j + r] += b[r];
            }
        }
        if (a.act != S2_ACT_NONE)
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = activate(v[e], a.act);
        const long at = row * a.y_stride + col;
        if (a.res) {
            const long rt = row * a.res_stride + col;
            if (a.y_kind == 0) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const f32x4 b = *reinterpret_cast<const f32x4*>((const float*)a.res + rt + 4 * j);
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[4 * j + r] += b[r];
                }
            } else {
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    const uint4 raw = *reinterpret_cast<const uint4*>((const uint16_t*)a.res + rt + 8 * h);
                    const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        const uint16_t b = (uint16_t)(w[e >> 1] >> (16 * (e & 1)));
                        v[8 * h + e] += a.y_kind == 1 ? bf16_to_f32(b)
                                                      : (float)__builtin_bit_cast(_Float16, b);
                    }
                }
            }
        }
        if (a.y_kind == 0) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f32x4*>((float*)a.y + at + 4 * j) =
                    f32x4{v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]};
        } else {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                uint32_t w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    w[e] = a.y_kind == 1 ? pack2_bf16_rne(v[8 * h + 2 * e], v[8 * h + 2 * e + 1])
                                         : pack2_f16_rne(v[8 * h + 2 * e], v[8 * h + 2 * e + 1]);
                *reinterpret_cast<uint4*>((uint16_t*)a.y + at + 8 * h) =
                    make_uint4(w[0], w[1], w[2], w[3]);
            }
        }
    } else {
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            if (col + e < a.n) {
                float u = activate(v[e] + (bias ? bias[e] : 0.f), a.act);
                if (a.res) u += load1(a.res, row * a.res_stride + col + e, a.y_kind);
                store1(a.y, row * a.y_stride + col + e, u, a.y_kind);
            }
        }
    }
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

// Any strides, alignment, n and k; fp32 activations.  Block tile 128x128,
// k-step 32, four waves in a 2x2 grid of 64x64, both operands through registers
// into double-buffered LDS.  XP: bf16 planes that stand for an fp32 x (0: x is of
// the weight's type).  GRAN: elements loaded at once, 4 where rows allow it, or 1.
template <int T, int XP, int GRAN>
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

    // thread -> (LDS row, quarter of 8 k) twice per operand; LDS row 16 j + 4 g + r
    // of a wave's weight rows holds column 16 g + 4 j + r
    float xf[XP ? 2 : 1][8];
    alignas(16) uint16_t xr[2][8], wr[2][8];
    auto load = [&](int k0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = (tid >> 2) + 64 * c;
            const int kc = k0 + (tid & 3) * 8;
            const int col = col0 + (r & ~63) + 16 * ((r >> 2) & 3) + 4 * ((r >> 4) & 3) + (r & 3);
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
                for (int j = 0; j < 4; ++j) acc[i][j] = mfma<T>(fw[j], fx, acc[i][j]);
            }
        if (kt + 1 < nk) put(buf ^ 1);
        __syncthreads();
    }
    const bool whole = vector_ends(a);
    const int col = col0 + wn * 64 + 16 * g;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int r = wm * 64 + 16 * i + l16;
        float v[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) v[e] = acc[i][e >> 2][e & 3];
        if (r < rows && col < a.n) finish16(a, rt.group, rt.row0 + r, col, v, whole);
    }
}

template <int T, int XP>
hipError_t launch_any(const MatmulArgs& a, hipStream_t stream) {
    const int ntiles = (a.n + 127) / 128;
    const long blocks = row_tiles(a, 128) * ntiles;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    const size_t xe = XP ? 16 : 8;
    const bool four = a.k % 4 == 0 && a.x_stride % 4 == 0 && (uintptr_t)a.x % xe == 0 &&
                      (uintptr_t)a.w % 8 == 0;
    if (four)
        matmul_any_kernel<T, XP, 4><<<(unsigned)blocks, 256, 0, stream>>>(a, ntiles);
    else
        matmul_any_kernel<T, XP, 1><<<(unsigned)blocks, 256, 0, stream>>>(a, ntiles);
    return hipGetLastError();
}

}  // namespace

size_t matmul_workspace(int, int, int, int) { return 0; }

hipError_t launch_matmul(const MatmulArgs& a, void*, size_t, hipStream_t stream) {
    if (a.m <= 0) return hipSuccess;
    if (a.w_kind == 2) return launch_any<2, 0>(a, stream);
    if (a.x_kind == 0) return a.y_kind == 0 ? launch_any<1, 3>(a, stream) : launch_any<1, 2>(a, stream);
    return launch_any<1, 0>(a, stream);
}

}  // namespace s2
