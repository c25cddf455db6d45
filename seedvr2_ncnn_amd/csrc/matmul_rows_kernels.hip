// Linear and grouped linear over few rows.
#include "matmul_device.h"

namespace s2 {

namespace {

// Up to 16 MT rows by 16 NT columns a workgroup of up to eight waves.  What costs is
// reading the weight: every wave takes every other 64 k (128 bytes of each weight row)
// straight into the MFMAs' operand registers, the next loads in flight under the MFMAs;
// x comes from the caches.  The waves' sums meet in LDS.  Rows and columns past the end
// repeat the last one, and are dropped.
//
// SPLIT: an fp32 x as bf16 terms, by every workgroup; else x is of the weight's type.
template <int T, bool SPLIT, int MT, int NT, bool ODD>
__global__ __launch_bounds__(512) void matmul_rows_kernel(MatmulArgs a, int ntiles) {
    constexpr int PL = SPLIT ? kTerms : 1;
    constexpr int REGS = 2 * 4 * (NT + MT * (SPLIT ? 2 : 1));   // of a 64-k chunk
    constexpr int U = REGS >= 40 ? 1 : REGS >= 24 ? 2 : 4;  // chunks of a batch
    constexpr bool TWO = U * REGS <= 80;                    // the next batch in flight
    __shared__ float sums[8][MT * NT * 256];
    const RowTile rt = RowTiles(a, 16 * MT, gridDim.x / ntiles).at(blockIdx.x / ntiles);
    const int col0 = blockIdx.x % ntiles * 16 * NT;
    const int rows = min(rt.end - rt.row0, 16 * MT);
    if (rows <= 0) return;   // the whole workgroup
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int l16 = lane & 15, g = lane >> 4;
    const uint16_t* w[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j)
        w[j] = (const uint16_t*)a.w +
               ((long)rt.group * a.n + min(col0 + 16 * j + l16, a.n - 1)) * a.k + 8 * g;
    long xo[MT];
#pragma unroll
    for (int i = 0; i < MT; ++i) xo[i] = (long)(rt.row0 + min(16 * i + l16, rows - 1)) * a.x_stride + 8 * g;
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // C chunks of 64 k, waves * 64 apart
    struct Batch {
        uint4 w[2 * U][NT];
        uint4 x[SPLIT ? 1 : 2 * U][SPLIT ? 1 : MT];
        float f[SPLIT ? 2 * U : 1][SPLIT ? MT : 1][8];
    };
    auto load = [&](Batch& b, int k0, auto count, auto full) {
        constexpr int C = decltype(count)::value;
        constexpr bool FULL = decltype(full)::value;
#pragma unroll
        for (int c = 0; c < 2 * C; ++c) {
            const int kc = k0 + (c >> 1) * waves * 64 + (c & 1) * 32;
            const int left = a.k - kc - 8 * g;
#pragma unroll
            for (int j = 0; j < NT; ++j) b.w[c][j] = piece16<FULL, ODD>(w[j] + kc, left);
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                if constexpr (SPLIT)
                    piece32<FULL>((const float*)a.x + xo[i] + kc, left, b.f[c][i]);
                else
                    b.x[c][i] = piece16<FULL, ODD>((const uint16_t*)a.x + xo[i] + kc, left);
            }
        }
    };
    auto use = [&](const Batch& b, auto count) {
        constexpr int C = decltype(count)::value;
#pragma unroll
        for (int c = 0; c < 2 * C; ++c)
#pragma unroll
            for (int i = 0; i < MT; ++i) {
                uint4 t[PL];
                if constexpr (SPLIT)
                    split8(b.f[c][i], t);
                else
                    t[0] = b.x[c][i];
#pragma unroll
                for (int q = 0; q < PL; ++q)
#pragma unroll
                    for (int j = 0; j < NT; ++j) acc[i][j] = mfma<T>(b.w[c][j], t[q], acc[i][j]);
            }
    };
    typedef std::integral_constant<int, U> Many;
    typedef std::integral_constant<int, 1> One;
    const int step = waves * 64;
    const int reach = (U - 1) * step + 64;   // of a batch
    int k0 = wave * 64;
    Batch b0, b1;
    if constexpr (!TWO) {
        for (; k0 + reach <= a.k; k0 += U * step) {
            load(b0, k0, Many{}, std::true_type{});
            use(b0, Many{});
        }
    } else if (k0 + reach <= a.k) {
        load(b0, k0, Many{}, std::true_type{});
        k0 += U * step;
        while (true) {
            const bool more = k0 + reach <= a.k;
            if (more) load(b1, k0, Many{}, std::true_type{});
            use(b0, Many{});
            if (!more) break;
            k0 += U * step;
            const bool again = k0 + reach <= a.k;
            if (again) load(b0, k0, Many{}, std::true_type{});
            use(b1, Many{});
            if (!again) break;
            k0 += U * step;
        }
    }
    for (; k0 + 64 <= a.k; k0 += step) {
        load(b0, k0, One{}, std::true_type{});
        use(b0, One{});
    }
    if (k0 < a.k) {
        load(b0, k0, One{}, std::false_type{});
        use(b0, One{});
    }

    // accumulator register r: column 4 g + r of row l16
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j)
            *reinterpret_cast<f32x4*>(&sums[wave][((i * 16 + l16) * NT + j) * 16 + 4 * g]) = acc[i][j];
    __syncthreads();
    for (int o = threadIdx.x; o < rows * 16 * NT; o += blockDim.x) {
        const int col = col0 + o % (16 * NT);
        if (col >= a.n) continue;
        const long row = rt.row0 + o / (16 * NT);
        float v = sums[0][o];
        for (int s = 1; s < waves; ++s) v += sums[s][o];
        if (a.bias) v += a.bias[(long)rt.group * a.n + col];
        v = a.y_kind ? activate<false>(v, a.act) : activate<true>(v, a.act);
        if (a.res) v += load1(a.res, row * a.res_stride + col, a.y_kind);
        store1(a.y, row * a.y_stride + col, v, a.y_kind);
    }
}

template <int T, bool SPLIT, int MT, int NT, bool ODD>
hipError_t run(const MatmulArgs& a, hipStream_t stream) {
    const int ntiles = (a.n + 16 * NT - 1) / (16 * NT);
    const long blocks = row_tiles(a, 16 * MT) * ntiles;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    const int waves = std::min(8, (a.k + 63) / 64);
    matmul_rows_kernel<T, SPLIT, MT, NT, ODD><<<(unsigned)blocks, 64 * waves, 0, stream>>>(a, ntiles);
    return hipGetLastError();
}

template <int T, bool SPLIT, int MT>
hipError_t pick(const MatmulArgs& a, int cols, hipStream_t stream) {
    constexpr int MOST = MT * (SPLIT ? kTerms : 1) <= 4 ? 4 : 2;   // by registers
    const bool odd = (a.k & 1) || (uintptr_t)a.w % 4 || (a.x_kind && ((a.x_stride & 1) || (uintptr_t)a.x % 4));
    if (odd) return run<T, SPLIT, MT, 1, true>(a, stream);
    if (cols == 64) return run<T, SPLIT, MT, MOST, false>(a, stream);
    return cols == 32 ? run<T, SPLIT, MT, 2, false>(a, stream) : run<T, SPLIT, MT, 1, false>(a, stream);
}

template <int T, bool SPLIT>
hipError_t pick_rows(const MatmulArgs& a, const MatmulPlan& plan, hipStream_t stream) {
    return plan.rows == 16   ? pick<T, SPLIT, 1>(a, plan.cols, stream)
           : plan.rows == 32 ? pick<T, SPLIT, 2>(a, plan.cols, stream)
                             : pick<T, SPLIT, 4>(a, plan.cols, stream);
}

}  // namespace

hipError_t launch_matmul_rows(const MatmulArgs& a, const MatmulPlan& plan, hipStream_t stream) {
    if (a.w_kind == 2) return pick_rows<2, false>(a, plan, stream);
    return a.x_kind ? pick_rows<1, false>(a, plan, stream) : pick_rows<1, true>(a, plan, stream);
}

}  // namespace s2
