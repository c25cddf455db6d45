// Products with weights in MXFP4: y = residual + act(x W^T + bias).
//
// This file: which kernel takes a call, and the kernel for few rows.
#include "mx_device.h"

namespace s2 {

namespace {

// x as the matrix cores take it: codes (XT 0), or a sum of bf16 terms that holds it exactly
// (bf16: one, fp16: two, fp32: three) against weights as bf16, which hold a code times
// its scale exactly.
template <int XT>
constexpr int kXTerms = XT == 0 ? 1 : XT == S2_DTYPE_BF16 + 1 ? 1 : XT == S2_DTYPE_F16 + 1 ? 2 : 3;

// Up to 16 MT rows by 16 NT columns a workgroup of up to eight waves.  What costs is
// reading the weight: every wave takes every other 256 k (128 bytes of each weight row)
// straight into operand registers, the next ones in flight under the products; x comes
// from the caches.  The waves' sums meet in LDS.  Lane (row l16, group g) holds blocks 2 g
// and 2 g + 1 of the 256 k, of both operands; rows and columns past the end repeat the
// last one, and are dropped.  XT: 0 MXFP4, else 1 + x's kind.
template <int XT, int MT, int NT>
__global__ __launch_bounds__(512) void mx_rows_kernel(MxLinearArgs a, int ntiles) {
    constexpr int TERMS = kXTerms<XT>;
    __shared__ float sums[8][MT * NT * 256];
    const int row0 = blockIdx.x / ntiles * 16 * MT;
    const int col0 = blockIdx.x % ntiles * 16 * NT;
    const int rows = min(a.m - row0, 16 * MT);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int l16 = lane & 15, g = lane >> 4;
    const int blocks = mx_blocks(a.k);
    long wrow[NT], xrow[MT];
#pragma unroll
    for (int j = 0; j < NT; ++j) wrow[j] = min(col0 + 16 * j + l16, a.n - 1);
#pragma unroll
    for (int i = 0; i < MT; ++i) xrow[i] = row0 + min(16 * i + l16, rows - 1);
    f32x4 acc[MT][NT];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int j = 0; j < NT; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Part {   // of 256 k
        uint4 w[2][NT];
        uint32_t ws[2][NT];
        uint4 x[XT ? 1 : 2][XT ? 1 : MT];
        uint32_t xs[XT ? 1 : 2][XT ? 1 : MT];
    };
    auto load = [&](Part& p, int part) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int b = part * 8 + 2 * g + c;
            const bool in = b < blocks;   // past it: zeros
            const int at = in ? b : 0;
#pragma unroll
            for (int j = 0; j < NT; ++j) {
                p.w[c][j] = *reinterpret_cast<const uint4*>(a.w.codes + wrow[j] * a.w.code_stride + 16 * at);
                p.ws[c][j] = a.w.scales[wrow[j] * a.w.scale_stride + at];
                if (!in) p.w[c][j] = make_uint4(0, 0, 0, 0), p.ws[c][j] = 127;
            }
            if constexpr (XT == 0)
#pragma unroll
                for (int i = 0; i < MT; ++i) {
                    p.x[c][i] =
                        *reinterpret_cast<const uint4*>(a.xq.codes + xrow[i] * a.xq.code_stride + 16 * at);
                    p.xs[c][i] = a.xq.scales[xrow[i] * a.xq.scale_stride + at];
                    if (!in) p.x[c][i] = make_uint4(0, 0, 0, 0), p.xs[c][i] = 127;
                }
        }
    };
    auto use = [&](const Part& p, int part) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if constexpr (XT == 0) {
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int j = 0; j < NT; ++j)
                        acc[i][j] = mx_mfma<0, 0>(p.w[c][j], p.x[c][i], acc[i][j], p.ws[c][j], p.xs[c][i]);
            } else {
                const int k0 = (part * 8 + 2 * g + c) * 32;
#pragma unroll
                for (int e = 0; e < 4; ++e) {   // eight k
                    uint4 w[NT];
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const uint32_t q[4] = {p.w[c][j].x, p.w[c][j].y, p.w[c][j].z, p.w[c][j].w};
                        w[j] = mx_bf16(q[e], mx_scale(p.ws[c][j]));
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        uint4 t[TERMS];
                        mx_terms<XT - 1, TERMS>(a.x, xrow[i] * a.x_stride + k0 + 8 * e, a.k - k0 - 8 * e, t);
#pragma unroll
                        for (int q = 0; q < TERMS; ++q)
#pragma unroll
                            for (int j = 0; j < NT; ++j) acc[i][j] = mfma<1>(w[j], t[q], acc[i][j]);
                    }
                }
            }
        }
    };
    const int parts = (blocks + 7) / 8;
    Part p0, p1;
    int part = wave;
    if (part < parts) load(p0, part);
    while (part < parts) {
        if (part + waves < parts) load(p1, part + waves);
        use(p0, part);
        part += waves;
        if (part >= parts) break;
        if (part + waves < parts) load(p0, part + waves);
        use(p1, part);
        part += waves;
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
        const long row = row0 + o / (16 * NT);
        float v = sums[0][o];
        for (int s = 1; s < waves; ++s) v += sums[s][o];
        if (a.bias) v += a.bias[col];
        v = a.y_kind ? activate<false>(v, a.act) : activate<true>(v, a.act);
        if (a.res) v += load1(a.res, row * a.res_stride + col, a.y_kind);
        store1(a.y, row * a.y_stride + col, v, a.y_kind);
    }
}

template <int XT, int MT, int NT>
hipError_t run_rows(const MxLinearArgs& a, hipStream_t stream) {
    const int ntiles = (a.n + 16 * NT - 1) / (16 * NT);
    const long blocks = ((long)a.m + 16 * MT - 1) / (16 * MT) * ntiles;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    const int waves = std::min(8, (mx_blocks(a.k) + 7) / 8);
    mx_rows_kernel<XT, MT, NT><<<(unsigned)blocks, 64 * waves, 0, stream>>>(a, ntiles);
    return hipGetLastError();
}

template <int XT>
hipError_t launch_rows(const MxLinearArgs& a, hipStream_t stream) {
    return a.m <= 16 ? run_rows<XT, 1, 2>(a, stream) : run_rows<XT, 2, 2>(a, stream);
}

}  // namespace

size_t mx_linear_workspace(const MxLinearArgs&) { return 0; }

hipError_t launch_mx_linear(const MxLinearArgs& args, void*, size_t, hipStream_t stream) {
    if (args.m <= 0) return hipSuccess;
    MxLinearArgs a = args;
    if (a.m == 1) {   // the strides of a single row say nothing
        a.x_stride = a.k;
        a.res_stride = a.y_stride = a.n;
        a.xq.code_stride = 16L * mx_blocks(a.k);
        a.xq.scale_stride = mx_blocks(a.k);
    }
    if (a.mx) return launch_rows<0>(a, stream);
    return a.x_kind == 0   ? launch_rows<1>(a, stream)
           : a.x_kind == 1 ? launch_rows<2>(a, stream)
                           : launch_rows<3>(a, stream);
}

}  // namespace s2
