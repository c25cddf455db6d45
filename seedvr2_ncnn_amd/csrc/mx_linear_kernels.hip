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

// Scales of x's and of the weight's rows to rows of `width` bytes, either of which may have
// none.
struct ScaleJob {
    const uint8_t* src;
    long stride, rows;
    uint8_t* dst;
};

__global__ __launch_bounds__(256) void mx_scales_kernel(ScaleJob x, ScaleJob w, int blocks, int width) {
    const long nx = x.rows * blocks, all = nx + w.rows * blocks;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) {
        const ScaleJob& job = i < nx ? x : w;
        const long at = i < nx ? i : i - nx;
        const long row = at / blocks;
        const int b = (int)(at - row * blocks);
        job.dst[row * width + b] = job.src[row * job.stride + b];
    }
}

long round_up(long v, long to) { return (v + to - 1) / to * to; }

// The weight's values as bf16 rows of k, for rows of x of other types.
size_t weight_bytes(const MxLinearArgs& a) { return round_up((size_t)a.n * a.k * 2, 256); }

MatmulArgs values_args(const MxLinearArgs& a, const void* w) {
    MatmulArgs m{};
    m.x = a.x;
    m.x_kind = a.x_kind;
    m.x_stride = a.x_stride;
    m.m = a.m;
    m.groups = 1;
    m.w = w;
    m.w_kind = S2_DTYPE_BF16;
    m.bias = a.bias;
    m.n = a.n;
    m.k = a.k;
    m.act = a.act;
    m.res = a.res;
    m.res_stride = a.res_stride;
    m.y = a.y;
    m.y_kind = a.y_kind;
    m.y_stride = a.y_stride;
    m.planes = 1;
    return m;
}

// The product with rows of codes as 16-bit elements.
MatmulArgs codes_args(const MxLinearArgs& a) {
    MatmulArgs m = values_args(a, a.w.codes);
    m.x = a.xq.codes;
    m.x_kind = S2_DTYPE_BF16;
    m.x_stride = a.xq.code_stride / 2;
    m.k = 8 * mx_blocks(a.k);
    return m;
}

constexpr int kRowsMost = 32;   // of x that the kernel for few rows takes

// Ranges of k, at most, whose sums fit `bytes`.
long ranges(const MxLinearArgs& a, size_t bytes) {
    return std::min<long>(16, (long)(bytes / ((size_t)a.m * round_up(a.n, 4) * sizeof(float))));
}

bool scales16(const uint8_t* s, long stride) { return (uintptr_t)s % 16 == 0 && stride % 16 == 0; }

// A product on tiles: what the scales take in the workspace (for 256 x 256 as they are
// dealt out, else rows that begin at no 16 bytes copied), then the sums.
struct MxPlan {
    TileChoice tile;
    size_t scales, sums;
    size_t bytes() const { return scales + sums; }
};

MxPlan mx_plan(const MxLinearArgs& a, bool pack_x, bool pack_w, size_t workspace_bytes) {
    const MatmulArgs m = codes_args(a);
    const int blocks = mx_blocks(a.k);
    const DealtBytes dealt = mx_dealt_bytes(a.m, a.n, blocks);
    const size_t copied = ((pack_x ? (size_t)a.m : 0) + (pack_w ? (size_t)a.n : 0)) * round_up(blocks, 16);
    MxPlan p{};
    for (int largest : {256, 128}) {
        const size_t least = round_up(largest == 256 ? dealt.x + dealt.w : copied, 256);
        if (least > workspace_bytes) continue;
        p.tile = choose_tiles(m, (m.k + 63) / 64, ranges(a, workspace_bytes - least), largest);
        p.scales = round_up(p.tile.bm == 256 ? dealt.x + dealt.w : copied, 256);
        p.sums = p.tile.parts > 1 ? (size_t)p.tile.parts * a.m * round_up(a.n, 4) * sizeof(float) : 0;
        if (p.bytes() <= workspace_bytes) return p;
    }
    p.tile.bm = 0;   // not on tiles
    return p;
}

}  // namespace

size_t mx_linear_workspace(const MxLinearArgs& a) {
    if (a.m <= kRowsMost) return 0;
    return mx_plan(a, true, true, (size_t)1 << 62).bytes();
}

hipError_t launch_mx_linear(const MxLinearArgs& args, void* workspace, size_t workspace_bytes,
                            hipStream_t stream) {
    if (args.m <= 0) return hipSuccess;
    MxLinearArgs a = args;
    const int blocks = mx_blocks(a.k);
    if (a.m == 1) {   // the strides of a single row say nothing
        a.x_stride = a.k;
        a.res_stride = a.y_stride = a.n;
        a.xq.code_stride = 16L * blocks;
        a.xq.scale_stride = round_up(blocks, 16);
    }
    if (a.n == 1) a.w.scale_stride = round_up(blocks, 16);
    if (!a.mx)
        return a.x_kind == 0   ? launch_rows<1>(a, stream)
               : a.x_kind == 1 ? launch_rows<2>(a, stream)
                               : launch_rows<3>(a, stream);
    const long out = std::max(a.y_stride, a.res ? a.res_stride : 0L) * (a.y_kind ? 2 : 4);
    const long far = 0x7fffffffL;   // 32-bit offsets
    const bool pack_x = !scales16(a.xq.scales, a.xq.scale_stride);
    const bool pack_w = !scales16(a.w.scales, a.w.scale_stride);
    MxPlan p{};
    if (a.m > kRowsMost && 256 * out < far && (long)a.n * 4 < far && 256 * a.xq.code_stride < far &&
        256 * 16L * blocks < far && 256 * std::max(a.xq.scale_stride, a.w.scale_stride) < far)
        p = mx_plan(a, pack_x, pack_w, workspace_bytes);
    if (p.tile.bm == 0) return launch_rows<0>(a, stream);
    MxTileScales sc{a.xq.scales, a.xq.scale_stride, a.w.scales, a.w.scale_stride, blocks};
    if (p.tile.bm < 256 && (pack_x || pack_w)) {
        const int width = (int)round_up(blocks, 16);
        uint8_t* at = (uint8_t*)workspace;
        const ScaleJob x{a.xq.scales, a.xq.scale_stride, pack_x ? a.m : 0, at};
        const ScaleJob w{a.w.scales, a.w.scale_stride, pack_w ? a.n : 0, at + (pack_x ? (size_t)a.m * width : 0)};
        const long all = (x.rows + w.rows) * blocks;
        mx_scales_kernel<<<(unsigned)std::min<long>((all + 255) / 256, 4096), 256, 0, stream>>>(x, w, blocks, width);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
        if (pack_x) sc.x = x.dst, sc.x_stride = width;
        if (pack_w) sc.w = w.dst, sc.w_stride = width;
    }
    return launch_mx_tiles(codes_args(a), sc, p.tile, (float*)((char*)workspace + p.scales), workspace, stream);
}

}  // namespace s2
