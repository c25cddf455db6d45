// Products with weights in MXFP4: y = residual + act(x W^T + bias).
//
// This file: which kernel takes a call, and the kernel for few rows.
#include "mx_device.h"

namespace s2 {

namespace {

// A block of x as it is loaded, and eight k of it as the matrix cores take them: codes (XT
// 0), or a sum of bf16 terms that holds it exactly (bf16: one, fp16: two, fp32: three, from 2^-110 on)
// against weights as bf16, which hold a code times its scale exactly.  XT: 0 MXFP4, else 1
// + x's kind.
template <int XT>
struct MxX {   // 16-bit rows
    static constexpr int TERMS = XT - 1;
    struct Block {
        uint4 v[4];
    };
    static __device__ __forceinline__ void load(const MxLinearArgs& a, long row, int block, bool, Block& x) {
        const uint16_t* p = (const uint16_t*)a.x + row * a.x_stride + 32L * block;
#pragma unroll
        for (int e = 0; e < 4; ++e) x.v[e] = piece16<false>(p + 8 * e, a.k - 32 * block - 8 * e);
    }
    static __device__ __forceinline__ void terms(uint4 v, uint4 (&t)[TERMS]) {
        if constexpr (TERMS == 1)
            t[0] = v;
        else
            mx_terms16(v, t);
    }
    // eight k from `at` on
    static __device__ __forceinline__ void terms_of(const MxLinearArgs& a, long row, int at, uint4 (&t)[TERMS]) {
        terms(piece16<false>((const uint16_t*)a.x + row * a.x_stride + at, a.k - at), t);
    }
};
template <>
struct MxX<0> {
    static constexpr int TERMS = 1;
    struct Block {
        uint4 codes;
        uint32_t scale;
    };
    static __device__ __forceinline__ void load(const MxLinearArgs& a, long row, int block, bool in, Block& x) {
        const int at = in ? block : 0;
        x.codes = *reinterpret_cast<const uint4*>(a.xq.codes + row * a.xq.code_stride + 16 * at);
        x.scale = a.xq.scales[row * a.xq.scale_stride + at];
        if (!in) x.codes = make_uint4(0, 0, 0, 0), x.scale = 127;
    }
};
template <>
struct MxX<1> {   // fp32, split by way of LDS alone
    static constexpr int TERMS = kTerms;
    struct Block {};
    static __device__ __forceinline__ void terms_of(const MxLinearArgs& a, long row, int at, uint4 (&t)[TERMS]) {
        float v[8];
        piece32<false>((const float*)a.x + row * a.x_stride + at, a.k - at, v);
        split8(v, t);
    }
};

// Up to 16 rows by 16 NT columns a workgroup of up to eight waves.  What costs is reading
// the weight: every wave takes every other 256 k (128 bytes of each weight row) straight
// into operand registers, the next ones in flight under the products.  Lane (row l16, group
// g) holds blocks 2 g and 2 g + 1 of the 256 k, of both operands; rows and columns past the
// end repeat the last one, and are dropped.  The waves' sums meet in LDS.
//
// SPLIT: x is split into its terms once a workgroup, `span` k at a time, which LDS holds (1 x
// 2560 in fp32 by 15360 x 2560 8.5 us, 18 with each wave splitting what it takes); else each
// wave loads its x with the weight.
template <int XT, int NT, bool SPLIT>
__global__ __launch_bounds__(512) void mx_rows_kernel(MxLinearArgs a, int ntiles, int span) {
    typedef MxX<XT> X;
    __shared__ float sums[8][NT * 256];
    extern __shared__ __attribute__((aligned(16))) uint16_t split[];   // [TERMS][rows][span]
    const int row0 = blockIdx.x / ntiles * 16;
    const int col0 = blockIdx.x % ntiles * 16 * NT;
    const int rows = min(a.m - row0, 16);
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int waves = blockDim.x >> 6;
    const int l16 = lane & 15, g = lane >> 4;
    const int blocks = mx_blocks(a.k);
    const int xr = min(l16, rows - 1);
    long wrow[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) wrow[j] = min(col0 + 16 * j + l16, a.n - 1);
    f32x4 acc[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};

    struct Part {   // of 256 k
        uint4 w[2][NT];
        uint32_t ws[2][NT];
        typename X::Block x[2];
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
            if constexpr (!SPLIT) X::load(a, row0 + xr, b, in, p.x[c]);
        }
    };
    auto use = [&](const Part& p, int part, int k0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            if constexpr (XT == 0) {
#pragma unroll
                for (int j = 0; j < NT; ++j)
                    acc[j] = mx_mfma<0, 0>(p.w[c][j], p.x[c].codes, acc[j], p.ws[c][j], p.x[c].scale);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e) {   // eight k
                    uint4 t[X::TERMS];
                    if constexpr (SPLIT) {
                        const int at = (part * 8 + 2 * g + c) * 32 + 8 * e - k0;
#pragma unroll
                        for (int q = 0; q < X::TERMS; ++q)
                            t[q] = *reinterpret_cast<const uint4*>(&split[(q * rows + xr) * span + at]);
                    } else {
                        X::terms(p.x[c].v[e], t);
                    }
#pragma unroll
                    for (int j = 0; j < NT; ++j) {
                        const uint32_t q4[4] = {p.w[c][j].x, p.w[c][j].y, p.w[c][j].z, p.w[c][j].w};
                        const uint4 w = mx_bf16(q4[e], mx_scale_of(p.ws[c][j], 0));
#pragma unroll
                        for (int q = 0; q < X::TERMS; ++q) acc[j] = mfma<1>(w, t[q], acc[j]);
                    }
                }
            }
        }
    };
    const int parts = (blocks + 7) / 8;
    Part p0, p1;
    int part = wave;
    if (part < parts) load(p0, part);
    for (int k0 = 0; k0 < a.k; k0 += span) {
        int end = parts;
        if constexpr (SPLIT) {
            end = min(end, (k0 + span) / 256);
            if (k0) __syncthreads();
            for (int i = threadIdx.x; i < rows * (span / 8); i += blockDim.x) {
                const int r = i / (span / 8), at = i % (span / 8) * 8;
                uint4 t[X::TERMS];
                X::terms_of(a, row0 + r, k0 + at, t);
#pragma unroll
                for (int q = 0; q < X::TERMS; ++q)
                    *reinterpret_cast<uint4*>(&split[(q * rows + r) * span + at]) = t[q];
            }
            __syncthreads();
        }
        while (part < end) {
            if (part + waves < parts) load(p1, part + waves);
            use(p0, part, k0);
            part += waves;
            if (part >= end) {
                p0 = p1;
                break;
            }
            if (part + waves < parts) load(p0, part + waves);
            use(p1, part, k0);
            part += waves;
        }
        if constexpr (!SPLIT) break;
    }

    // accumulator register r: column 4 g + r of row l16
#pragma unroll
    for (int j = 0; j < NT; ++j)
        *reinterpret_cast<f32x4*>(&sums[wave][(l16 * NT + j) * 16 + 4 * g]) = acc[j];
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

constexpr int kSplitBytes = 48 << 10;   // of LDS for terms of x

template <int XT, int NT>
hipError_t run_rows(const MxLinearArgs& a, hipStream_t stream) {
    const int ntiles = (a.n + 16 * NT - 1) / (16 * NT);
    const int parts = (mx_blocks(a.k) + 7) / 8;
    const int waves = std::min(8, parts);
    const unsigned nb = (unsigned)(((long)a.m + 15) / 16 * ntiles);
    if constexpr (XT == 1 || XT == 3) {
        const int part = std::min(a.m, 16) * MxX<XT>::TERMS * 2 * 256;   // bytes of 256 k
        // fp16 rows that several rounds of splitting would take are split by each wave (16 x
        // 2560 by 15360 x 2560 11.4 us so, 1 x 2560 9.8, by way of LDS 7.6)
        if (XT == 1 || part * waves <= kSplitBytes) {
            const int span = std::min(parts, std::max(1, kSplitBytes / part));
            mx_rows_kernel<XT, NT, true><<<nb, 64 * waves, (size_t)span * part, stream>>>(a, ntiles, 256 * span);
            return hipGetLastError();
        }
    }
    if constexpr (XT != 1) mx_rows_kernel<XT, NT, false><<<nb, 64 * waves, 0, stream>>>(a, ntiles, 0);
    return hipGetLastError();
}

constexpr int kUnits = 256;   // compute units of an MI355X

// Workgroups of 512 threads of a launch, whose threads 32 bits count.
constexpr long kWorkgroupsMost = (1L << 23) - 1;

// Tiles of 16 columns of a workgroup: the more there are, the fewer times x is read from the
// L2; as long as three quarters of the compute units have a workgroup (1 x 2560 in bf16 by
// 15360 x 2560 8.8 us with one, 7.3 with four; 1 x 5120 by 2560 x 5120 5.9 and 13).
int rows_tiles(const MxLinearArgs& a) {
    const long row_blocks = ((long)a.m + 15) / 16;
    for (int t : {4, 2})
        if (row_blocks * ((a.n + 16 * t - 1) / (16 * t)) >= kUnits * 3 / 4) return t;
    return 1;
}

// What the kernel for few rows takes with x in other types, in microseconds: a workgroup's
// rounds of 256 k a wave, and the splitting of fp32 rows.
double rows_us(const MxLinearArgs& a) {
    const int t = rows_tiles(a), at = t / 2;
    constexpr double one[3][3] = {{1.1, 1.7, 2.3}, {2.3, 3.0, 4.3}, {3.0, 3.8, 5.3}};   // by x's type
    const double split = a.x_kind == S2_DTYPE_F32 ? 1. + 0.066 * std::min(a.m, 16) * ((mx_blocks(a.k) + 7) / 8) : 0.;
    const double each = one[a.x_kind][at] * ((mx_blocks(a.k) + 63) / 64) + split;
    const long blocks = ((long)a.m + 15) / 16 * ((a.n + 16 * t - 1) / (16 * t));
    // a unit runs two workgroups at once, 1.6 times as long
    const double rounds = (double)((blocks + 2 * kUnits - 1) / (2 * kUnits)) * (blocks > kUnits ? 1.6 : 1.);
    return 2.5 + rounds * each;
}

template <int XT>
hipError_t launch_rows(const MxLinearArgs& a, hipStream_t stream) {
    const int t = rows_tiles(a);
    const long row_blocks = ((long)a.m + 15) / 16, columns = (a.n + 16L * t - 1) / (16 * t);
    if (row_blocks * columns > kWorkgroupsMost) {   // halves of the rows, or of the columns
        MxLinearArgs first = a, second = a;
        const long ye = a.y_kind ? 2 : 4;
        long at, res_at;   // of the second half in y and the residual
        if (row_blocks > 1) {
            const long m = row_blocks / 2 * 16;
            first.m = (int)m;
            second.m -= (int)m;
            if (XT == 0) {
                second.xq.codes += m * a.xq.code_stride;
                second.xq.scales += m * a.xq.scale_stride;
            } else {
                second.x = (const char*)a.x + m * a.x_stride * (XT == 1 ? 4 : 2);
            }
            at = m * a.y_stride;
            res_at = m * a.res_stride;
        } else {
            const long n = columns / 2 * 16 * t;
            first.n = (int)n;
            second.n -= (int)n;
            second.w.codes += n * a.w.code_stride;
            second.w.scales += n * a.w.scale_stride;
            if (a.bias) second.bias += n;
            at = res_at = n;
        }
        if (a.res) second.res = (const char*)a.res + res_at * ye;
        second.y = (char*)a.y + at * ye;
        const hipError_t e = launch_rows<XT>(first, stream);
        return e != hipSuccess ? e : launch_rows<XT>(second, stream);
    }
    return t == 4 ? run_rows<XT, 4>(a, stream) : t == 2 ? run_rows<XT, 2>(a, stream) : run_rows<XT, 1>(a, stream);
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

// Rows of codes that the kernel for few rows takes, one round of 16: 16 x 2560 by 15360 x 2560 8.1
// us, 17 rows 13.1, 7.6 on tiles; 17 x 10240 by 2560 x 10240 13.4 and 9.4, 17 x 2560 by 2560 x
// 2560 5.5 and 7.3.
constexpr int kRowsMost = 16;

// Rows of other types on tiles (none: bm of nought): x as planes of bf16 terms (or as it is, in bf16 with 16-byte
// rows), the weight's codes as they are, or its values in bf16 for the tile kernels of
// 16-bit operands, where the largest tiles pay for that.
struct ValuesPlan {
    TileChoice tile;
    bool pack_x, codes;
    int planes, width;       // of packed x; k rounded up to 8 where it is not packed
    size_t x_bytes, w_bytes, sum_bytes;
    size_t bytes() const { return x_bytes + w_bytes + sum_bytes; }
    // launches, bytes a microsecond read and written
    double us() const { return tile.us + 2. + (codes && pack_x ? 3. : 0.) + (2.3 * x_bytes + 1.3 * w_bytes) / 5.5e6; }
};

// Threads that 32 bits count: 512 a workgroup of 256 x 256 tiles, else 256.
bool one_launch(const MxLinearArgs& a, const TileChoice& t) {
    const long blocks = ((long)a.m + t.bm - 1) / t.bm * ((a.n + t.bn - 1) / t.bn) * t.parts;
    return blocks * (t.bm == 256 ? 512 : 256) < 1L << 32;
}

// What tiles of the weight's codes take, in microseconds: a workgroup's first loads and
// epilogue, and 256 k, for which its compute unit takes in 50 or 41 KB; by
// rows in fp16, whose blocks' sums take their scales one by one.
struct WeightCost {
    int bm, bn;
    double round, step, step_f16;
};
constexpr WeightCost kWeightCosts[] = {{64, 128, 2.8, 1.28, 1.8}, {64, 64, 3., 0.8, 1.27}};

TileChoice weight_tiles(const MxLinearArgs& a, bool f16, long steps, long most) {
    TileChoice best{0., 0, 0, 1};
    const double each = (double)a.m * round_up(a.n, 4) * sizeof(float);   // a range's sums
    for (const WeightCost& t : kWeightCosts) {
        const long count = ((long)a.m + t.bm - 1) / t.bm * ((a.n + t.bn - 1) / t.bn);
        for (long parts = 1; parts <= std::max<long>(1, std::min(most, steps / 2)); ++parts) {
            if (count * parts > kWorkgroupsMost) break;
            const double rounds = (double)((count * parts + kUnits - 1) / kUnits);
            const double us = rounds * (t.round + (f16 ? t.step_f16 : t.step) * (double)((steps + parts - 1) / parts)) +
                              (parts > 1 ? 3. + 2. * parts * each / 9e6 : 0.);
            if (best.us == 0. || us < best.us) best = TileChoice{us, t.bm, t.bn, (int)parts};
        }
    }
    return best;
}

ValuesPlan values_plan(const MxLinearArgs& a, bool codes, size_t workspace_bytes) {
    ValuesPlan p{};
    const long k8 = round_up(a.k, 8);
    p.codes = codes;
    const bool rows16 = a.k % 8 == 0 && a.x_stride % 8 == 0 && (uintptr_t)a.x % 16 == 0;
    p.planes = a.x_kind == S2_DTYPE_F32 ? kTerms : a.x_kind == S2_DTYPE_F16 && !(codes && rows16) ? 2 : 1;
    p.pack_x = p.planes > 1 || !rows16;
    p.width = (int)round_up(a.k, 64);
    if (p.pack_x) p.x_bytes = round_up((size_t)a.m * p.planes * p.width * 2, 256);
    if (!codes) p.w_bytes = round_up((size_t)a.n * k8 * 2, 256);
    if (p.bytes() > workspace_bytes) return p;
    MatmulArgs m = values_args(a, nullptr);
    m.k = (int)k8;
    const size_t each = (size_t)a.m * round_up(a.n, 4) * sizeof(float);
    const long most = std::min<long>(16, (long)((workspace_bytes - p.bytes()) / each));
    p.tile = codes ? weight_tiles(a, a.x_kind == S2_DTYPE_F16 && p.planes == 1, (k8 + 255) / 256 * p.planes, most)
                   : choose_tiles(m, (k8 + 63) / 64 * p.planes, most);
    if (!codes && !one_launch(a, p.tile)) p.tile.bm = 0;
    p.sum_bytes = p.tile.parts > 1 ? p.tile.parts * each : 0;
    return p;
}

// Pieces of eight: x's first (`xw` a row and plane), then the weight's.
template <int XT>
__global__ __launch_bounds__(256) void mx_values_kernel(MxLinearArgs a, uint16_t* x, int xw, uint16_t* w, int ww) {
    typedef MxX<XT> X;
    const long nx = (long)a.m * xw, all = nx + (long)a.n * ww;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) {
        if (i < nx) {
            const long row = i / xw;
            const int at = (int)(i - row * xw) * 8;
            uint4 t[X::TERMS];
            X::terms_of(a, row, at, t);
#pragma unroll
            for (int q = 0; q < X::TERMS; ++q)
                *reinterpret_cast<uint4*>(x + (row * X::TERMS + q) * xw * 8 + at) = t[q];
        } else {
            const long row = (i - nx) / ww;
            const int at = (int)(i - nx - row * ww);   // of four bytes
            const uint32_t codes = *reinterpret_cast<const uint32_t*>(a.w.codes + row * a.w.code_stride + 4 * at);
            *reinterpret_cast<uint4*>(w + (row * ww + at) * 8) =
                mx_bf16(codes, mx_scale_of(a.w.scales[row * a.w.scale_stride + (at >> 2)], 0));
        }
    }
}

template <int XT>
hipError_t launch_values(const MxLinearArgs& a, const ValuesPlan& p, void* workspace, hipStream_t stream) {
    uint16_t* x = (uint16_t*)workspace;
    uint16_t* w = (uint16_t*)((char*)workspace + p.x_bytes);
    MatmulArgs m = values_args(a, w);
    m.k = (int)round_up(a.k, 8);
    const int xw = p.pack_x ? p.width / 8 : 0, ww = m.k / 8;
    MxLinearArgs job = a;
    if (!p.pack_x) job.m = 0;
    if (p.codes) job.n = 0;
    if (const long all = (long)job.m * xw + (long)job.n * ww) {
        mx_values_kernel<XT><<<(unsigned)std::min<long>((all + 255) / 256, 65536), 256, 0, stream>>>(job, x, xw, w, ww);
        const hipError_t e = hipGetLastError();
        if (e != hipSuccess) return e;
    }
    if (p.pack_x || !p.codes) m.x_kind = S2_DTYPE_BF16;   // else fp16 stays
    if (p.pack_x) {
        m.x = x;
        m.x_stride = (long)p.planes * p.width;
        m.planes = p.planes;
        m.plane = p.width;
    }
    float* sums = (float*)((char*)w + p.w_bytes);
    if (p.codes) {
        m.w = a.w.codes;
        return launch_mx_weight_tiles(m, {nullptr, 0, a.w.scales, a.w.scale_stride, mx_blocks(a.k)}, p.tile, sums, stream);
    }
    MatmulPlan t{};
    t.kernel = MatmulPlan::kTiles;
    t.bm = p.tile.bm;
    t.bn = p.tile.bn;
    t.parts = p.tile.parts;
    t.whole = whole_pieces(m);
    return launch_matmul_tiles(m, t, sums, stream);
}

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
    // what a tile's own scales leave is for the sums, so that the bytes of a plan give it again
    for (int largest : {256, 128}) {
        const size_t scales = round_up(largest == 256 ? dealt.x + dealt.w : copied, 256);
        if (scales > workspace_bytes) continue;
        const TileChoice t = choose_tiles(m, (m.k + 63) / 64, ranges(a, workspace_bytes - scales), largest);
        if ((largest == 256 && t.bm < 256) || (p.tile.bm && p.tile.us <= t.us) || !one_launch(a, t)) continue;
        p.tile = t;
        p.scales = scales;
        p.sums = t.parts > 1 ? (size_t)t.parts * a.m * round_up(a.n, 4) * sizeof(float) : 0;
    }
    return p;   // no tile: not on tiles
}

}  // namespace

size_t mx_linear_workspace(const MxLinearArgs& a) {
    if (!a.mx) {
        MxLinearArgs near = a, far = a;
        near.x_stride = round_up(a.k, 8);
        far.x_stride = a.k + 1;   // rows that are packed
        size_t most = 0;
        for (bool codes : {false, true})
            for (const MxLinearArgs& b : {near, far}) {
                const ValuesPlan p = values_plan(b, codes, (size_t)1 << 62);
                if (p.tile.bm && p.us() < rows_us(a)) most = std::max(most, p.bytes());
            }
        return most;
    }
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
    const long out = std::max(a.y_stride, a.res ? a.res_stride : 0L) * (a.y_kind ? 2 : 4);
    const long far = 0x7fffffffL;   // 32-bit offsets
    if (!a.mx) {
        if (256 * out < far && (long)a.n * 4 < far && 256 * 2 * a.x_stride < far &&
            256 * 2 * kTerms * (a.k + 64L) < far) {
            ValuesPlan p = values_plan(a, false, workspace_bytes);
            if (scales16(a.w.scales, a.w.scale_stride) && 256 * a.w.scale_stride < far) {
                const ValuesPlan c = values_plan(a, true, workspace_bytes);
                if (c.tile.bm && (!p.tile.bm || c.us() < p.us())) p = c;
            }
            // In bf16 by rows, with the weight's values and with its codes on tiles: 77 x 5120 by
            // 2560 x 5120 14.6, 26, 12.9 us; 128 x 2560 by 15360 x 2560 66, 41, 17; 500 x 2560 by
            // the same 242, 60, 64; 1000 x 2560 77 and 127; 48 x 2560 by 2560 x 2560 7.2, 18, 8.8.
            if (p.tile.bm && p.us() < rows_us(a))
                return a.x_kind == 0   ? launch_values<1>(a, p, workspace, stream)
                       : a.x_kind == 1 ? launch_values<2>(a, p, workspace, stream)
                                       : launch_values<3>(a, p, workspace, stream);
        }
        return a.x_kind == 0   ? launch_rows<1>(a, stream)
               : a.x_kind == 1 ? launch_rows<2>(a, stream)
                               : launch_rows<3>(a, stream);
    }
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
