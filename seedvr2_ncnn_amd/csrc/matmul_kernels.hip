// Matrix products with bias, activation and residual in the epilogue, over all
// rows (s2_linear) or over ragged row groups with a weight each
// (s2_grouped_linear):  y = residual + act(x W^T + bias).
//
// x [m][k] and W [n][k] are both k-contiguous, the operand layout of the 16-bit
// MFMAs.  Row 16 j + c of the 64 weight rows of a wave stands in LDS for column
// 4 c + j, so that accumulators j = 0 .. 3 of a lane are four neighbours of a row
// of y, and 16 lanes hold 64: the epilogue adds bias and residual and stores whole
// 128-byte row pieces straight from the registers, with one rounding at the end.
//
// This file: which kernel takes a call, the packing of rows that the tile kernels
// cannot read, and the kernel for any shape and alignment.
#include <cmath>

#include "matmul_device.h"

namespace s2 {

bool whole_pieces(const MatmulArgs& a) {
    const size_t e = a.y_kind ? 8 : 16;
    return a.n % 4 == 0 && a.y_stride % 4 == 0 && (uintptr_t)a.y % e == 0 &&
           (uintptr_t)a.bias % 16 == 0 &&
           (!a.res || (a.res_stride % 4 == 0 && (uintptr_t)a.res % e == 0));
}

namespace {

// Any strides, alignment, n and k; fp32 activations.  Block tile 128x128,
// k-step 32, four waves in a 2x2 grid of 64x64, both operands through registers
// into double-buffered LDS.  SPLIT: an fp32 x as bf16 terms (else x is of the weight's
// type).
template <int T, bool SPLIT, int YK>
__global__ __launch_bounds__(256, 2) void matmul_any_kernel(MatmulArgs a, int ntiles, bool whole) {
    constexpr int BM = 128, BN = 128, BK = 32, P = BK + 8, PL = SPLIT ? kTerms : 1;
    __shared__ __attribute__((aligned(16))) uint16_t x_lds[2][PL][BM * P];
    __shared__ __attribute__((aligned(16))) uint16_t w_lds[2][BN * P];
    RowTiles rts(a, BM, gridDim.x / ntiles);
    const int blocks = rts.count * ntiles;
    if ((int)blockIdx.x >= blocks) return;   // the whole workgroup
    const int lid = xcd_remap(blockIdx.x, blocks);
    const RowTile rt = rts.at(lid / ntiles);
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
    float xf[SPLIT ? 2 : 1][8];
    uint4 xr[2], wr[2];
    auto load = [&](int k0) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = (tid >> 2) + 64 * c;
            const int kc = k0 + (tid & 3) * 8;
            const int col = col0 + (r & ~63) + 4 * (r & 15) + ((r >> 4) & 3);
            const long xo = (long)(rt.row0 + r) * a.x_stride + kc;
            wr[c] = piece16<false>(w + (long)col * a.k + kc, col < a.n ? a.k - kc : 0);
            const int left = r < rows ? a.k - kc : 0;
            if constexpr (SPLIT)
                piece32<false>((const float*)a.x + xo, left, xf[c]);
            else
                xr[c] = piece16<false>((const uint16_t*)a.x + xo, left);
        }
    };
    auto put = [&](int buf) {
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            const int r = (tid >> 2) + 64 * c;
            const int at = r * P + (tid & 3) * 8;
            *reinterpret_cast<uint4*>(&w_lds[buf][at]) = wr[c];
            if constexpr (SPLIT) {
                uint4 h[PL];
                split8(xf[c], h);
#pragma unroll
                for (int i = 0; i < PL; ++i) *reinterpret_cast<uint4*>(&x_lds[buf][i][at]) = h[i];
            } else {
                *reinterpret_cast<uint4*>(&x_lds[buf][0][at]) = xr[c];
            }
        }
    };

    TileEnd<YK, 4> end(a, rt, rows, wm * 64, col0 + wn * 64 + 4 * l16, whole);
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
    end.finish(a, acc);
}

template <int T, bool SPLIT, int YK>
hipError_t launch_any(const MatmulArgs& a, hipStream_t stream) {
    const int ntiles = (a.n + 127) / 128;
    const long blocks = row_tiles(a, 128) * ntiles;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    matmul_any_kernel<T, SPLIT, YK><<<(unsigned)blocks, 256, 0, stream>>>(a, ntiles, whole_pieces(a));
    return hipGetLastError();
}

// Rows for the tile kernels: [rows][planes][width] from [rows][k], zeros from k to
// width, in pieces of eight elements.  An fp32 row is packed as `planes` bf16 terms, a
// 16-bit one as it is, `planes` times.
struct PackJob {
    const void* src;
    int kind;           // 0 fp32, else 16 bits
    long stride, rows;
    int planes, width;
    uint16_t* dst;
};

__device__ __forceinline__ void pack_piece(const PackJob& job, int k, long i) {
    const int pieces = job.width / 8;
    const long row = i / pieces;
    const int kc = (int)(i - row * pieces) * 8;
    uint16_t* out = job.dst + row * job.planes * job.width + kc;
    if (job.kind == 0) {
        float v[8];
        uint4 h[kTerms];
        piece32<false>((const float*)job.src + row * job.stride + kc, k - kc, v);
        split8(v, h);
#pragma unroll
        for (int q = 0; q < kTerms; ++q) *reinterpret_cast<uint4*>(out + (long)q * job.width) = h[q];
    } else {
        const uint4 h = piece16<false>((const uint16_t*)job.src + row * job.stride + kc, k - kc);
        for (int q = 0; q < job.planes; ++q) *reinterpret_cast<uint4*>(out + (long)q * job.width) = h;
    }
}

// x, then the weight, either of which may have no rows.
__global__ __launch_bounds__(256) void matmul_pack_kernel(PackJob x, PackJob w, int k) {
    const long nx = x.rows * (x.width / 8), all = nx + w.rows * (w.width / 8);
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < all; i += (long)gridDim.x * 256) {
        if (i < nx)
            pack_piece(x, k, i);
        else
            pack_piece(w, k, i - nx);
    }
}

hipError_t launch_pack(const PackJob& x, const PackJob& w, int k, hipStream_t stream) {
    const long all = x.rows * (x.width / 8) + w.rows * (w.width / 8);
    const unsigned nb = (unsigned)std::min<long>((all + 255) / 256, 65536);
    matmul_pack_kernel<<<nb, 256, 0, stream>>>(x, w, k);
    return hipGetLastError();
}

template <int YK>
hipError_t launch_any_y(const MatmulArgs& a, hipStream_t stream) {
    if (a.w_kind == 2) return launch_any<2, false, YK>(a, stream);
    if (a.x_kind == 0) return launch_any<1, true, YK>(a, stream);
    return launch_any<1, false, YK>(a, stream);
}

constexpr int kUnits = 256;   // compute units of an MI355X

// What tiles take, in microseconds, from which the tile and the ranges of k are
// chosen: a compute unit holds `each` workgroups of a kind at once; such a round costs
// `round` for first loads and epilogues and, for 64 k, `one` step of a single workgroup
// or `full` of all of them.  Measured with bf16 rows, 72 to 2048 of them, k of 256 to
// 10240 and n of 512 to 15360.  Against the best of the four tiles and 1 to 12 ranges:
// 77 x 5120 by 2560 x 5120 15 us either way (one range of 128 x 128: 48); 512 x 512 by
// 512 x 512 6.5 (128 x 128: 11); 14400 x 512 by 512 x 512 15 (256 x 256: 19); 1024 x
// 2560 by 2560 x 2560 28 (256 x 256: 47); 2048 x 2560 by 15360 x 2560 136 (128 x 128:
// 186).
struct TileCost {
    int bm, bn, each;
    double round, one, full;
};
constexpr TileCost kTileCosts[] = {{256, 256, 1, 6.5, 1.3, 1.3},
                                   {128, 128, 2, 4.5, 0.57, 0.88},
                                   {128, 64, 2, 3.5, 0.38, 0.57},
                                   {64, 64, 2, 2.5, 0.3, 0.45}};

double tiles_us(const TileCost& t, double blocks, double steps) {
    const double slots = (double)kUnits * t.each;
    const double rounds = std::floor(blocks / slots), rest = blocks - rounds * slots;
    return rounds * (t.round + steps * t.full) +
           (rest > 0 ? t.round + steps * (rest <= kUnits ? t.one : t.full) : 0.);
}

// a group's last tile is half empty, on average
double tile_count(const MatmulArgs& a, const TileCost& t) {
    return (a.offsets ? (double)a.m / t.bm + 0.5 * std::min(a.groups, a.m) : (double)row_tiles(a, t.bm)) *
           (double)((a.n + t.bn - 1) / t.bn);
}

// The kernel for any shape with 16-bit rows, by the same measure, against packing those
// rows (and the weight) first: a launch, and bytes a microsecond read and written.  Rows
// apart by four elements too many: 8000 x 2560 by 2560 x 2560 177 us here and 118 packed,
// 300 x 2560 by 512 x 2560 66 and 14, 14400 x 1024 by 512 x 1024 37 and 34, but x 512 19
// and 25, 100000 x 512 by 64 x 512 39 and 52, 2000 x 128 by 512 x 128 8 and 11.
constexpr TileCost kAnyCost = {128, 128, 2, 2.5, 1.5, 2.1};
constexpr double kPackUs = 5., kPackBytesUs = 5e6;

// The sums of k ranges: a launch, and bytes a microsecond written and read again.
constexpr double kSumUs = 3., kSumBytesUs = 9e6;

// Reading the weight once, at 5 TB/s.
double weight_us(const MatmulArgs& a) {
    return (double)std::min(a.groups, a.m) * a.n * a.k * 2 / 5e6;
}

// A call on the rows kernel: a workgroup gets its weight rows and its rows of x through
// the caches at about 30 KB a microsecond.
double rows_us(const MatmulArgs& a, const MatmulPlan& r, long rows) {
    const double blocks = (double)row_tiles(a, r.rows) * ((a.n + r.cols - 1) / r.cols);
    return std::max(1., blocks / kUnits) * (r.cols + rows) * (double)a.k * 2 / 30e3;
}

long round_up(long v, long to) { return (v + to - 1) / to * to; }

// bf16 terms of a value of x
int packed_planes(const MatmulArgs& a) { return a.x_kind ? 1 : kTerms; }

// Elements of a packed plane.  Where the weight is packed too it is repeated for each
// plane of x, so that the planes are one longer row; else its rows are read once for
// each plane, in steps of 64 k that x has to fill.
long packed_width(const MatmulArgs& a, bool pack_w) { return round_up(a.k, pack_w ? 8 : 64); }

// 16-byte rows of 16-bit elements
bool rows16(const void* p, long stride) { return stride % 8 == 0 && (uintptr_t)p % 16 == 0; }

}  // namespace

TileChoice choose_tiles(const MatmulArgs& a, long steps, long most, int largest) {
    TileChoice best{0., 0, 0, 1};
    const double each = (double)a.m * round_up(a.n, 4) * sizeof(float);   // a range's sums
    for (const TileCost& t : kTileCosts) {
        if (t.bm > largest) continue;
        const double count = tile_count(a, t);
        for (long parts = 1; parts <= std::max<long>(1, std::min(most, steps / 4)); ++parts) {
            const double us = std::max(tiles_us(t, count * parts, (double)steps / parts), weight_us(a)) +
                              (parts > 1 ? kSumUs + 2. * parts * each / kSumBytesUs : 0.);
            if (best.us == 0. || us < best.us) best = TileChoice{us, t.bm, t.bn, (int)parts};
        }
    }
    return best;
}

MatmulPlan plan_matmul(const MatmulArgs& a, size_t workspace_bytes) {
    MatmulPlan p{};
    p.parts = 1;
    const long rows = a.offsets ? ((long)a.m + a.groups - 1) / a.groups : a.m;   // of a group
    // what the tile kernels need: 16-byte rows, packed here where a call's are not
    p.pack_x = a.x_kind == 0 || a.k % 8 != 0 || !rows16(a.x, a.x_stride);
    p.pack_w = a.k % 8 != 0 || (uintptr_t)a.w % 16 != 0;
    const bool direct = !p.pack_x && !p.pack_w;
    const long row = packed_planes(a) * packed_width(a, p.pack_w);
    if (p.pack_w) p.pack_x = true;   // a weight of padded rows needs padded x
    if (p.pack_x) p.x_bytes = round_up((size_t)a.m * row * 2, 256);
    if (p.pack_w) p.w_bytes = round_up((size_t)a.groups * a.n * row * 2, 256);
    const bool room = p.bytes() <= workspace_bytes;
    const long pitch = p.pack_x ? row : a.x_stride;
    const long out = std::max(a.y_stride, a.res ? a.res_stride : 0L) * (a.y_kind ? 2 : 4);
    const bool near = 256 * out < 0x7fffffffL && (long)a.n * 4 < 0x7fffffffL;   // 32-bit offsets
    const bool tiles = near && room && 256 * pitch * 2 < 0x7fffffffL &&
                       256 * std::max<long>(a.k, p.pack_w ? row : 0) * 2 < 0x7fffffffL;

    // many fp32 rows of a short k, packed and on tiles -> here: by 2560 x 132 2700 rows 20
    // -> 15 us, 21600 80 -> 60; by 2560 x 160 19 -> 17 and 83 -> 60; with fp32 results 91 ->
    // 56 and 95 -> 62; by 1024 x 64 5000 rows 14.4 -> 13.7, 7000 14.1 -> 12.3, 21600 29 ->
    // 21.  Fewer outputs gain only where the weight would be packed too.
    if (a.x_kind == 0 && !a.offsets && rows > 32 && (long)a.m * a.n >= 6L << 20 && near &&
        a.k <= kShortMost &&
        a.x_stride < 1L << 24) {
        MatmulPlan s{};
        s.kernel = MatmulPlan::kShort;
        s.parts = std::max(1, kUnits / ((a.n + 255) / 256));
        s.whole = whole_pieces(a);
        return s;
    }

    double tile_us = 0.;
    if (tiles) {
        p.kernel = MatmulPlan::kTiles;
        p.whole = whole_pieces(a);
        const long steps = p.pack_w ? (row + 63) / 64 : ((long)a.k + 63) / 64 * packed_planes(a);
        const size_t each = (size_t)a.m * round_up(a.n, 4) * sizeof(float);   // a range's sums
        const long most =
            a.offsets ? 1 : std::min<long>(16, (long)((workspace_bytes - p.bytes()) / each));
        const TileChoice t = choose_tiles(a, steps, most);
        tile_us = t.us;
        p.bm = t.bm;
        p.bn = t.bn;
        p.parts = t.parts;
        if (p.parts > 1) p.sum_bytes = p.parts * each;
        const bool any = a.x_kind != 0 && p.pack_x &&
                         tiles_us(kAnyCost, tile_count(a, kAnyCost), (a.k + 63) / 64) <
                             tile_us + kPackUs + 2. * (double)(p.x_bytes + p.w_bytes) / kPackBytesUs;
        if (rows > 32 && !any) return p;
    }

    // few rows
    MatmulPlan r{};
    r.rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    // the more columns a workgroup has, the fewer times x is read from the L2; as long as
    // three quarters of the compute units have one (1 x 2560 by 15360 x 2560: 19.0 us by
    // 16 columns, 15.9 by 32, 14.9 by 64; by 2560 x 2560: 6.8, 9.2, 13.2)
    const long row_blocks = row_tiles(a, r.rows);
    r.cols = 16;
    for (int c : {32, 64})
        if (row_blocks * ((a.n + c - 1) / c) >= kUnits * 3 / 4) r.cols = c;
    if (rows <= 32) {
        r.kernel = MatmulPlan::kRows;
        r.parts = 1;
        // against the tiles where those need no packing (16 x 10240 by 2560 x 10240 15 us
        // on tiles, 22 on rows; 1 x 10240 18 and 15); more than a few fp32 rows are packed
        // rather than split by every workgroup (32 rows by 2560 x 10240 26 us and 49, by
        // 2560 x 5120 18 and 26, by 2560 x 2560 15 both, but by 1024 x 1024 13 and 8)
        const bool use_tiles = direct ? tile_us < rows_us(a, r, std::min(rows, (long)a.m))
                                      : a.x_kind == 0 && rows > 16 && !p.pack_w;
        return tiles && use_tiles ? p : r;
    }
    // any shape, unpacked; rows that 32-bit offsets do not reach
    r.kernel = near ? MatmulPlan::kAny : MatmulPlan::kRows;
    r.parts = 1;
    return r;
}

hipError_t launch_matmul(const MatmulArgs& args, void* workspace, size_t workspace_bytes,
                         hipStream_t stream) {
    if (args.m <= 0) return hipSuccess;
    MatmulArgs a = args;
    a.planes = 1;
    a.plane = 0;
    if (a.m == 1) {   // the strides of a single row say nothing
        a.x_stride = a.k;
        a.res_stride = a.y_stride = a.n;
    }
    const MatmulPlan p = plan_matmul(a, workspace_bytes);
    char* at = (char*)workspace;
    if (p.pack_x) {
        const int planes = packed_planes(a), width = (int)packed_width(a, p.pack_w);
        const PackJob x{a.x, a.x_kind, a.x_stride, a.m, planes, width, (uint16_t*)at};
        const PackJob w{a.w, a.w_kind, a.k, p.pack_w ? (long)a.groups * a.n : 0, planes, width,
                        (uint16_t*)(at + p.x_bytes)};
        const hipError_t e = launch_pack(x, w, a.k, stream);
        if (e != hipSuccess) return e;
        a.x = x.dst;
        a.x_kind = a.w_kind;
        a.x_stride = (long)planes * width;
        if (p.pack_w) {   // one long row
            a.w = w.dst;
            a.k = planes * width;
        } else {
            a.planes = planes;
            a.plane = width;
        }
        at += p.x_bytes + p.w_bytes;
    }
    switch (p.kernel) {
        case MatmulPlan::kRows: return launch_matmul_rows(a, p, stream);
        case MatmulPlan::kShort: return launch_matmul_short(a, p, stream);
        case MatmulPlan::kTiles: return launch_matmul_tiles(a, p, (float*)at, stream);
        default:
            return a.y_kind == 0   ? launch_any_y<0>(a, stream)
                   : a.y_kind == 1 ? launch_any_y<1>(a, stream)
                                   : launch_any_y<2>(a, stream);
    }
}

}  // namespace s2
