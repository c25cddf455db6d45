// Cross attention: softmax(scale q k^T) v per sample and head, keys of another length
// than the queries.
#include <cmath>

#include "cross_attention_device.h"

namespace s2 {

namespace {

constexpr int kJoinFew = 4;

// Four columns of a row a thread, for few parts: their sums, by how far their maxima lie
// below the largest.
__global__ __launch_bounds__(256) void cross_join_few_kernel(CrossArgs a, CrossParts p, long rows) {
    const int quads = a.d / 4;
    const long i = (long)blockIdx.x * 256 + threadIdx.x;
    if (i >= rows * a.heads * quads) return;
    const long rh = i / quads;
    const int col = (int)(i - rh * quads) * 4;
    const long row = rh / a.heads;
    const int h = (int)(rh - row * a.heads);
    // rows in no sample
    if (a.q_offsets && (row < clamped(a.q_offsets[0], a.lq) || row >= clamped(a.q_offsets[a.batch], a.lq))) return;
    float2 w[kJoinFew];
    f32x4 o[kJoinFew];
#pragma unroll
    for (int q = 0; q < kJoinFew; ++q) {
        const long at = rh * p.parts + min(q, p.parts - 1);
        w[q] = p.weights[at];
        o[q] = *reinterpret_cast<const f32x4*>(p.sums + at * a.d + col);
    }
    const float c = weight_scale(a);
    float m = w[0].x, l = 0.f;
#pragma unroll
    for (int q = 1; q < kJoinFew; ++q) m = fmaxf(m, w[q].x);
    f32x4 sum = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < kJoinFew; ++q) {
        if (q >= p.parts) break;
        const float f = __builtin_amdgcn_exp2f((w[q].x - m) * c);
        l += f * w[q].y;
        sum += f * o[q];
    }
    const long b = a.q_offsets ? 0 : row / a.lq;
    store4_out(a, b * a.os.batch + (row - b * a.lq) * a.os.row + h * a.os.head + col,
               sum * (l == 0.f ? 0.f : 1.f / l));
}

// The same for many parts, a wave a row and head.
// `lanes` lanes (a power of two, at least d / 4) have four columns each, and every 64 /
// lanes-th part.
__global__ __launch_bounds__(256) void cross_join_kernel(CrossArgs a, CrossParts p, long rows, int lanes) {
    const long rh = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (rh >= rows * a.heads) return;
    const long row = rh / a.heads;
    const int h = (int)(rh - row * a.heads);
    // rows in no sample
    if (a.q_offsets && (row < clamped(a.q_offsets[0], a.lq) || row >= clamped(a.q_offsets[a.batch], a.lq))) return;
    const int lane = threadIdx.x & 63;
    const float2 w = lane < p.parts ? p.weights[rh * p.parts + lane] : make_float2(kLowest, 0.f);
    float m = w.x;
#pragma unroll
    for (int x = 32; x; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    const float f = __builtin_amdgcn_exp2f((w.x - m) * weight_scale(a));
    float l = f * w.y;
#pragma unroll
    for (int x = 32; x; x >>= 1) l += __shfl_xor(l, x);
    const int col = (lane & (lanes - 1)) * 4, step = 64 / lanes;
    const float* sums = p.sums + rh * p.parts * a.d + min(col, a.d - 4);
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int q0 = 0; q0 < p.parts; q0 += step) {
        const int q = q0 + lane / lanes;   // (parts past the last one have weight 0)
        const float fq = __shfl(f, min(q, 63));
        if (q < p.parts) o += fq * *reinterpret_cast<const f32x4*>(sums + (long)q * a.d);
    }
    for (int x = lanes; x < 64; x <<= 1)
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
    if (lane >= lanes || col >= a.d) return;
    const long b = a.q_offsets ? 0 : row / a.lq;
    store4_out(a, b * a.os.batch + (row - b * a.lq) * a.os.row + h * a.os.head + col, o * (l == 0.f ? 0.f : 1.f / l));
}

long all_rows(const CrossArgs& a) { return a.q_offsets ? (long)a.lq : (long)a.batch * a.lq; }

size_t part_bytes(const CrossArgs& a) { return (size_t)all_rows(a) * a.heads * (a.d * sizeof(float) + sizeof(float2)); }

constexpr int kUnits = 256;   // compute units of an MI355X

// Microseconds that a compute unit takes for a tile of keys with 1, 2, .. workgroups on it,
// `each` at most, for d up to 64, 128 and 256: 4096 x 21600 with 20 heads of 128 in one
// range of keys is three workgroups on half of the units and two on the others, 875 us; in
// two ranges five in turn, 792.  1024 x 4096 82 us in one, 57 in three; 300 x 20000, two
// heads, 377 and 31 in 32; in fp32 508 and 359, 1376 and 75.
struct CrossCost {
    int each;
    double us[4];
};
constexpr CrossCost kCrossCosts[2][3] = {
    {{4, {0.54, 0.7, 0.88, 1.1}}, {3, {0.7, 1.03, 1.43, 0.}}, {2, {1.45, 2.2, 0., 0.}}},
    {{4, {1.3, 2., 2.7, 3.5}}, {2, {2.5, 3.7, 0., 0.}}, {1, {5., 0., 0., 0.}}}};   // fp32
constexpr double kJoinUs = 4., kJoinBytesUs = 6e6;   // the joining launch; bytes written and read

CrossPlan cross_plan(const CrossArgs& a, size_t workspace_bytes) {
    const long group = a.heads / a.kv_heads;
    const long rows = (long)a.lq * group;
    const int each = a.kind ? kTileRows : kTileRows32;
    auto tiles_of = [&](long each) {
        const long last = a.batch <= kScanSamples ? std::min(a.batch, a.lq) : a.batch;   // tiles that are not full
        return std::min<long>(a.q_offsets ? rows / each + last : a.batch * ((rows + each - 1) / each), 0x7fffffffL);
    };
    CrossPlan p;
    p.run = 1;
    p.tiles = (int)tiles_of(each);
    // a sample's last tile is half empty, on average
    const double blocks = a.kv_heads * (a.q_offsets ? (double)rows / each + 0.5 * std::min(a.batch, a.lq)
                                                    : (double)p.tiles);
    const long keys = a.q_offsets ? ((long)a.lk + a.batch - 1) / std::max(a.batch, 1) : a.lk;   // of a sample
    if (a.kind && a.d > 64 && a.d <= 128 && keys <= kShortKeys) {
        // the run by which the compute units' turns, of `run` rounds and one to begin, are
        // fewest; worth it from about four on (4096 queries on 77 keys, 20 heads: two rounds 18.5
        // us, 15.2 by the other kernel)
        const long slots = (long)kUnits * kShortEach;
        long least = 0;
        for (int run = 1; run <= 64; ++run) {
            const long turns = (tiles_of((long)each * run) * a.kv_heads + slots - 1) / slots * (run + 1);
            if (run == 1 || turns < least) least = turns, p.run = run;
        }
        if (p.run >= 4) {
            p.tiles = (int)tiles_of((long)each * p.run);
            p.parts = 1;
            return p;
        }
        p.run = 1;
    }
    const double tiles = (double)((keys + kTileKeys - 1) / kTileKeys);
    // 32 bits count the workgroups, and the threads of a join's launch, 64 a row at most
    const bool joined = (double)all_rows(a) * a.heads * 64. < 0x1p32;
    const long most = joined ? std::min(std::min(64L, (long)(workspace_bytes / part_bytes(a))),
                                        0x7fffffffL / ((long)p.tiles * a.kv_heads))
                             : 1;
    const CrossCost& c = kCrossCosts[a.kind == 0][a.d <= 64 ? 0 : a.d <= 128 ? 1 : 2];
    double best = 0.;
    p.parts = 1;
    for (long parts = 1; parts <= std::max<long>(1, std::min<long>(most, (long)tiles / 2)); ++parts) {
        const double all = blocks * parts, slots = (double)kUnits * c.each;
        const double rest = all - std::floor(all / slots) * slots;
        double us = std::floor(all / slots) * c.us[c.each - 1];
        if (rest > 0) us += c.us[(int)std::ceil(rest / kUnits) - 1];
        us *= std::ceil(tiles / parts);
        if (parts > 1) us += kJoinUs + 2. * parts * part_bytes(a) / kJoinBytesUs;
        if (parts == 1 || us < best) best = us, p.parts = (int)parts;
    }
    return p;
}

}  // namespace

CrossParts cross_parts(const CrossArgs& a, const CrossPlan& plan, void* workspace) {
    float* sums = (float*)workspace;
    return CrossParts{plan.parts, sums,
                      (float2*)(sums + (size_t)all_rows(a) * a.heads * plan.parts * (plan.parts > 1 ? a.d : 0))};
}

size_t cross_attention_workspace(const CrossArgs& a) {
    const CrossPlan p = cross_plan(a, (size_t)1 << 62);
    return p.parts > 1 ? p.parts * part_bytes(a) : 0;
}

hipError_t launch_cross_attention(const CrossArgs& a, void* workspace, size_t workspace_bytes,
                                  hipStream_t stream) {
    const long rows = all_rows(a);
    if (rows <= 0) return hipSuccess;
    const CrossPlan p = cross_plan(a, workspace_bytes);
    if ((long)p.tiles * a.kv_heads * p.parts >= 0x7fffffffL) {   // workgroups that 32 bits do not count: halves of the heads
        if (a.kv_heads == 1) return hipErrorInvalidValue;   // no memory holds so many rows of out
        const size_t e = a.kind ? 2 : 4, oe = a.out_kind ? 2 : 4;
        CrossArgs first = a, second = a;
        auto past = [](const void* at, long n, size_t each) { return (const void*)((const char*)at + n * (long)each); };
        const int h = a.kv_heads / 2, qh = h * (a.heads / a.kv_heads);
        first.kv_heads = h;
        first.heads = qh;
        second.kv_heads -= h;
        second.heads -= qh;
        second.q = past(a.q, qh * a.qs.head, e);
        second.k = past(a.k, h * a.ks.head, e);
        second.v = past(a.v, h * a.vs.head, e);
        second.out = (void*)past(a.out, qh * a.os.head, oe);
        const hipError_t e1 = launch_cross_attention(first, workspace, workspace_bytes, stream);
        return e1 != hipSuccess ? e1 : launch_cross_attention(second, workspace, workspace_bytes, stream);
    }
    const hipError_t e = a.kind ? launch_cross_tiles(a, p, workspace, stream) : launch_cross_f32(a, p, workspace, stream);
    if (e != hipSuccess || p.parts == 1) return e;
    int lanes = 2;
    while (lanes * 4 < a.d) lanes *= 2;
    const CrossParts parts = cross_parts(a, p, workspace);
    const bool few = p.parts <= kJoinFew;
    const long blocks = few ? (rows * a.heads * (a.d / 4) + 255) / 256 : (rows * a.heads + 3) / 4;
    if (few)
        cross_join_few_kernel<<<(unsigned)blocks, 256, 0, stream>>>(a, parts, rows);
    else
        cross_join_kernel<<<(unsigned)blocks, 256, 0, stream>>>(a, parts, rows, lanes);
    return hipGetLastError();
}

}  // namespace s2
