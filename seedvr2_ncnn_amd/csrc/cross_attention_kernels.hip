// Cross attention: softmax(scale q k^T) v per sample and head, keys of another length
// than the queries.
#include <cmath>

#include "cross_attention_device.h"

namespace s2 {

namespace {

// A wave a query and head, a lane every 64th element of d, key after key with the running
// maximum and sum.
__global__ __launch_bounds__(256) void cross_any_kernel(CrossArgs a) {
    const long item = (long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int h = (int)(item % a.heads);
    long i = item / a.heads;
    int b;
    long q0 = 0, k0 = 0, keys = a.lk;
    if (a.q_offsets) {
        if (i >= a.lq) return;
        for (b = 0; b < a.batch; ++b)
            if (i >= a.q_offsets[b] && i < a.q_offsets[b + 1]) break;
        if (b == a.batch) return;
        k0 = min(max(a.k_offsets[b], 0), a.lk);
        keys = min(max(a.k_offsets[b + 1], 0), a.lk) - k0;
    } else {
        if (i >= (long)a.batch * a.lq) return;
        b = (int)(i / a.lq);
        i -= (long)b * a.lq;
        if (a.key_lengths) keys = min(max(a.key_lengths[b], 0), a.lk);
    }
    const int hk = h / (a.heads / a.kv_heads);
    const long qa = b * a.qs.batch + (q0 + i) * a.qs.row + h * a.qs.head;
    float q[4], o[4] = {0.f, 0.f, 0.f, 0.f};
    for (int e = 0; e < 4; ++e) q[e] = lane + 64 * e < a.d ? load1(a.q, qa + lane + 64 * e, a.kind) : 0.f;
    float m = -__builtin_inff(), l = 0.f;
    for (long j = 0; j < keys; ++j) {
        if (a.key_mask && !a.key_mask[b * a.mask_batch + k0 + j]) continue;
        const long ka = b * a.ks.batch + (k0 + j) * a.ks.row + hk * a.ks.head;
        const long va = b * a.vs.batch + (k0 + j) * a.vs.row + hk * a.vs.head;
        float s = 0.f;
        for (int e = 0; e < 4; ++e)
            if (lane + 64 * e < a.d) s += q[e] * load1(a.k, ka + lane + 64 * e, a.kind);
        for (int x = 1; x < 64; x <<= 1) s += __shfl_xor(s, x);
        s *= a.scale;
        const float top = fmaxf(m, s);
        const float fade = m == top ? 1.f : expf(m - top);
        const float p = expf(s - (top == -__builtin_inff() ? 0.f : top));
        m = top;
        l = l * fade + p;
        for (int e = 0; e < 4; ++e)
            if (lane + 64 * e < a.d) o[e] = o[e] * fade + p * load1(a.v, va + lane + 64 * e, a.kind);
    }
    const long oa = b * a.os.batch + (q0 + i) * a.os.row + h * a.os.head;
    for (int e = 0; e < 4; ++e)
        if (lane + 64 * e < a.d) store1(a.out, oa + lane + 64 * e, l == 0.f ? 0.f : o[e] / l, a.out_kind);
}

// Four columns of a row a thread: its parts' sums, by how far their maxima lie below the
// largest.
__global__ __launch_bounds__(256) void cross_join_kernel(CrossArgs a, CrossParts p, long rows) {
    const int quads = a.d / 4;
    const long first = a.q_offsets ? clamped(a.q_offsets[0], a.lq) : 0;
    const long end = a.q_offsets ? clamped(a.q_offsets[a.batch], a.lq) : rows;
    for (long i = (long)blockIdx.x * 256 + threadIdx.x; i < rows * a.heads * quads; i += (long)gridDim.x * 256) {
        const long rh = i / quads;
        const int col = (int)(i - rh * quads) * 4;
        const long row = rh / a.heads;
        const int h = (int)(rh - row * a.heads);
        if (row < first || row >= end) continue;   // in no sample
        const float2* w = p.weights + rh * p.parts;
        float m = kLowest;
        for (int q = 0; q < p.parts; ++q) m = fmaxf(m, w[q].x);
        float l = 0.f;
        f32x4 o = {0.f, 0.f, 0.f, 0.f};
        for (int q = 0; q < p.parts; ++q) {
            const float f = __builtin_amdgcn_exp2f(w[q].x - m);
            l += f * w[q].y;
            o += f * *reinterpret_cast<const f32x4*>(p.sums + (rh * p.parts + q) * a.d + col);
        }
        const long b = a.q_offsets ? 0 : row / a.lq;
        const long at = b * a.os.batch + (row - b * a.lq) * a.os.row + h * a.os.head + col;
        store4_out(a, at, o * (l == 0.f ? 0.f : 1.f / l));
    }
}

long all_rows(const CrossArgs& a) { return a.q_offsets ? (long)a.lq : (long)a.batch * a.lq; }

size_t part_bytes(const CrossArgs& a) { return (size_t)all_rows(a) * a.heads * (a.d * sizeof(float) + sizeof(float2)); }

constexpr int kUnits = 256;   // compute units of an MI355X

// Microseconds that a compute unit takes for a tile of keys with 1, 2, .. workgroups on it,
// `each` at most, for d up to 64, 128 and 256: 4096 x 21600 with 20 heads of 128 in one
// range of keys is three workgroups on half of the units and two on the others, 899 us; in
// two ranges five in turn, 837.  1024 x 4096 96 us in one, 62 in three; 300 x 20000, two
// heads, 429 and 37 in 32.
struct CrossCost {
    int each;
    double us[4];
};
constexpr CrossCost kCrossCosts[] = {{4, {0.54, 0.7, 0.88, 1.1}}, {3, {0.7, 1.03, 1.43, 0.}}, {2, {1.45, 2.2, 0., 0.}}};
constexpr double kJoinUs = 4., kJoinBytesUs = 6e6;   // the joining launch; bytes written and read

CrossPlan cross_plan(const CrossArgs& a, size_t workspace_bytes) {
    const long group = a.heads / a.kv_heads;
    const long rows = (long)a.lq * group;
    CrossPlan p;
    p.tiles = (int)std::min<long>(a.q_offsets ? rows / kTileRows + std::min(a.batch, a.lq)
                                              : a.batch * ((rows + kTileRows - 1) / kTileRows),
                                  0x7fffffffL);
    // a sample's last tile is half empty, on average
    const double blocks = a.kv_heads * (a.q_offsets ? (double)rows / kTileRows + 0.5 * std::min(a.batch, a.lq)
                                                    : (double)p.tiles);
    const long keys = a.q_offsets ? ((long)a.lk + a.batch - 1) / std::max(a.batch, 1) : a.lk;   // of a sample
    const double tiles = (double)((keys + kTileKeys - 1) / kTileKeys);
    const long most = std::min<long>(64, (long)(workspace_bytes / part_bytes(a)));
    const CrossCost& c = kCrossCosts[a.d <= 64 ? 0 : a.d <= 128 ? 1 : 2];
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
    if (a.kind == 0) return 0;
    const CrossPlan p = cross_plan(a, (size_t)1 << 62);
    return p.parts > 1 ? p.parts * part_bytes(a) : 0;
}

hipError_t launch_cross_attention(const CrossArgs& a, void* workspace, size_t workspace_bytes,
                                  hipStream_t stream) {
    const long rows = all_rows(a);
    if (rows <= 0) return hipSuccess;
    if (a.kind) {
        const CrossPlan p = cross_plan(a, workspace_bytes);
        if ((long)p.tiles * a.kv_heads * p.parts > 0x7fffffffL) return hipErrorInvalidValue;
        const hipError_t e = launch_cross_tiles(a, p, workspace, stream);
        if (e != hipSuccess || p.parts == 1) return e;
        const long all = rows * a.heads * (a.d / 4);
        cross_join_kernel<<<(unsigned)std::min<long>((all + 255) / 256, 8192), 256, 0, stream>>>(
            a, cross_parts(a, p, workspace), rows);
        return hipGetLastError();
    }
    const long blocks = (rows * a.heads + 3) / 4;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    cross_any_kernel<<<(unsigned)blocks, 256, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace s2
