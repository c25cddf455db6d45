// Cross attention: softmax(scale q k^T) v per sample and head, keys of another length
// than the queries.
#include "cross_attention_kernels.h"
#include "matmul_device.h"

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

}  // namespace

size_t cross_attention_workspace(const CrossArgs&) { return 0; }

hipError_t launch_cross_attention(const CrossArgs& a, void*, size_t, hipStream_t stream) {
    const long rows = a.q_offsets ? (long)a.lq : (long)a.batch * a.lq;
    const long blocks = (rows * a.heads + 3) / 4;
    if (blocks <= 0) return hipSuccess;
    if (blocks > 0x7fffffffL) return hipErrorInvalidValue;
    cross_any_kernel<<<(unsigned)blocks, 256, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace s2
