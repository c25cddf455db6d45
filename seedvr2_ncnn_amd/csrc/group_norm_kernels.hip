// Group norm of channels-last frames with an activation:
//   y[f][p][c] = act((x[f][p][c] - mean[f][g]) * rstd[f][g] * gamma[c] + beta[c]),
// g = c / (channels / groups), mean and variance over the pixels of a frame and
// the channels of a group.
//
// Bound by memory: x is read for the statistics and again for the result, which
// only caches can make cheaper than two passes.
//
// Statistics.  A thread sums x - K and (x - K)^2 of its channels over its pixels,
// K being its own first value of each channel: no cancellation where a mean is
// many deviations large, and one outlying K spoils a single thread's part at
// most.  Parts meet as (mean, sum of squared deviations) by the parallel variance
// formula (Chan, Golub, LeVeque), in double.  Every order of summation is fixed.
#include "group_norm_kernels.h"

#include <algorithm>

#include "activations.h"
#include "s2_device.h"

namespace s2 {

namespace {

constexpr int kThreads = 256;
constexpr int kMaxChannels = 4096;

// Frames whose groups hold at most this many values take one launch, a
// workgroup per frame and group.
constexpr long kSmallGroup = 16384;

template <int KIND>
struct Elem;
template <>
struct Elem<0> { typedef float T; };
template <>
struct Elem<1> { typedef uint16_t T; };
template <>
struct Elem<2> { typedef _Float16 T; };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(uint16_t v) { return bf16_to_f32(v); }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }

// V consecutive elements as floats; V elements are aligned to min(16, their size) bytes
template <int V, typename T>
__device__ __forceinline__ void load_v(const T* p, float (&v)[V]) {
    constexpr int B = V * (int)sizeof(T);
    if constexpr (V == 1) {
        v[0] = to_f32(*p);
    } else {
        alignas(16) T e[V];
        if constexpr (B == 8) {
            *reinterpret_cast<uint2*>(e) = *reinterpret_cast<const uint2*>(p);
        } else {
#pragma unroll
            for (int i = 0; i < B / 16; ++i)
                reinterpret_cast<uint4*>(e)[i] = reinterpret_cast<const uint4*>(p)[i];
        }
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f32(e[i]);
    }
}

template <int V, int KIND>
__device__ __forceinline__ void store_v(void* base, long idx, const float (&v)[V]) {
    if constexpr (V == 1) {
        if (KIND == 1)
            ((uint16_t*)base)[idx] = f32_to_bf16(v[0]);
        else if (KIND == 2)
            ((_Float16*)base)[idx] = f32_to_f16(v[0]);
        else
            ((float*)base)[idx] = v[0];
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4) store4(base, idx + i, v[i], v[i + 1], v[i + 2], v[i + 3], KIND);
    }
}

__device__ __forceinline__ double wave_sum(double v) {
#pragma unroll
    for (int o = 32; o; o >>= 1) v += __shfl_xor(v, o);
    return v;
}

// A chunk's (mean, sum of squared deviations) of every group:
// parts[frame][chunk][group].
template <int XK, int V>
__global__ __launch_bounds__(kThreads) void group_norm_stats_kernel(GroupNormArgs p, int chunk,
                                                                   float2* __restrict__ parts) {
    typedef typename Elem<XK>::T T;
    __shared__ float2 rows_lds[kThreads * V];
    __shared__ float2 chan_lds[kMaxChannels];
    const int tid = threadIdx.x;
    const int f = blockIdx.y;
    const long p0 = (long)blockIdx.x * chunk;
    const int np = (int)min((long)chunk, p.pixels - p0);
    const int cv = p.channels / V;
    const T* x = (const T*)p.x + f * p.x_frame + p0 * p.x_pixel;
    for (int c0 = 0; c0 < cv; c0 += kThreads) {
        const int seg = min(cv - c0, kThreads);   // vectors of channels in this sweep
        const int rows = kThreads / seg;
        const int row = tid / seg;
        const int col = tid - row * seg;
        if (row < rows && row < np) {
            const T* q = x + (long)row * p.x_pixel + (long)(c0 + col) * V;
            const long step = (long)rows * p.x_pixel;
            const int count = (np - row + rows - 1) / rows;
            float first[V], s1[V], s2[V], v[V];
            load_v<V>(q, first);
#pragma unroll
            for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
#pragma unroll 4
            for (int j = 1; j < count; ++j) {
                load_v<V>(q + j * step, v);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = v[i] - first[i];
                    s1[i] += d;
                    s2[i] = fmaf(d, d, s2[i]);
                }
            }
            const float inv = 1.f / (float)count;
#pragma unroll
            for (int i = 0; i < V; ++i)
                rows_lds[(row * seg + col) * V + i] =
                    make_float2(first[i] + s1[i] * inv, fmaxf(s2[i] - s1[i] * s1[i] * inv, 0.f));
        }
        __syncthreads();
        // the rows of each channel
        const int used = min(rows, np);
        for (int c = tid; c < seg * V; c += kThreads) {
            double sum = 0., m2 = 0.;
            for (int r = 0; r < used; ++r)
                sum += (double)((np - r + rows - 1) / rows) * rows_lds[r * seg * V + c].x;
            const double mean = sum / np;
            for (int r = 0; r < used; ++r) {
                const float2 e = rows_lds[r * seg * V + c];
                const double d = e.x - mean;
                m2 += e.y + (double)((np - r + rows - 1) / rows) * d * d;
            }
            chan_lds[c0 * V + c] = make_float2((float)mean, (float)m2);
        }
        __syncthreads();
    }
    // the channels of each group
    const int each = p.channels / p.groups;
    const int lane = tid & 63;
    for (int g = tid >> 6; g < p.groups; g += kThreads / 64) {
        double sum = 0.;
        for (int c = lane; c < each; c += 64) sum += chan_lds[g * each + c].x;
        const double mean = wave_sum(sum) / each;
        double m2 = 0.;
        for (int c = lane; c < each; c += 64) {
            const float2 e = chan_lds[g * each + c];
            const double d = e.x - mean;
            m2 += e.y + np * d * d;
        }
        m2 = wave_sum(m2);
        if (lane == 0)
            parts[((long)f * gridDim.x + blockIdx.x) * p.groups + g] = make_float2((float)mean, (float)m2);
    }
}

template <int XK, int YK, int V>
__global__ __launch_bounds__(kThreads) void group_norm_apply_kernel(GroupNormArgs p, int chunk,
                                                                   const float2* __restrict__ parts) {
    typedef typename Elem<XK>::T T;
    __shared__ float2 stat[kMaxChannels];   // (mean, rstd) of each group
    const int tid = threadIdx.x;
    const int f = blockIdx.y;
    const int chunks = gridDim.x;
    const int each = p.channels / p.groups;
    const int lane = tid & 63;
    const float2* fp = parts + (long)f * chunks * p.groups;
    for (int g = tid >> 6; g < p.groups; g += kThreads / 64) {
        double sum = 0.;
        for (int c = lane; c < chunks; c += 64)
            sum += (double)min((long)chunk, p.pixels - (long)c * chunk) * fp[(long)c * p.groups + g].x;
        const double mean = wave_sum(sum) / p.pixels;
        double m2 = 0.;
        for (int c = lane; c < chunks; c += 64) {
            const float2 e = fp[(long)c * p.groups + g];
            const double d = e.x - mean;
            m2 += e.y + (double)min((long)chunk, p.pixels - (long)c * chunk) * each * d * d;
        }
        m2 = wave_sum(m2);
        if (lane == 0)
            stat[g] = make_float2((float)mean,
                                  (float)(1. / sqrt(m2 / ((double)p.pixels * each) + (double)p.eps)));
    }
    __syncthreads();
    const long p0 = (long)blockIdx.x * chunk;
    const int np = (int)min((long)chunk, p.pixels - p0);
    const int cv = p.channels / V;
    const T* x = (const T*)p.x + f * p.x_frame + p0 * p.x_pixel;
    for (int c0 = 0; c0 < cv; c0 += kThreads) {
        const int seg = min(cv - c0, kThreads);
        const int rows = kThreads / seg;
        const int row = tid / seg;
        const int c = (c0 + tid - row * seg) * V;
        if (row >= rows) continue;
        float mean[V], scale[V], shift[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 s = stat[(c + i) / each];
            mean[i] = s.x;
            scale[i] = s.y * (p.gamma ? p.gamma[c + i] : 1.f);
            shift[i] = p.beta ? p.beta[c + i] : 0.f;
        }
#pragma unroll 4
        for (int j = row; j < np; j += rows) {
            float v[V];
            load_v<V>(x + (long)j * p.x_pixel + c, v);
#pragma unroll
            for (int i = 0; i < V; ++i) v[i] = activate(fmaf(v[i] - mean[i], scale[i], shift[i]), p.act);
            store_v<V, YK>(p.y, f * p.y_frame + (p0 + j) * p.y_pixel + c, v);
        }
    }
}

// How a frame's pixels are cut: enough workgroups to fill the chip, each with
// enough pixels to be worth its reductions.
int chunk_pixels(int frames, int pixels, int channels) {
    const long want = std::max<long>(1, 1024 / frames);                  // chunks of a frame
    const long least = std::max<long>(1, 16384 / channels);              // pixels of a chunk
    return (int)std::min<long>(pixels, std::max(least, (pixels + want - 1) / want));
}

template <int XK, int YK, int V>
hipError_t run(const GroupNormArgs& p, float2* parts, hipStream_t stream) {
    const int chunk = chunk_pixels(p.frames, p.pixels, p.channels);
    const dim3 grid((unsigned)((p.pixels + (long)chunk - 1) / chunk), (unsigned)p.frames);
    group_norm_stats_kernel<XK, V><<<grid, kThreads, 0, stream>>>(p, chunk, parts);
    group_norm_apply_kernel<XK, YK, V><<<grid, kThreads, 0, stream>>>(p, chunk, parts);
    return hipGetLastError();
}

// V consecutive channels are whole 16-byte pieces (8 bytes: four 16-bit ones)
// of every row of a view
bool fits(const void* base, int kind, long frame, long pixel, int v) {
    const int bytes = std::min(16, v * (kind ? 2 : 4));
    return (uintptr_t)base % bytes == 0 && frame % v == 0 && pixel % v == 0;
}

template <int XK, int YK>
hipError_t pick(const GroupNormArgs& p, float2* parts, hipStream_t stream) {
    for (int v : {8, 4})
        if (p.channels % v == 0 && fits(p.x, XK, p.x_frame, p.x_pixel, v) &&
            fits(p.y, YK, p.y_frame, p.y_pixel, v))
            return v == 8 ? run<XK, YK, 8>(p, parts, stream) : run<XK, YK, 4>(p, parts, stream);
    return run<XK, YK, 1>(p, parts, stream);
}

template <int XK>
hipError_t pick_y(const GroupNormArgs& p, float2* parts, hipStream_t stream) {
    return p.y_kind == 1   ? pick<XK, 1>(p, parts, stream)
           : p.y_kind == 2 ? pick<XK, 2>(p, parts, stream)
                           : pick<XK, 0>(p, parts, stream);
}

}  // namespace

size_t group_norm_workspace(int frames, int pixels, int channels, int groups) {
    if (frames <= 0 || pixels <= 0) return 0;
    const int chunk = chunk_pixels(frames, pixels, channels);
    return (size_t)frames * (size_t)((pixels + (long)chunk - 1) / chunk) * groups * sizeof(float2);
}

hipError_t launch_group_norm(const GroupNormArgs& p, void* workspace, hipStream_t stream) {
    if (p.frames <= 0 || p.pixels <= 0) return hipSuccess;
    return p.x_kind == 1   ? pick_y<1>(p, (float2*)workspace, stream)
           : p.x_kind == 2 ? pick_y<2>(p, (float2*)workspace, stream)
                           : pick_y<0>(p, (float2*)workspace, stream);
}

}  // namespace s2
