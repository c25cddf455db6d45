// Group norm of channels-last frames with an activation:
//   y[f][p][c] = act((x[f][p][c] - mean[f][g]) * rstd[f][g] * gamma[c] + beta[c]),
// g = c / (channels / groups), mean and variance over the pixels of a frame and
// the channels of a group.
//
// Bound by memory: x is read for the statistics and again for the result, which
// only caches can make cheaper than two passes; groups of few values are held in
// registers between the two.
//
// Statistics.  A thread sums x - K and (x - K)^2 of its channels over its pixels,
// K being its own first value of each channel: no cancellation where a mean is
// many deviations large, and one outlying K spoils a single thread's part at
// most.  Parts meet as (mean, sum of squared deviations) by the parallel variance
// formula (Chan, Golub, LeVeque).  Every order of summation is fixed.
#include "group_norm_kernels.h"

#include <algorithm>

#include "activations.h"
#include "s2_device.h"

namespace s2 {

namespace {

constexpr int kMaxChannels = 4096;

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

// Sum over aligned runs of `lanes` lanes, a power of two.
__device__ __forceinline__ float lanes_sum(float v, int lanes) {
    for (int o = 1; o < lanes; o <<= 1) v += __shfl_xor(v, o);
    return v;
}

// Lanes that share a group's sums: a power of two, at most a wave, that lets all the
// groups have theirs at once where there are enough.
__device__ __forceinline__ int lanes_per_group(int groups, int threads) {
    int l = 64;
    while (l > 1 && l * groups > threads) l >>= 1;
    return l;
}

// The division of a chunk's pixels and channels among the threads: `seg` vectors of V
// channels side by side, `rows` pixels at once.  More vectors than threads: sweeps of
// one pixel row each.
struct Split {
    int cv, seg, rows;
    __device__ Split(int channels, int v, int threads) {
        cv = channels / v;
        seg = min(cv, threads);
        rows = cv > threads ? 1 : threads / seg;
    }
};

constexpr int kThreads = 512;

// A chunk's (mean, sum of squared deviations) of every group: parts[frame][group][chunk].
template <int XK, int V>
__global__ __launch_bounds__(kThreads) void group_norm_stats_kernel(GroupNormArgs p, int chunk,
                                                                   float2* __restrict__ parts) {
    typedef typename Elem<XK>::T T;
    constexpr int ENTRIES = kThreads * V > kMaxChannels ? kThreads * V : kMaxChannels;
    __shared__ float2 entry[ENTRIES];   // [row][channel]
    const int tid = threadIdx.x;
    const int f = blockIdx.y;
    const long p0 = (long)blockIdx.x * chunk;
    const int np = (int)min((long)chunk, p.pixels - p0);
    const Split sp(p.channels, V, kThreads);
    const int row = tid / sp.seg;
    const int col = tid - row * sp.seg;
    const int base = np / sp.rows, extra = np - base * sp.rows;   // pixels of a row
    const T* x = (const T*)p.x + f * p.x_frame + p0 * p.x_pixel + (long)row * p.x_pixel;
    const int count = row < sp.rows ? base + (row < extra) : 0;
    const long step = (long)sp.rows * p.x_pixel;
    for (int c = col; c < sp.cv && count > 0; c += sp.seg) {
        const T* q = x + (long)c * V;
        float first[V], s1[V], s2[V];
        load_v<V>(q, first);
#pragma unroll
        for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
#pragma unroll 8
        for (int j = 1; j < count; ++j) {
            float v[V];
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
            entry[row * p.channels + c * V + i] =
                make_float2(fmaf(s1[i], inv, first[i]), fmaxf(fmaf(-s1[i] * inv, s1[i], s2[i]), 0.f));
    }
    __syncthreads();
    const int each = p.channels / p.groups;
    const int used = min(sp.rows, np);
    const int lanes = lanes_per_group(p.groups, kThreads);
    const int lane = tid & (lanes - 1);
    const float per_value = 1.f / ((float)np * (float)each);
    for (int g0 = 0; g0 < p.groups; g0 += kThreads / lanes) {   // the same count in every thread
        const int g = g0 + tid / lanes;
        const float2* e = entry + g * each;
        const float ref = g < p.groups ? e[0].x : 0.f;
        float sum = 0.f;
        if (g < p.groups)
            for (int r = 0; r < used; ++r) {
                const float n = (float)(base + (r < extra));
                for (int c = lane; c < each; c += lanes) sum = fmaf(n, e[r * p.channels + c].x - ref, sum);
            }
        const float mean = fmaf(lanes_sum(sum, lanes), per_value, ref);
        float m2 = 0.f;
        if (g < p.groups)
            for (int r = 0; r < used; ++r) {
                const float n = (float)(base + (r < extra));
                for (int c = lane; c < each; c += lanes) {
                    const float2 v = e[r * p.channels + c];
                    const float d = v.x - mean;
                    m2 += fmaf(n * d, d, v.y);
                }
            }
        m2 = lanes_sum(m2, lanes);
        if (g < p.groups && lane == 0)
            parts[((long)f * p.groups + g) * gridDim.x + blockIdx.x] = make_float2(mean, m2);
    }
}

template <int XK, int YK, int V>
__global__ __launch_bounds__(kThreads) void group_norm_apply_kernel(GroupNormArgs p, int part_chunk,
                                                                   int chunks, int chunk,
                                                                   const float2* __restrict__ parts) {
    typedef typename Elem<XK>::T T;
    __shared__ float2 stat[kMaxChannels];   // (mean, rstd) of each group
    const int tid = threadIdx.x;
    const int f = blockIdx.y;
    const int each = p.channels / p.groups;
    const int lanes = lanes_per_group(p.groups, kThreads);
    const int lane = tid & (lanes - 1);
    for (int g0 = 0; g0 < p.groups; g0 += kThreads / lanes) {
        const int g = g0 + tid / lanes;
        const float2* e = parts + ((long)f * p.groups + min(g, p.groups - 1)) * chunks;
        // deviations from the first part's mean: as far from it as the parts are from
        // one another
        const float ref = e[0].x;
        float sum = 0.f, sq = 0.f, m2 = 0.f;
#pragma unroll 4
        for (int c = lane; c < chunks; c += lanes) {
            const float2 v = e[c];
            const float n = (float)min((long)part_chunk, p.pixels - (long)c * part_chunk);
            const float d = v.x - ref;
            sum = fmaf(n, d, sum);
            sq = fmaf(n * d, d, sq);
            m2 += v.y;
        }
        sum = lanes_sum(sum, lanes);
        sq = lanes_sum(sq, lanes);
        m2 = lanes_sum(m2, lanes);
        if (g < p.groups && lane == 0) {
            const float mean = sum / (float)p.pixels;
            const float var = (fmaxf(fmaf(-mean, sum, sq), 0.f) * (float)each + m2) /
                              ((float)p.pixels * (float)each);
            // an infinity or NaN in any part makes m2 NaN
            stat[g] = make_float2(ref + mean, 1.f / sqrtf(var + p.eps));
        }
    }
    __syncthreads();
    const long p0 = (long)blockIdx.x * chunk;
    const int np = (int)min((long)chunk, p.pixels - p0);
    const Split sp(p.channels, V, kThreads);
    const int row = tid / sp.seg;
    const int col = tid - row * sp.seg;
    if (row >= sp.rows) return;
    const T* x = (const T*)p.x + f * p.x_frame + p0 * p.x_pixel;
    const long y0 = f * p.y_frame + p0 * p.y_pixel;
    for (int cc = col; cc < sp.cv; cc += sp.seg) {
        const int c = cc * V;
        float mean[V], scale[V], shift[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 s = stat[(c + i) / each];
            mean[i] = s.x;
            scale[i] = s.y * (p.gamma ? p.gamma[c + i] : 1.f);
            shift[i] = p.beta ? p.beta[c + i] : 0.f;
        }
        constexpr int U = 4;   // pixels in flight
        for (int j = row; j < np; j += U * sp.rows) {
            float v[U][V];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j + u * sp.rows < np) load_v<V>(x + (long)(j + u * sp.rows) * p.x_pixel + c, v[u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (j + u * sp.rows < np) {
#pragma unroll
                    for (int i = 0; i < V; ++i)
                        v[u][i] = activate(fmaf(v[u][i] - mean[i], scale[i], shift[i]), p.act);
                    store_v<V, YK>(p.y, y0 + (long)(j + u * sp.rows) * p.y_pixel + c, v[u]);
                }
        }
    }
}

// Few values: a workgroup holds a frame's group in registers, one launch in all.  The
// mean first, then the deviations from it.
constexpr int kSmallThreads = 256;
constexpr int kSmallVectors = 8;   // of a thread

__device__ __forceinline__ float block_sum(float v, float* lds) {
    v = lanes_sum(v, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < kSmallThreads / 64; ++i) v += lds[i];
    return v;
}

template <int XK, int YK, int V>
__global__ __launch_bounds__(kSmallThreads) void group_norm_small_kernel(GroupNormArgs p) {
    typedef typename Elem<XK>::T T;
    __shared__ float lds[2][kSmallThreads / 64];
    const int f = blockIdx.y, g = blockIdx.x;
    const int each = p.channels / p.groups;
    const int ev = each / V;   // vectors of a pixel
    const int all = p.pixels * ev;
    const T* x = (const T*)p.x + f * p.x_frame + (long)g * each;
    float v[kSmallVectors][V];
    int pix[kSmallVectors], ch[kSmallVectors];
#pragma unroll
    for (int u = 0; u < kSmallVectors; ++u) {
        const int i = threadIdx.x + u * kSmallThreads;
        pix[u] = i / ev;
        ch[u] = (i - pix[u] * ev) * V;
        if (i < all) load_v<V>(x + pix[u] * p.x_pixel + ch[u], v[u]);
    }
    // deviations from the first value: no digits are lost to a large mean
    const float ref = to_f32(*x);
    float sum = 0.f;
#pragma unroll
    for (int u = 0; u < kSmallVectors; ++u)
        if (threadIdx.x + u * kSmallThreads < all)
#pragma unroll
            for (int i = 0; i < V; ++i) sum += v[u][i] - ref;
    const float count = (float)all * V;
    const float mean = ref + block_sum(sum, lds[0]) / count;
    float m2 = 0.f;
#pragma unroll
    for (int u = 0; u < kSmallVectors; ++u)
        if (threadIdx.x + u * kSmallThreads < all)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = v[u][i] - mean;
                m2 = fmaf(d, d, m2);
            }
    const float rstd = 1.f / sqrtf(block_sum(m2, lds[1]) / count + p.eps);
#pragma unroll
    for (int u = 0; u < kSmallVectors; ++u)
        if (threadIdx.x + u * kSmallThreads < all) {
            const int c = g * each + ch[u];
#pragma unroll
            for (int i = 0; i < V; ++i)
                v[u][i] = activate(fmaf(v[u][i] - mean, rstd * (p.gamma ? p.gamma[c + i] : 1.f),
                                        p.beta ? p.beta[c + i] : 0.f),
                                   p.act);
            store_v<V, YK>(p.y, f * p.y_frame + pix[u] * p.y_pixel + c, v[u]);
        }
}

// V channels are whole 16-byte pieces (8 bytes: four 16-bit ones) of every row of a view
bool fits(const void* base, int kind, long frame, long pixel, int v) {
    const int bytes = std::min(16, v * (kind ? 2 : 4));
    return (uintptr_t)base % bytes == 0 && frame % v == 0 && pixel % v == 0;
}

bool fits(const GroupNormArgs& p, int width, int v) {
    return width % v == 0 && fits(p.x, p.x_kind, p.x_frame, p.x_pixel, v) &&
           fits(p.y, p.y_kind, p.y_frame, p.y_pixel, v);
}

// How a frame's pixels are cut: into at most 256 chunks, whose parts every workgroup of
// the second kernel reads, and about 512 workgroups in all.
int chunk_pixels(int frames, int pixels, int channels) {
    const long want = std::min<long>(256, std::max<long>(1, 512 / frames));   // chunks of a frame
    const long least = std::max<long>(1, 8192 / channels);                    // pixels of a chunk
    return (int)std::min<long>(pixels, std::max(least, (pixels + want - 1) / want));
}

long chunks_of(int pixels, int chunk) { return ((long)pixels + chunk - 1) / chunk; }

template <int XK, int YK, int V>
hipError_t run(const GroupNormArgs& p, float2* parts, hipStream_t stream) {
    const int part = chunk_pixels(p.frames, p.pixels, p.channels);
    const int chunks = (int)chunks_of(p.pixels, part);
    group_norm_stats_kernel<XK, V>
        <<<dim3((unsigned)chunks, (unsigned)p.frames), kThreads, 0, stream>>>(p, part, parts);
    const int chunk = part;
    group_norm_apply_kernel<XK, YK, V>
        <<<dim3((unsigned)chunks_of(p.pixels, chunk), (unsigned)p.frames), kThreads, 0, stream>>>(
            p, part, chunks, chunk, parts);
    return hipGetLastError();
}

template <int XK, int YK>
hipError_t pick(const GroupNormArgs& p, float2* parts, hipStream_t stream) {
    const int each = p.channels / p.groups;
    for (int v : {8, 4, 1}) {
        if (v > 1 && !fits(p, each, v)) continue;
        if ((long)p.pixels * (each / v) > kSmallThreads * kSmallVectors) break;
        const dim3 grid((unsigned)p.groups, (unsigned)p.frames);
        if (v == 8)
            group_norm_small_kernel<XK, YK, 8><<<grid, kSmallThreads, 0, stream>>>(p);
        else if (v == 4)
            group_norm_small_kernel<XK, YK, 4><<<grid, kSmallThreads, 0, stream>>>(p);
        else
            group_norm_small_kernel<XK, YK, 1><<<grid, kSmallThreads, 0, stream>>>(p);
        return hipGetLastError();
    }
    if (fits(p, p.channels, 8)) return run<XK, YK, 8>(p, parts, stream);
    if (fits(p, p.channels, 4)) return run<XK, YK, 4>(p, parts, stream);
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
    return (size_t)frames * (size_t)chunks_of(pixels, chunk) * groups * sizeof(float2);
}

hipError_t launch_group_norm(const GroupNormArgs& args, void* workspace, hipStream_t stream) {
    if (args.frames <= 0 || args.pixels <= 0) return hipSuccess;
    GroupNormArgs p = args;
    if (p.frames == 1) p.x_frame = p.y_frame = 0;   // strides of single ones say nothing
    if (p.pixels == 1) p.x_pixel = p.y_pixel = 0;
    return p.x_kind == 1   ? pick_y<1>(p, (float2*)workspace, stream)
           : p.x_kind == 2 ? pick_y<2>(p, (float2*)workspace, stream)
                           : pick_y<0>(p, (float2*)workspace, stream);
}

}  // namespace s2
