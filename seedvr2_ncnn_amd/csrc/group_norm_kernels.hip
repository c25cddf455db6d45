// Group norm of channels-last frames with an activation:
//   y[f][p][c] = act((x[f][p][c] - mean[f][g]) * rstd[f][g] * gamma[c] + beta[c]),
// g = c / (channels / groups), mean and variance over the pixels of a frame and
// the channels of a group.
//
// Bound by memory: x is read for the statistics and again for the result, which
// only caches can make cheaper than two passes; groups of few values are held in
// registers between the two.
//
// Statistics.  A thread sums x - K and (x - K)^2 of its channels over eight of its
// pixels, K being the first of them: no cancellation where a mean is many deviations
// large, and a K far from all others, whose square the difference of the two sums would
// lose digits of, stands against seven values only (against all of a thread's 450 it
// left a frame's variance off by 3e-3, now 2e-6).  Those sums and all parts after them
// meet as (mean, sum of squared deviations) by the parallel variance formula (Chan,
// Golub, LeVeque).  Every order of summation is fixed.
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

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));
// in memory
typedef u32x2 u32x2_at4 __attribute__((aligned(4)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
typedef f32x4 f32x4_at4 __attribute__((aligned(4)));

// V consecutive elements as they lie in memory
template <typename T, int V>
struct Raw {
    alignas(V * sizeof(T) > 16 ? 16 : V * sizeof(T)) T e[V];
    __device__ __forceinline__ void load(const T* p) {
        // vectors lie on four bytes (on two they take several times as long)
        __builtin_memcpy(e, V > 1 ? __builtin_assume_aligned(p, 4) : p, sizeof(e));
    }
    __device__ __forceinline__ void get(float (&v)[V]) const {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = to_f32(e[i]);
    }
};

template <bool NT, typename P, typename Q>
__device__ __forceinline__ void put(P* at, Q q) {
    if constexpr (NT)
        __builtin_nontemporal_store(q, at);
    else
        *at = q;
}

template <int V, int KIND, bool NT = false>
__device__ __forceinline__ void store_v(void* base, long idx, const float (&v)[V]) {
    if constexpr (V == 1) {
        if (KIND == 1)
            ((uint16_t*)base)[idx] = f32_to_bf16(v[0]);
        else if (KIND == 2)
            ((_Float16*)base)[idx] = f32_to_f16(v[0]);
        else
            ((float*)base)[idx] = v[0];
    } else if constexpr (KIND != 0) {
        uint32_t w[V / 2];
#pragma unroll
        for (int i = 0; i < V / 2; ++i)
            w[i] = KIND == 1 ? pack2_bf16_rne(v[2 * i], v[2 * i + 1]) : pack2_f16_rne(v[2 * i], v[2 * i + 1]);
        if constexpr (V == 2) {
            put<NT>((u32_any*)((uint16_t*)base + idx), w[0]);
        } else if constexpr (V == 4) {
            put<NT>((u32x2_at4*)((uint16_t*)base + idx), u32x2{w[0], w[1]});
        } else {
            put<NT>((u32x4_at4*)((uint16_t*)base + idx), u32x4{w[0], w[1], w[2], w[3]});
        }
    } else if constexpr (V == 2) {
        put<NT>((u32x2_at4*)((float*)base + idx), u32x2{__float_as_uint(v[0]), __float_as_uint(v[1])});
    } else {
#pragma unroll
        for (int i = 0; i < V; i += 4)
            put<NT>((f32x4_at4*)((float*)base + idx + i), f32x4{v[i], v[i + 1], v[i + 2], v[i + 3]});
    }
}

// Sum over aligned runs of 2^bits lanes, the same bits in every lane.  Within a row of
// 16 by DPP moves (quad permutations, then the half-row and row mirrors, whose lanes
// hold the same partial sums as lane ^ 4 and lane ^ 8): no LDS round trips.
template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xF, 0xF, false));
}

__device__ __forceinline__ float lanes_sum(float v, int bits) {
    if (bits > 0) v += dpp_move<0xB1>(v);
    if (bits > 1) v += dpp_move<0x4E>(v);
    if (bits > 2) v += dpp_move<0x141>(v);
    if (bits > 3) v += dpp_move<0x140>(v);
    if (bits > 4) v += __shfl_xor(v, 16);
    if (bits > 5) v += __shfl_xor(v, 32);
    return v;
}

constexpr int kThreads = 512;

// How a workgroup's threads divide a chunk, made on the host: `seg` vectors of V
// channels side by side and `rows` pixels at once (more vectors than threads: one
// pixel, in sweeps), and 2^lane_bits lanes that share a group's sums, at most a wave,
// as many as let all the groups have theirs at once where that can be.
struct Split {
    int cv, seg, rows;
    int inv_seg;     // thread / seg = thread * inv_seg >> 20
    int lane_bits;
    Split(int channels, int groups, int v) {
        cv = channels / v;
        seg = std::min(cv, kThreads);
        rows = cv > kThreads ? 1 : kThreads / seg;
        inv_seg = (1 << 20) / seg + 1;   // exact below 2^20 / seg threads
        lane_bits = 6;
        while (lane_bits > 0 && (groups << lane_bits) > kThreads) --lane_bits;
    }
};

// A thread's (mean, sum of squared deviations) of V channels, in two floats each: as
// many joinings as a thread has pixels would round them otherwise.
template <int V>
struct Part {
    float mean[V], mean_rest[V], m2[V], m2_rest[V];

    // `count` pixels of raw, at most U, to the `before` that are in
    template <int U, typename T>
    __device__ __forceinline__ void add(const Raw<T, V> (&raw)[U], int count, int before) {
        float first[V], s1[V], s2[V];
        raw[0].get(first);
        if (before == 0)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                mean[i] = first[i];
                mean_rest[i] = m2[i] = m2_rest[i] = 0.f;
            }
#pragma unroll
        for (int i = 0; i < V; ++i) s1[i] = s2[i] = 0.f;
#pragma unroll
        for (int u = 1; u < U; ++u)
            if (u < count) {
                float v[V];
                raw[u].get(v);
#pragma unroll
                for (int i = 0; i < V; ++i) {
                    const float d = v[i] - first[i];
                    s1[i] += d;
                    s2[i] = fmaf(d, d, s2[i]);
                }
            }
        const float share = (float)count / (float)(before + count), each = 1.f / (float)count;
        const float weight = share * (float)before;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float off = s1[i] * each;   // of these pixels' mean from the first
            const float own = fmaxf(fmaf(-off, s1[i], s2[i]), 0.f);
            const float d = (first[i] - mean[i]) + (off - mean_rest[i]);
            const float step = d * share, sum = mean[i] + step;
            mean_rest[i] += (mean[i] - sum) + step;
            mean[i] = sum;
            const float more = fmaf(d * weight, d, own), total = m2[i] + more;
            m2_rest[i] += (m2[i] - total) + more;
            m2[i] = total;
        }
    }
};

// A chunk's (mean, sum of squared deviations) of every group: parts[frame][group][chunk].
// A thread joins runs of SUB of its channels, which divides a group's.
template <int XK, int V, int SUB>
__global__ __launch_bounds__(kThreads) void group_norm_stats_kernel(GroupNormArgs p, Split sp,
                                                                   int chunk,
                                                                   float2* __restrict__ parts) {
    typedef typename Elem<XK>::T T;
    constexpr int ENTRIES = (kThreads * V > kMaxChannels ? kThreads * V : kMaxChannels) / SUB;
    __shared__ float2 entry[ENTRIES];   // [row][run of channels]
    const int runs = p.channels / SUB;
    const int tid = threadIdx.x;
    const int f = blockIdx.y;
    const long p0 = (long)blockIdx.x * chunk;
    const int np = (int)min((long)chunk, p.pixels - p0);
    const int row = tid * sp.inv_seg >> 20;
    const int col = tid - row * sp.seg;
    const int base = np / sp.rows, extra = np - base * sp.rows;   // pixels of a row
    const T* x = (const T*)p.x + f * p.x_frame + p0 * p.x_pixel + (long)row * p.x_pixel;
    const int count = row < sp.rows ? base + (row < extra) : 0;
    const long step = (long)sp.rows * p.x_pixel;
    for (int c = col; c < sp.cv && count > 0; c += sp.seg) {
        const T* q = x + (long)c * V;
        Part<V> part;
        constexpr int U = 8;   // pixels in flight
        Raw<T, V> raw[U];
        int j = 0;
        for (; j + U <= count; j += U) {
#pragma unroll
            for (int u = 0; u < U; ++u) raw[u].load(q + (j + u) * step);
            part.template add<U>(raw, U, j);
        }
        if (j < count) {
#pragma unroll
            for (int u = 0; u < U - 1; ++u)
                if (j + u < count) raw[u].load(q + (j + u) * step);
            part.template add<U>(raw, count - j, j);
        }
        const float n = (float)count;
        float first[V], s2[V];   // mean and sum of squared deviations
#pragma unroll
        for (int i = 0; i < V; ++i) {
            first[i] = part.mean[i] + part.mean_rest[i];
            s2[i] = part.m2[i] + part.m2_rest[i];
        }
#pragma unroll
        for (int i = 0; i < V; i += SUB) {
            float off = 0.f, m2 = 0.f;
#pragma unroll
            for (int e = 1; e < SUB; ++e) off += first[i + e] - first[i];
            const float mean = fmaf(off, 1.f / SUB, first[i]);
#pragma unroll
            for (int e = 0; e < SUB; ++e) {
                const float d = SUB > 1 ? first[i + e] - mean : 0.f;
                m2 += fmaf(n * d, d, s2[i + e]);
            }
            entry[row * runs + (c * V + i) / SUB] = make_float2(mean, m2);
        }
    }
    __syncthreads();
    const int each = runs / p.groups;   // runs of a group
    const int used = min(sp.rows, np);
    const int lanes = 1 << sp.lane_bits;
    // of a group's lanes, `across` take neighbouring runs, the others rows
    const int across_bits = min(sp.lane_bits, 32 - __clz(each - 1));
    const int across = 1 << across_bits;
    const int lane = tid & (lanes - 1);
    const int c0 = lane & (across - 1), r0 = lane >> across_bits, dr = lanes >> across_bits;
    const float per_run = 1.f / ((float)np * (float)each);
    for (int g0 = 0; g0 < p.groups; g0 += kThreads >> sp.lane_bits) {   // as often in every thread
        const int g = g0 + (tid >> sp.lane_bits);
        const float2* e = entry + min(g, p.groups - 1) * each;
        const float ref = e[0].x;
        float sum = 0.f;
        for (int c = c0; c < each; c += across)
#pragma unroll 4
            for (int r = r0; r < used; r += dr)
                sum = fmaf((float)(base + (r < extra)), e[r * runs + c].x - ref, sum);
        const float mean = fmaf(lanes_sum(sum, sp.lane_bits), per_run, ref);
        float m2 = 0.f;
        sum = 0.f;   // what the mean is off by, where ref is far from it
        for (int c = c0; c < each; c += across)
#pragma unroll 4
            for (int r = r0; r < used; r += dr) {
                const float2 v = e[r * runs + c];
                const float n = (float)(base + (r < extra)), d = v.x - mean;
                sum = fmaf(n, d, sum);
                m2 += fmaf(n * (float)SUB * d, d, v.y);
            }
        m2 = lanes_sum(m2, sp.lane_bits);
        sum = lanes_sum(sum, sp.lane_bits);
        if (g < p.groups && lane == 0)
            parts[((long)f * p.groups + g) * gridDim.x + blockIdx.x] =
                make_float2(fmaf(sum, per_run, mean), m2);
    }
}

// V consecutive values of gamma or beta, or `none` without one
template <int V>
__device__ __forceinline__ void load_affine(const float* p, int c, float none, float (&v)[V]) {
    if (!p) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = none;
    } else {
        __builtin_memcpy(v, p + c, sizeof(v));
    }
}

// y.  Frames and chunks in the reverse of the first kernel's order, and stores that pass
// the caches by: what of x was read last is still there to be read again (118 MB of x:
// 66 us, 82 with plain stores; 944 MB: 528 against 542).
template <int XK, int YK, int V>
__global__ __launch_bounds__(kThreads) void group_norm_apply_kernel(GroupNormArgs p, Split sp,
                                                                   int part_chunk, int chunks,
                                                                   int chunk,
                                                                   const float2* __restrict__ parts) {
    typedef typename Elem<XK>::T T;
    __shared__ float2 stat[kMaxChannels];   // (mean, rstd) of each group
    const int tid = threadIdx.x;
    const int f = gridDim.y - 1 - blockIdx.y;
    const int each = p.channels / p.groups;
    const long p0 = (long)(gridDim.x - 1 - blockIdx.x) * chunk;
    const int np = (int)min((long)chunk, p.pixels - p0);
    const int row = tid * sp.inv_seg >> 20;
    const int col = tid - row * sp.seg;
    const T* x = (const T*)p.x + f * p.x_frame + p0 * p.x_pixel;
    constexpr int U = 4;   // pixels in flight
    Raw<T, V> raw[U];
    // (pixels past the end repeat the last one)
    auto fetch = [&](int c, int j) {
#pragma unroll
        for (int u = 0; u < U; ++u) raw[u].load(x + (long)min(j + u * sp.rows, np - 1) * p.x_pixel + c);
    };
    float scale[V], shift[V];
    auto affine = [&](int c) {
        load_affine<V>(p.gamma, c, 1.f, scale);
        load_affine<V>(p.beta, c, 0.f, shift);
    };
    const int lanes = 1 << sp.lane_bits;
    const int lane = tid & (lanes - 1);
    const float whole = (float)part_chunk;
    const float rest = (float)(p.pixels - (long)(chunks - 1) * part_chunk);   // the last part
    for (int g0 = 0; g0 < p.groups; g0 += kThreads >> sp.lane_bits) {
        const int g = g0 + (tid >> sp.lane_bits);
        const float2* e = parts + ((long)f * p.groups + min(g, p.groups - 1)) * chunks;
        const float ref = e[0].x;
        constexpr int C = 4;   // parts in flight
        float2 v[C];
        auto get = [&](int i0) {
#pragma unroll
            for (int c = 0; c < C; ++c) v[c] = e[min(i0 + c * lanes, chunks - 1)];
        };
        auto pixels = [&](int at) { return at + 1 < chunks ? whole : at + 1 == chunks ? rest : 0.f; };
        get(lane);
        if (g0 == 0) {
            // once the parts are there, the thread's first pixels: under the arithmetic
#pragma unroll
            for (int c = 0; c < C; ++c) asm volatile("" : "+v"(v[c].x), "+v"(v[c].y)::"memory");
            fetch(col * V, row);
            affine(col * V);
        }
        float sum = 0.f, m2 = 0.f;
        for (int i0 = lane;;) {
#pragma unroll
            for (int c = 0; c < C; ++c) sum = fmaf(pixels(i0 + c * lanes), v[c].x - ref, sum);
            i0 += C * lanes;
            if (i0 >= chunks) break;
            get(i0);
        }
        const float off = lanes_sum(sum, sp.lane_bits) / (float)p.pixels;   // of the mean from ref
        if (chunks > C * lanes) get(lane);
        for (int i0 = lane;;) {
#pragma unroll
            for (int c = 0; c < C; ++c) {
                const int at = i0 + c * lanes;
                const float d = v[c].x - ref - off;
                m2 += at < chunks ? fmaf(pixels(at) * (float)each * d, d, v[c].y) : 0.f;
            }
            i0 += C * lanes;
            if (i0 >= chunks) break;
            get(i0);
        }
        m2 = lanes_sum(m2, sp.lane_bits);
        if (g < p.groups && lane == 0) {
            const float var = m2 / ((float)p.pixels * (float)each);
            stat[g] = make_float2(ref + off, 1.f / sqrtf(var + p.eps));
        }
    }
    __syncthreads();
    if (row >= sp.rows) return;
    const long y0 = f * p.y_frame + p0 * p.y_pixel;
    for (int cc = col; cc < sp.cv; cc += sp.seg) {
        const int c = cc * V;
        if (cc != col) {
            fetch(c, row);
            affine(c);
        }
        float mean[V];
        int g = c / each, in = c - g * each;
#pragma unroll
        for (int i = 0; i < V; ++i) {
            const float2 st = stat[g];
            mean[i] = st.x;
            scale[i] *= st.y;
            if (++in == each) {
                in = 0;
                ++g;
            }
        }
        with_activation(p.act, [&](auto act) {
            for (int j = row; j < np; j += U * sp.rows) {
                float v[U][V];
#pragma unroll
                for (int u = 0; u < U; ++u) raw[u].get(v[u]);
                if (j + U * sp.rows < np) fetch(c, j + U * sp.rows);
#pragma unroll
                for (int u = 0; u < U; ++u)
                    if (j + u * sp.rows < np) {
#pragma unroll
                        for (int i = 0; i < V; ++i)
                            v[u][i] = activate<YK == 0>(fmaf(v[u][i] - mean[i], scale[i], shift[i]),
                                                        decltype(act)::value);
                        store_v<V, YK, true>(p.y, y0 + (long)(j + u * sp.rows) * p.y_pixel + c, v[u]);
                    }
            }
        });
    }
}

// Few values: a workgroup holds a frame's group in registers, one launch in all.  The
// mean first, from deviations from the first value; then the deviations from it, whose
// own mean corrects it where the first value is far from it.
// A thread holds up to 4 vectors of 8, or 8 of 4, 2 or 1; 256 threads, or 1024 (2000 x 512
// in bf16 in 32 groups 7.3 us, 12 by two launches; 4000 x 512 with 8 vectors of 8 a
// thread 16.6 and 13: the group's pieces of 32 bytes come to one compute unit).
constexpr int kSmallMost = 1024;   // threads
constexpr int small_vectors(int v) { return v == 8 ? 4 : 8; }

template <int THREADS, int N>
__device__ __forceinline__ void block_sum(float (&v)[N], float (*lds)[THREADS / 64]) {
#pragma unroll
    for (int j = 0; j < N; ++j) {
        v[j] = lanes_sum(v[j], 6);
        if ((threadIdx.x & 63) == 0) lds[j][threadIdx.x >> 6] = v[j];
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < N; ++j) {
        v[j] = 0.f;
#pragma unroll
        for (int i = 0; i < THREADS / 64; ++i) v[j] += lds[j][i];
    }
}

template <int XK, int YK, int V, int THREADS>
__global__ __launch_bounds__(THREADS) void group_norm_small_kernel(GroupNormArgs p) {
    typedef typename Elem<XK>::T T;
    constexpr int VECS = small_vectors(V);
    __shared__ float lds[3][THREADS / 64];
    const int f = blockIdx.y, g = blockIdx.x;
    const int each = p.channels / p.groups;
    const int ev = each / V;   // vectors of a pixel, at most the threads
    const int rows = THREADS / ev;
    const int row = threadIdx.x / ev;
    const int c = g * each + (threadIdx.x - row * ev) * V;
    const int count = row < rows ? (p.pixels - row + rows - 1) / rows : 0;   // of this thread
    const T* x = (const T*)p.x + f * p.x_frame;
    Raw<T, V> raw[VECS];
#pragma unroll
    for (int u = 0; u < VECS; ++u)
        if (u < count) raw[u].load(x + (long)(row + u * rows) * p.x_pixel + c);
    float scale[V], shift[V];
    if (count > 0) {
        load_affine<V>(p.gamma, c, 1.f, scale);
        load_affine<V>(p.beta, c, 0.f, shift);
    }
    // deviations from the first value: no digits are lost to a large mean
    const float ref = to_f32(x[g * each]);
    float v[VECS][V];
    float sum[1] = {0.f};
#pragma unroll
    for (int u = 0; u < VECS; ++u)
        if (u < count) {
            raw[u].get(v[u]);
#pragma unroll
            for (int i = 0; i < V; ++i) sum[0] += v[u][i] - ref;
        }
    const float per_value = 1.f / ((float)p.pixels * (float)each);
    block_sum<THREADS>(sum, lds);
    const float near = fmaf(sum[0], per_value, ref);
    float dev[2] = {0.f, 0.f};   // deviations' squares, deviations
#pragma unroll
    for (int u = 0; u < VECS; ++u)
        if (u < count)
#pragma unroll
            for (int i = 0; i < V; ++i) {
                const float d = v[u][i] - near;
                dev[0] = fmaf(d, d, dev[0]);
                dev[1] += d;
            }
    block_sum<THREADS>(dev, lds + 1);
    const float off = dev[1] * per_value, mean = near + off;
    const float rstd = 1.f / sqrtf(fmaf(-off, off, dev[0] * per_value) + p.eps);
    if (count == 0) return;
#pragma unroll
    for (int i = 0; i < V; ++i) scale[i] *= rstd;
    with_activation(p.act, [&](auto act) {
#pragma unroll
        for (int u = 0; u < VECS; ++u)
            if (u < count) {
#pragma unroll
                for (int i = 0; i < V; ++i)
                    v[u][i] = activate<YK == 0>(fmaf(v[u][i] - mean, scale[i], shift[i]),
                                                decltype(act)::value);
                store_v<V, YK>(p.y, f * p.y_frame + (long)(row + u * rows) * p.y_pixel + c, v[u]);
            }
    });
}

// Rows of a view, every one of them, start on four bytes.
bool fits(const void* base, int kind, long frame, long pixel) {
    return (uintptr_t)base % 4 == 0 && (!kind || (frame % 2 == 0 && pixel % 2 == 0));
}

// Channels can be taken v at a time.
bool fits(const GroupNormArgs& p, int width, int v) {
    return width % v == 0 && fits(p.x, p.x_kind, p.x_frame, p.x_pixel) &&
           fits(p.y, p.y_kind, p.y_frame, p.y_pixel);
}

// Whether a workgroup of so many threads can hold a frame's group of `each` channels in
// vectors of v.
bool small_holds(int pixels, int each, int v, int threads) {
    const int vectors = each / v;   // of a pixel
    return vectors <= threads && pixels <= threads / vectors * small_vectors(v);
}

// How a frame's pixels are cut for the statistics: about one workgroup for each compute
// unit, and 64 to 256 parts, which every workgroup of the second kernel joins.
int chunk_pixels(int frames, int pixels, int channels) {
    const long want = std::min(256, std::max(64, 256 / frames));   // chunks of a frame
    const long least = std::max<long>(1, 8192 / channels);         // pixels of a chunk
    return (int)std::min<long>(pixels, std::max(least, (pixels + want - 1) / want));
}

long chunks_of(int pixels, int chunk) { return ((long)pixels + chunk - 1) / chunk; }

template <int XK, int YK, int V>
hipError_t run(const GroupNormArgs& p, float2* parts, hipStream_t stream) {
    const int each = p.channels / p.groups;
    const Split sp(p.channels, p.groups, V);
    const int part = chunk_pixels(p.frames, p.pixels, p.channels);
    const int chunks = (int)chunks_of(p.pixels, part);
    // the second kernel's workgroups have 512 KB of x each where that makes 256 to 2048
    // of them: a workgroup costs microseconds before its first result, and few have too
    // little in flight.  14400 x 512 in bf16 (14.7 MB): 17 us with 256, 25 with 1024;
    // 230400 x 256 (118 MB): 66 with 256, 76 with 2048; four frames of 921600 x 128
    // (944 MB): 547 with 256, 528 with 2048.
    const long bytes = (long)p.frames * p.pixels * p.channels * (XK ? 2 : 4);
    const long blocks = std::min(2048L, std::max(256L, bytes >> 19));
    const long least = std::max<long>(1, 8192 / p.channels);
    const int chunk =
        (int)std::min<long>(p.pixels, std::max(least, ((long)p.pixels * p.frames + blocks - 1) / blocks));
    const dim3 grid((unsigned)chunks, (unsigned)p.frames);
    if (each % V == 0)
        group_norm_stats_kernel<XK, V, V><<<grid, kThreads, 0, stream>>>(p, sp, part, parts);
    else if (V == 8 && each % 4 == 0)
        group_norm_stats_kernel<XK, V, V == 8 ? 4 : 1><<<grid, kThreads, 0, stream>>>(p, sp, part, parts);
    else
        group_norm_stats_kernel<XK, V, 1><<<grid, kThreads, 0, stream>>>(p, sp, part, parts);
    const dim3 grid2((unsigned)chunks_of(p.pixels, chunk), (unsigned)p.frames);
    group_norm_apply_kernel<XK, YK, V>
        <<<grid2, kThreads, 0, stream>>>(p, sp, part, chunks, chunk, parts);
    return hipGetLastError();
}

template <int XK, int YK, int V>
hipError_t run_small(const GroupNormArgs& p, hipStream_t stream) {
    const dim3 grid((unsigned)p.groups, (unsigned)p.frames);
    if (small_holds(p.pixels, p.channels / p.groups, V, 256))
        group_norm_small_kernel<XK, YK, V, 256><<<grid, 256, 0, stream>>>(p);
    else
        group_norm_small_kernel<XK, YK, V, kSmallMost><<<grid, kSmallMost, 0, stream>>>(p);
    return hipGetLastError();
}

template <int XK, int YK>
hipError_t pick(const GroupNormArgs& p, float2* parts, hipStream_t stream) {
    const int each = p.channels / p.groups;
    for (int v : {8, 4, 2, 1}) {
        if (v > 1 && !fits(p, each, v)) continue;
        if (!small_holds(p.pixels, each, v, kSmallMost)) break;
        return v == 8   ? run_small<XK, YK, 8>(p, stream)
               : v == 4 ? run_small<XK, YK, 4>(p, stream)
               : v == 2 ? run_small<XK, YK, 2>(p, stream)
                        : run_small<XK, YK, 1>(p, stream);
    }
    if (fits(p, p.channels, 8)) return run<XK, YK, 8>(p, parts, stream);
    if (fits(p, p.channels, 4)) return run<XK, YK, 4>(p, parts, stream);
    if (fits(p, p.channels, 2)) return run<XK, YK, 2>(p, parts, stream);
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
    // groups in registers, by single elements if need be
    if (small_holds(pixels, channels / groups, 1, kSmallMost)) return 0;
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
