// Linear of many fp32 rows with a short k: the weight stays in LDS.
//
// On block tiles a workgroup's first loads and its epilogue are as long as a few k
// steps, and fp32 rows are packed before.  Here a workgroup keeps the weight rows of
// 256 columns in LDS for its whole life, and each of its waves takes 16 rows at a time
// on its own: their k straight from memory into registers, split there into bf16 terms
// once for the 256 columns, then 64 columns after 64.  No wave waits for another once
// the weight is there, so that one stores or loads while another multiplies.
//
// 21600 x 132 by 2560 x 132, bf16 results: 58 us.  The 110 MB of y take 21, the matrix
// instructions (three terms, k as 160) 23 at their peak rate; the vector (terms, epilogue)
// and LDS pipes are busy for 15 to 20 each.  With two terms, which hold 16 bits of x, the
// kernel took 47; then 32 rows a wave, which halve the LDS reads but leave registers for
// eight waves only, took 9% longer.
#include "matmul_device.h"

namespace s2 {

namespace {

constexpr int kCols = 256, kRows = 16;

// Waves of a workgroup, by registers.
constexpr int waves_of(int steps) { return steps == 3 ? 16 : 12; }

// Four of a row's k, zeros from `left` of them on.
__device__ __forceinline__ u32x2 four16(const uint16_t* p, int left) {
    if (left >= 4) return *reinterpret_cast<const u32x2_at2*>(p);
    uint32_t h[3];
#pragma unroll
    for (int e = 0; e < 3; ++e) h[e] = left > e ? p[e] : 0;
    return u32x2{h[0] | h[1] << 16, h[2]};
}

// STEPS: k steps of 32, zeros past k.
template <int YK, int STEPS>
__global__ __launch_bounds__(64 * waves_of(STEPS)) void matmul_short_kernel(MatmulArgs a, int blocks_n,
                                                                            int splits, bool whole) {
    // an odd number of 16-byte pieces a row: 16 rows' reads spread over all banks
    constexpr int P = STEPS * 32 + 8, PIECES = STEPS * 4;
    constexpr int kWaves = waves_of(STEPS), kThreads = 64 * kWaves;
    __shared__ __attribute__((aligned(16))) uint16_t w_lds[kCols * P];
    __shared__ __attribute__((aligned(16))) float bias[kCols];
    const int tid = threadIdx.x;
    const int lane = tid & 63, l16 = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    // the column blocks of the same rows are neighbours on an XCD, which share its L2
    const int lid = xcd_remap(blockIdx.x, gridDim.x);
    const int col0 = lid % blocks_n * kCols;
    const int cols = min(a.n - col0, kCols);
    const int tiles = (a.m + kRows - 1) / kRows;
    const int split = lid / blocks_n;
    const int t0 = (int)((long)tiles * split / splits) + wave;
    const int t1 = (int)((long)tiles * (split + 1) / splits);

    // through descriptors that end with the rows: what lies past them or past k is zero
    float f[STEPS][8];
    const uint32_t x_row = (uint32_t)(a.x_stride * 4);
    auto load = [&](int t) {
        const int rows = (int)min((long)a.m - (long)t * kRows, (long)kRows);
        const __amdgpu_buffer_rsrc_t xs = __builtin_amdgcn_make_buffer_rsrc(
            (void*)((const float*)a.x + (long)t * kRows * a.x_stride), (short)0,
            rows > 0 ? (int)((rows - 1) * x_row + a.k * 4) : 0, kRawBufferFormat);
        int g4 = 4 * g;   // not known, else 20 offsets are kept, and spilled
        asm volatile("" : "+v"(g4));
#pragma unroll
        for (int s = 0; s < STEPS; ++s)
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const int k = 32 * s + g4 + 4 * e;
                const uint32_t past = k < a.k ? 0u : kOutside;
                const u32x4 q =
                    __builtin_amdgcn_raw_buffer_load_b128(xs, (l16 * x_row + 4 * k) | past, 0, 0);
#pragma unroll
                for (int v = 0; v < 4; ++v) f[s][e + v] = __uint_as_float(q[v]);
            }
    };
    load(t0);
    const uint16_t* w = (const uint16_t*)a.w + (long)col0 * a.k;
    constexpr int ALL = kCols * PIECES, EACH = (ALL + kThreads - 1) / kThreads;   // pieces of a thread
    u32x2 h[EACH][2];
#pragma unroll
    for (int b = 0; b < EACH; ++b) {
        const int i = tid + kThreads * b, r = i / PIECES, u = i % PIECES;
        const int k = 32 * (u >> 2) + 4 * (u & 3), col = (r & ~63) + 4 * (r & 15) + ((r >> 4) & 3);
#pragma unroll
        for (int e = 0; e < 2; ++e)
            h[b][e] = four16(w + (long)col * a.k + k + 16 * e, col < cols && i < ALL ? a.k - k - 16 * e : 0);
    }
#pragma unroll
    for (int b = 0; b < EACH; ++b) {
        const int i = tid + kThreads * b;
        if (ALL % kThreads == 0 || i < ALL)
            *reinterpret_cast<uint4*>(&w_lds[i / PIECES * P + i % PIECES * 8]) =
                make_uint4(h[b][0][0], h[b][0][1], h[b][1][0], h[b][1][1]);
    }
    if (tid < kCols) bias[tid] = a.bias && tid < cols ? a.bias[col0 + tid] : 0.f;
    __syncthreads();

    MatmulArgs rest = a;
    rest.bias = nullptr;   // from LDS
#pragma unroll 1
    for (int t = t0; t < t1; t += kWaves) {
        const RowTile rt{t * kRows, a.m, 0};
        const int rows = min(a.m - rt.row0, kRows);
        if (a.k % 4 != 0)   // four values may end in the next row
#pragma unroll
            for (int s = 0; s < STEPS; ++s)
#pragma unroll
                for (int e = 0; e < 8; e += 4)
#pragma unroll
                    for (int v = 1; v < 4; ++v)
                        if (32 * s + 4 * g + 4 * e + v >= a.k) f[s][e + v] = 0.f;
        uint4 fx[STEPS][kTerms];
#pragma unroll
        for (int s = 0; s < STEPS; ++s) split8(f[s], fx[s]);
        f32x4 acc[1][4];
        auto multiply = [&](int c) {
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[0][j] = f32x4{0.f, 0.f, 0.f, 0.f};
            const uint16_t* w = w_lds + (c + l16) * P + 8 * g;
            uint4 fw[2][2];
            auto read = [&](int u) {   // of k step u / 2, columns 2 (u % 2) and the next
#pragma unroll
                for (int j = 0; j < 2; ++j)
                    fw[u & 1][j] = *reinterpret_cast<const uint4*>(w + 16 * (2 * (u & 1) + j) * P + 32 * (u >> 1));
            };
            read(0);
#pragma unroll
            for (int u = 0; u < 2 * STEPS; ++u) {
                if (u + 1 < 2 * STEPS) read(u + 1);
                __builtin_amdgcn_sched_barrier(0);   // else all reads come first, and spill
#pragma unroll
                for (int q = 0; q < kTerms; ++q)
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        acc[0][2 * (u & 1) + j] =
                            mfma<1>(fx[u >> 1][q], fw[u & 1][j], acc[0][2 * (u & 1) + j]);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto finish = [&](int c) {
            // not known, else all offsets of the epilogue are kept, and spilled
            int row_w = 0;
            asm volatile("" : "+s"(row_w));
            const int col = c + 4 * l16;
            TileEnd<YK, 1> end(rest, rt, rows, row_w, col0 + col, whole);
            end.bias = *reinterpret_cast<const f32x4*>(bias + col);
            end.finish(rest, acc);
        };
        int c = 0;
#pragma unroll 1
        for (; c + 64 < cols; c += 64) {
            multiply(c);
            finish(c);
        }
        multiply(c);
        load(t + kWaves);   // before the stores, which a wait would include
        finish(c);
    }
}

template <int YK, int STEPS>
hipError_t run(const MatmulArgs& a, const MatmulPlan& p, hipStream_t stream) {
    const int blocks_n = (a.n + kCols - 1) / kCols;
    matmul_short_kernel<YK, STEPS>
        <<<(unsigned)(blocks_n * p.parts), 64 * waves_of(STEPS), 0, stream>>>(a, blocks_n, p.parts,
                                                                              p.whole);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_matmul_short(const MatmulArgs& a, const MatmulPlan& plan, hipStream_t stream) {
    if (a.k <= 96)
        return a.y_kind == 0   ? run<0, 3>(a, plan, stream)
               : a.y_kind == 1 ? run<1, 3>(a, plan, stream)
                               : run<2, 3>(a, plan, stream);
    return a.y_kind == 0   ? run<0, 5>(a, plan, stream)
           : a.y_kind == 1 ? run<1, 5>(a, plan, stream)
                           : run<2, 5>(a, plan, stream);
}

}  // namespace s2
