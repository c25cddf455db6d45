// Device side of the linear and grouped linear kernels: row tiles of ragged groups,
// the MFMA step, fp32 rows as bf16 terms, and the epilogue.
#pragma once

#include <type_traits>

#include "activations.h"
#include "matmul_kernels.h"
#include "s2_device.h"

namespace s2 {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// T: 1 bf16, 2 fp16
template <int T>
__device__ __forceinline__ f32x4 mfma(uint4 a, uint4 b, f32x4 c) {
    if constexpr (T == 1)
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(a), as_bf16x8(b), c, 0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                      __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// Rows [row0, end) of group `group` that tile t of tm rows starts at; end == row0
// when there is no such tile.
struct RowTile {
    int row0, end, group;
};

// Group g's rows, kept to [0, m] whatever the offsets hold, and its tiles of tm rows.
__device__ __forceinline__ int group_tiles(const MatmulArgs& a, int g, int tm, int& start, int& end) {
    start = end = 0;
    if (g < a.groups) {
        start = max(a.offsets[g], 0);
        end = min(a.offsets[g + 1], a.m);
    }
    return end > start ? (end - start + tm - 1) / tm : 0;
}

// The row tiles of a call: `count` of them, of at most mtiles.  Every wave counts for
// itself, 64 groups at a time, and keeps the count of up to 64 groups.
struct RowTiles {
    const MatmulArgs& a;
    int tm, count;
    int start, end, upto;   // of group `lane`; tiles of the groups up to it

    // groups g0 .. g0 + 63; returns the tiles in them
    __device__ __forceinline__ int scan(int g0) {
        const int lane = threadIdx.x & 63;
        upto = group_tiles(a, g0 + lane, tm, start, end);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int other = __shfl_up(upto, o);
            if (lane >= o) upto += other;
        }
        return __builtin_amdgcn_readfirstlane(__shfl(upto, 63));
    }

    __device__ __forceinline__ RowTiles(const MatmulArgs& args, int rows, int mtiles) : a(args), tm(rows) {
        count = mtiles;
        if (!a.offsets) return;
        // (descending offsets can make more than the grid has)
        count = 0;
        for (int g0 = 0; g0 < a.groups; g0 += 64) count = min(count + scan(g0), mtiles);
    }

    __device__ __forceinline__ RowTile at(int t) {
        if (!a.offsets) return RowTile{t * tm, a.m, 0};
        for (int g0 = 0; g0 < a.groups; g0 += 64) {
            const int sum = a.groups > 64 ? scan(g0) : count;
            const uint64_t past = __ballot(upto > t);
            if (past) {
                const int l = __ffsll((unsigned long long)past) - 1;
                const int before = l ? __shfl(upto, l - 1) : 0;   // (l is the wave's)
                return RowTile{__builtin_amdgcn_readfirstlane(__shfl(start, l) + (t - before) * tm),
                               __builtin_amdgcn_readfirstlane(__shfl(end, l)),
                               __builtin_amdgcn_readfirstlane(g0 + l)};
            }
            t -= sum;
        }
        return RowTile{0, 0, 0};
    }
};

__device__ __forceinline__ float load1(const void* p, long idx, int kind) {
    if (kind == 1) return bf16_to_f32(((const uint16_t*)p)[idx]);
    if (kind == 2) return (float)((const _Float16*)p)[idx];
    return ((const float*)p)[idx];
}

__device__ __forceinline__ void store1(void* p, long idx, float v, int kind) {
    if (kind == 1)
        ((uint16_t*)p)[idx] = f32_to_bf16(v);
    else if (kind == 2)
        ((_Float16*)p)[idx] = f32_to_f16(v);
    else
        ((float*)p)[idx] = v;
}

typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
typedef unsigned int u32x4 __attribute__((ext_vector_type(4)));

// Vectors at any element: loads and stores need no more alignment than that.
typedef u32x2 u32x2_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at2 __attribute__((aligned(2)));
typedef u32x4 u32x4_at4 __attribute__((aligned(4)));
typedef f32x4 f32x4_at4 __attribute__((aligned(4)));

// Four values at any element.
template <int YK>
__device__ __forceinline__ void store4_any(void* p, long idx, f32x4 v) {
    if constexpr (YK == 0)
        *reinterpret_cast<f32x4_at4*>((float*)p + idx) = v;
    else if constexpr (YK == 1)
        *reinterpret_cast<u32x2_at2*>((uint16_t*)p + idx) =
            u32x2{pack2_bf16_rne(v[0], v[1]), pack2_bf16_rne(v[2], v[3])};
    else
        *reinterpret_cast<u32x2_at2*>((uint16_t*)p + idx) =
            u32x2{pack2_f16_rne(v[0], v[1]), pack2_f16_rne(v[2], v[3])};
}

constexpr int kRawBufferFormat = 0x00020000;   // word 3 of an untyped buffer descriptor
constexpr uint32_t kOutside = 0x80000000u;     // an offset past every descriptor's end

// Epilogue of a wave's tile of 16 NI rows and 64 columns: accumulator [i][j][r] is row
// 16 i + 4 g + r from row_w on, column col + j.  y and the residual go through buffer
// descriptors that end with the block tile's rows, so the range check drops what lies
// outside, without a branch.  The residual of up to D row tiles is in flight.  Rows that
// four columns do not divide, or that begin anywhere: a lane whose four columns are in
// the row stores them by one unaligned store, the last ones one at a time (8000 x 2560 by
// 2001 x 2560 in bf16 66 us, 74 with single ones; 64 with 2000 columns).
//
// With 64-bit addresses, a branch a row and the residual of one row tile at a time this
// took 8.7 of 19.5 us of 14400 x 512 by 512 x 512 with a residual.
template <int YK, int NI>
struct TileEnd {
    static constexpr int ES = YK ? 2 : 4;
    static constexpr int D = NI < 4 ? NI : YK == 0 && NI == 8 ? 2 : 4;   // by registers
    typedef typename std::conditional<YK == 0, u32x4, u32x2>::type Piece;   // four columns

    char* y;
    const char* res;
    int y_bytes, res_bytes;
    uint32_t y_at, res_at, y_row, res_row;   // of the lane's first piece; bytes between rows
    uint32_t drop[4];                        // of column col + j
    bool whole;   // aligned pieces of four in every row
    bool four;    // else: this lane's four columns are all in the row
    f32x4 bias;
    Piece held[D][4];

    __device__ __forceinline__ TileEnd(const MatmulArgs& a, const RowTile& rt, int rows, int row_w,
                                       int col, bool whole_pieces) {
        const int g = (threadIdx.x & 63) >> 4;
        whole = whole_pieces;
        y = (char*)a.y + (long)rt.row0 * a.y_stride * ES;
        y_bytes = (int)(((long)(rows - 1) * a.y_stride + a.n) * ES);
        y_row = (uint32_t)(a.y_stride * ES);
        y_at = (row_w + 4 * g) * y_row + col * ES;
        res = a.res ? (const char*)a.res + (long)rt.row0 * a.res_stride * ES : nullptr;
        res_bytes = (int)(((long)(rows - 1) * a.res_stride + a.n) * ES);
        res_row = (uint32_t)(a.res_stride * ES);
        res_at = (row_w + 4 * g) * res_row + col * ES;
#pragma unroll
        for (int j = 0; j < 4; ++j) drop[j] = col + j < a.n ? 0u : kOutside;
        four = col + 3 < a.n;
        bias = f32x4{0.f, 0.f, 0.f, 0.f};
        if (a.bias) {
            const __amdgpu_buffer_rsrc_t rb = __builtin_amdgcn_make_buffer_rsrc(
                (void*)(a.bias + (long)rt.group * a.n), (short)0, a.n * 4, kRawBufferFormat);
#pragma unroll
            for (int j = 0; j < 4; ++j)
                bias[j] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(rb, (col + j) * 4, 0, 0));
        }
        if (res && whole)
#pragma unroll
            for (int i = 0; i < D; ++i) load<true>(i);
    }

    // the residual of row tile i
    template <bool WHOLE>
    __device__ __forceinline__ void load(int i) {
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc((void*)res, (short)0, res_bytes, kRawBufferFormat);
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const uint32_t at = res_at + (16 * i + r) * res_row;
            Piece& q = held[i % D][r];
            if constexpr (WHOLE) {
                if constexpr (YK == 0)
                    q = __builtin_amdgcn_raw_buffer_load_b128(rs, at | drop[0], 0, 0);
                else
                    q = __builtin_amdgcn_raw_buffer_load_b64(rs, at | drop[0], 0, 0);
            } else if (four) {
                if constexpr (YK == 0) {   // 16 bytes through a descriptor at any fourth
                    q = __builtin_amdgcn_raw_buffer_load_b128(rs, at, 0, 0);
                } else {
                    q = Piece{};
                    if (at < (uint32_t)res_bytes) q = *reinterpret_cast<const u32x2_at2*>(res + at);
                }
            } else {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const uint32_t o = (at + j * ES) | drop[j];
                    if constexpr (YK == 0) {
                        q[j] = __builtin_amdgcn_raw_buffer_load_b32(rs, o, 0, 0);
                    } else {
                        const uint32_t h = (uint16_t)__builtin_amdgcn_raw_buffer_load_b16(rs, o, 0, 0);
                        q[j >> 1] = j & 1 ? q[j >> 1] | (h << 16) : h;
                    }
                }
            }
        }
    }

    template <int ACT, bool WHOLE>
    __device__ __forceinline__ void emit(const f32x4 (&acc)[NI][4]) {
        const __amdgpu_buffer_rsrc_t rs =
            __builtin_amdgcn_make_buffer_rsrc((void*)y, (short)0, y_bytes, kRawBufferFormat);
        if (!WHOLE && res)
#pragma unroll
            for (int i = 0; i < D; ++i) load<false>(i);
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            float v[4][4];
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int j = 0; j < 4; ++j) v[r][j] = activate<YK == 0>(acc[i][j][r] + bias[j], ACT);
            if (res) {
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        if constexpr (YK == 0) {
                            v[r][j] += __uint_as_float(held[i % D][r][j]);
                        } else {
                            const uint16_t h = (uint16_t)(held[i % D][r][j >> 1] >> (16 * (j & 1)));
                            v[r][j] += YK == 1 ? bf16_to_f32(h) : (float)__builtin_bit_cast(_Float16, h);
                        }
                    }
                if (i + D < NI) load<WHOLE>(i + D);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const uint32_t at = y_at + (16 * i + r) * y_row;
                Piece q;
                if constexpr (YK == 0) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) q[j] = __float_as_uint(v[r][j]);
                } else {
#pragma unroll
                    for (int j = 0; j < 2; ++j)
                        q[j] = YK == 1 ? pack2_bf16_rne(v[r][2 * j], v[r][2 * j + 1])
                                       : pack2_f16_rne(v[r][2 * j], v[r][2 * j + 1]);
                }
                if constexpr (!WHOLE) {
                    if (four) {
                        if constexpr (YK == 0)
                            __builtin_amdgcn_raw_buffer_store_b128(q, rs, at, 0, 0);
                        else if (at < (uint32_t)y_bytes)
                            *reinterpret_cast<u32x2_at2*>(y + at) = q;
                    } else
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const uint32_t o = (at + j * ES) | drop[j];
                        if constexpr (YK == 0)
                            __builtin_amdgcn_raw_buffer_store_b32(q[j], rs, o, 0, 0);
                        else
                            __builtin_amdgcn_raw_buffer_store_b16((uint16_t)(q[j >> 1] >> (16 * (j & 1))),
                                                                  rs, o, 0, 0);
                    }
                } else if constexpr (YK == 0) {
                    __builtin_amdgcn_raw_buffer_store_b128(q, rs, at | drop[0], 0, 0);
                } else {
                    __builtin_amdgcn_raw_buffer_store_b64(q, rs, at | drop[0], 0, 0);
                }
            }
        }
    }

    __device__ __forceinline__ void finish(const MatmulArgs& a, const f32x4 (&acc)[NI][4]) {
        with_activation(a.act, [&](auto act) {
            if (whole)
                emit<decltype(act)::value, true>(acc);
            else
                emit<decltype(act)::value, false>(acc);
        });
    }
};

// fp32 as a sum of three bf16 values, exactly, whatever y's type: with two (off by 2^-17)
// a product whose leading bits cancel would be off by more than y's rounding.  The first
// two take the top 8 bits of what the ones before leave, by truncation, which cannot
// overflow and leaves an exact rest; the last holds the rest.  An infinity stays in the
// first term, a NaN reaches the later ones.  v: pairs of values, h[q]: their terms q
// packed.
constexpr int kTerms = 3;

__device__ __forceinline__ void split2(float v0, float v1, uint32_t (&h)[kTerms]) {
#pragma unroll
    for (int q = 0; q + 1 < kTerms; ++q) {
        const uint32_t b0 = __float_as_uint(v0) & 0xffff0000u, b1 = __float_as_uint(v1) & 0xffff0000u;
        h[q] = (b0 >> 16) | b1;
        v0 = fabsf(v0) == __builtin_inff() ? 0.f : v0 - __uint_as_float(b0);
        v1 = fabsf(v1) == __builtin_inff() ? 0.f : v1 - __uint_as_float(b1);
    }
    h[kTerms - 1] = pack2_bf16_rne(v0, v1);
}

__device__ __forceinline__ void split8(const float (&v)[8], uint4 (&out)[kTerms]) {
    uint32_t w[4][kTerms];
#pragma unroll
    for (int e = 0; e < 4; ++e) split2(v[2 * e], v[2 * e + 1], w[e]);
#pragma unroll
    for (int q = 0; q < kTerms; ++q) out[q] = make_uint4(w[0][q], w[1][q], w[2][q], w[3][q]);
}

// Eight consecutive k of a row as an MFMA operand piece, zeros from `left` of them on.
// FULL: all eight are there.  ODD: rows may begin in the middle of four bytes, where a
// 16-byte load takes several times as long (1 x 5001 by 5000 x 5001: 31 us): the four or
// five words that hold the eight are loaded and shifted.
template <bool FULL, bool ODD = false>
__device__ __forceinline__ uint4 piece16(const uint16_t* p, int left) {
    if constexpr (ODD) {
        if (FULL || left >= 8) {
            const uint32_t odd = (uintptr_t)p >> 1 & 1;
            const u32_any* a = (const u32_any*)(p - odd);
            const u32x4 q = *reinterpret_cast<const u32x4_at4*>(a);
            const uint32_t top = a[3 + odd], s = 16 * odd;
            return make_uint4(__builtin_amdgcn_alignbit(q[1], q[0], s), __builtin_amdgcn_alignbit(q[2], q[1], s),
                              __builtin_amdgcn_alignbit(q[3], q[2], s), __builtin_amdgcn_alignbit(top, q[3], s));
        }
    } else if (FULL || left >= 8) {
        const u32x4 q = *reinterpret_cast<const u32x4_at2*>(p);
        return make_uint4(q[0], q[1], q[2], q[3]);
    }
    alignas(16) uint16_t h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = left > e ? p[e] : (uint16_t)0;
    return pack8_bf16(h);
}

template <bool FULL>
__device__ __forceinline__ void piece32(const float* p, int left, float (&v)[8]) {
    if (FULL || left >= 8) {
#pragma unroll
        for (int e = 0; e < 8; e += 4) {
            const f32x4 q = *reinterpret_cast<const f32x4_at4*>(p + e);
#pragma unroll
            for (int i = 0; i < 4; ++i) v[e + i] = q[i];
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = left > e ? p[e] : 0.f;
    }
}

}  // namespace s2
