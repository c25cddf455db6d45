// Device side of cross attention: samples, tiles of their rows, masks of key tiles, and
// what every kernel does with its results.
//
// Rows: query i and head hk G + j of a sample, G = heads / kv_heads, are row i G + j of
// kv head hk, so that a group's heads share a tile's reads of k and v.
#pragma once

#include "cross_attention_kernels.h"
#include "matmul_device.h"

namespace s2 {

// A sample's queries and keys.
struct CrossSample {
    long q0, k0;   // first rows, of the operands without batch strides
    int b, nq, nk;
};

__device__ __forceinline__ int clamped(int v, int most) { return min(max(v, 0), most); }

__device__ __forceinline__ int sample_queries(const CrossArgs& a, int b) {
    if (!a.q_offsets) return a.lq;
    const int start = clamped(a.q_offsets[b], a.lq);
    return max(clamped(a.q_offsets[b + 1], a.lq) - start, 0);
}

__device__ __forceinline__ CrossSample cross_sample(const CrossArgs& a, int b) {
    CrossSample s{0, 0, b, a.lq, a.lk};
    if (a.q_offsets) {
        s.q0 = clamped(a.q_offsets[b], a.lq);
        s.nq = sample_queries(a, b);
        s.k0 = clamped(a.k_offsets[b], a.lk);
        s.nk = max(clamped(a.k_offsets[b + 1], a.lk) - (int)s.k0, 0);
    } else if (a.key_lengths) {
        s.nk = clamped(a.key_lengths[b], a.lk);
    }
    return s;
}

// Tile `tile` of `rows` rows of kv head `head`; the sample's tiles that there are.
struct CrossTile {
    CrossSample s;
    int head, row0, rows;   // of the sample's nq G rows
    int part;
};

// The workgroup's tile, or rows 0.  Ordered by part, tile, head: workgroups of one head's
// tiles follow each other on an XCD, whose L2 then holds the head's keys.  tiles: at most
// there are.  Samples of any lengths are dealt out over the tiles that they make, found by a
// scan of 64 offsets at a time.
__device__ __forceinline__ CrossTile cross_tile(const CrossArgs& a, int each, int tiles, int parts) {
    const int group = a.heads / a.kv_heads;
    const int lane = threadIdx.x & 63;
    CrossTile t;
    t.rows = 0;
    int count = tiles;
    if (a.q_offsets) {
        count = 0;
        for (int b0 = 0; b0 < a.batch; b0 += 64) {
            int n = b0 + lane < a.batch ? sample_queries(a, b0 + lane) : 0;
            n = (int)(((long)n * group + each - 1) / each);
#pragma unroll
            for (int o = 32; o; o >>= 1) n += __shfl_xor(n, o);
            count = min(count + n, tiles);   // (descending offsets can make more)
        }
        count = __builtin_amdgcn_readfirstlane(count);
    }
    const long blocks = (long)count * a.kv_heads * parts;
    if (blockIdx.x >= blocks) return t;
    const int lid = xcd_remap(blockIdx.x, (int)blocks);
    t.part = lid % parts;
    int i = lid / parts % count;
    t.head = lid / parts / count;
    if (!a.q_offsets) {
        const int of_sample = (int)(((long)a.lq * group + each - 1) / each);
        t.s = cross_sample(a, i / of_sample);
        t.row0 = i % of_sample * each;
        t.rows = (int)min((long)each, (long)a.lq * group - t.row0);
        return t;
    }
    for (int b0 = 0; b0 < a.batch; b0 += 64) {
        const int nq = b0 + lane < a.batch ? sample_queries(a, b0 + lane) : 0;
        const int n = (int)(((long)nq * group + each - 1) / each);
        int upto = n;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int other = __shfl_up(upto, o);
            if (lane >= o) upto += other;
        }
        const uint64_t past = __ballot(upto > i);
        if (past) {
            const int l = __ffsll((unsigned long long)past) - 1;
            const int before = l ? __shfl(upto, l - 1) : 0;
            t.s = cross_sample(a, __builtin_amdgcn_readfirstlane(b0 + l));
            t.row0 = __builtin_amdgcn_readfirstlane((i - before) * each);
            t.rows = (int)min((long)each, (long)t.s.nq * group - t.row0);
            return t;
        }
        i -= __builtin_amdgcn_readfirstlane(__shfl(upto, 63));
    }
    return t;
}

// Element offsets of a row of q or out.
__device__ __forceinline__ long cross_row(const CrossArgs& a, const CrossRows& r, const CrossTile& t, int row) {
    const int group = a.heads / a.kv_heads;
    const int i = row / group;
    return t.s.b * r.batch + (t.s.q0 + i) * r.row + (long)(t.head * group + row - i * group) * r.head;
}

// Index of a row's part.
__device__ __forceinline__ long cross_part(const CrossArgs& a, const CrossParts& p, const CrossTile& t, int row) {
    const int group = a.heads / a.kv_heads;
    const int i = row / group;
    const long q = (a.q_offsets ? 0 : (long)t.s.b * a.lq) + t.s.q0 + i;
    return (q * a.heads + t.head * group + row - i * group) * p.parts + t.part;
}

__device__ __forceinline__ void store4_out(const CrossArgs& a, long at, f32x4 v) {
    if (a.out_kind == 0)
        store4_any<0>(a.out, at, v);
    else if (a.out_kind == 1)
        store4_any<1>(a.out, at, v);
    else
        store4_any<2>(a.out, at, v);
}

constexpr float kLowest = -3.4028234663852886e38f;   // the maximum of no scores

}  // namespace s2
