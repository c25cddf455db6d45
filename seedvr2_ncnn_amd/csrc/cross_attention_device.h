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

// Sample b, of samples one after the other.
__device__ __forceinline__ CrossSample ragged_sample(const CrossArgs& a, int b) {
    const int q0 = clamped(a.q_offsets[b], a.lq), q1 = clamped(a.q_offsets[b + 1], a.lq);
    const int k0 = clamped(a.k_offsets[b], a.lk), k1 = clamped(a.k_offsets[b + 1], a.lk);
    return CrossSample{q0, k0, b, max(q1 - q0, 0), max(k1 - k0, 0)};
}

// Tile `tile` of `rows` rows of kv head `head`; the sample's tiles that there are.
struct CrossTile {
    CrossSample s;
    int head, row0, rows;   // of the sample's nq G rows
    int part;
};

// The workgroup's tile, or rows 0.  Ordered by part, tile, head: workgroups of one head's
// tiles follow each other on an XCD, whose L2 then holds the head's keys.  tiles: at most
// there are.
//
// Up to kScanSamples samples of any lengths, an offset a lane, are dealt out over the tiles that
// they make.  Of more each has places of its own: a sample's begin at that of its first row
// were all rows one sample's, plus its number, which leaves room for last tiles that are not
// full.  A workgroup searches for its place's sample, a 64th of those left at a time (32768
// samples of a row, eight heads of 128, 1.7 ms; 111 with a scan of all by each).
__device__ __forceinline__ CrossTile cross_tile(const CrossArgs& a, int each, int tiles, int parts) {
    const int group = a.heads / a.kv_heads;
    const int lane = threadIdx.x & 63;
    CrossTile t;
    t.rows = 0;
    int count = tiles;
    CrossSample s = {0, 0, 0, 0, 0};   // the lane's
    int upto = 0;                      // tiles of the samples up to it
    const bool scan = a.q_offsets && a.batch <= kScanSamples;
    if (scan) {
        if (lane < a.batch) s = ragged_sample(a, lane);
        upto = (int)(((long)s.nq * group + each - 1) / each);
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int other = __shfl_up(upto, o);
            if (lane >= o) upto += other;
        }
        count = min(__builtin_amdgcn_readlane(upto, 63), tiles);   // (descending offsets can make more)
    }
    const long blocks = (long)count * a.kv_heads * parts - a.first;
    if (blockIdx.x >= blocks) return t;
    const int lid = a.first + xcd_remap(blockIdx.x, (int)min(blocks, kLaunchBlocks));
    t.part = lid % parts;
    const int i = lid / parts % count;
    t.head = lid / parts / count;
    int before = 0;   // the sample's first tile
    if (!a.q_offsets) {
        const int of_sample = (int)(((long)a.lq * group + each - 1) / each);
        const int b = i / of_sample;
        t.s = CrossSample{0, 0, b, a.lq, a.key_lengths ? clamped(a.key_lengths[b], a.lk) : a.lk};
        before = b * of_sample;
    } else if (scan) {
        const uint64_t past = __ballot(upto > i);
        if (!past) return t;
        const int l = __builtin_amdgcn_readfirstlane(__ffsll((unsigned long long)past) - 1);
        auto of_lane = [&](int v) { return __builtin_amdgcn_readlane(v, l); };
        before = l ? __builtin_amdgcn_readlane(upto, max(l - 1, 0)) : 0;
        t.s = CrossSample{of_lane((int)s.q0), of_lane((int)s.k0), l, of_lane(s.nq), of_lane(s.nk)};
    } else {
        auto place = [&](int b) { return (int)((unsigned)(clamped(a.q_offsets[b], a.lq) * group) / (unsigned)each) + b; };
        int b = 0;   // the first of n samples, one of which has place i
        for (int n = a.batch; n > 1;) {
            const int step = (n + 63) / 64;
            const int l = __popcll(__ballot(lane * step < n && place(b + min(lane * step, n - 1)) <= i)) - 1;
            if (l < 0) return t;   // rows ahead of the first sample
            b += l * step;
            n = min(step, n - l * step);
        }
        b = __builtin_amdgcn_readfirstlane(b);
        const CrossSample found = ragged_sample(a, b);
        auto uniform = [](long v) { return __builtin_amdgcn_readfirstlane((int)v); };
        before = uniform(place(b));
        t.s = CrossSample{uniform(found.q0), uniform(found.k0), b, uniform(found.nq), uniform(found.nk)};
    }
    const long row0 = ((long)i - before) * each;
    if (row0 < 0) return t;   // (of descending offsets)
    t.row0 = (int)row0;
    t.rows = (int)max(min((long)each, (long)t.s.nq * group - row0), 0L);   // (none of a place without a tile)
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
constexpr float kLazy = 8.f;   // powers of two by which weights may pass 1 before m follows

// A weight is 2^((s - m) c), s a score and m a maximum of scores, c = |scale| log2 e (a negative
// scale turns q's signs).  The difference comes first: s c and m c, rounded or one of them
// rounded, would differ by more than weights reach where they pass 2^24.  c is within what a
// difference of nought or -inf can be multiplied by, and 2^-149 leaves the weights of a scale
// of nought 1 to 2^-21.
__device__ __forceinline__ float weight_scale(const CrossArgs& a) {
    return fminf(fmaxf(fabsf(a.scale) * 1.4426950408889634f, 0x1p-149f), 3.4028234663852886e38f);
}

// Of the wave's four groups of 16 lanes.
__device__ __forceinline__ float max_groups(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float sum_groups(float x) {
    auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// Keys of the workgroup's sample up to the last one that the mask keeps: padded prompts end
// there, and so do the ranges of keys.  A wave reads a kilobyte at a time from the end.
__device__ __forceinline__ int keys_kept(const CrossArgs& a, const CrossTile& t) {
    typedef uint32_t words __attribute__((ext_vector_type(4), aligned(1)));
    const uint8_t* mask = a.key_mask + t.s.b * a.mask_batch + t.s.k0;
    const int lane = threadIdx.x & 63;
    for (int end = t.s.nk; end > 0; end -= 1024) {
        const int at = end - 16 * (lane + 1);   // the lane's 16 bytes, or what is left of them
        int last = -1;
        if (at >= 0) {
            const words v = *reinterpret_cast<const words*>(mask + at);
#pragma unroll
            for (int w = 0; w < 4; ++w)
                if (v[w]) last = at + 4 * w + (31 - __builtin_clz(v[w])) / 8;
        } else {
            for (int i = 0; i < at + 16; ++i)
                if (mask[i]) last = i;
        }
        const uint64_t some = __ballot(last >= 0);
        if (some) return __builtin_amdgcn_readlane(last, __ffsll((unsigned long long)some) - 1) + 1;
    }
    return 0;
}

constexpr int kMaskWords = 128;                // of 64 keys: a block of mask bits
constexpr int kMaskBits = 2 * kMaskWords;      // two blocks in LDS

// The tiles of k and v of a workgroup of four waves: DMA into STAGES stages of LDS, a tile of
// k and then one of v of kTileKeys rows of DP elements of ES bytes each.  Chunk c (16 bytes)
// of row r stands at c ^ Swizzle::key(r) or value(r).  Keys that do not count, by the
// sample's length or the mask, and columns from d on are zeros, whatever is there.
template <int ES, int DP, int STAGES, bool MASK, typename Swizzle>
struct KeyTiles {
    static constexpr int RB = DP * ES, KB = kTileKeys * RB, SB = 2 * KB;   // bytes: a row, a tile, a stage
    static constexpr int CH = RB / 16;      // chunks of a row
    static constexpr int KI = KB / 4096;    // DMA instructions of a wave and operand
    int nk, wave;
    uint32_t base;
    uint64_t* bits;
    const uint8_t* mask;
    long kr, vr;                            // bytes between rows
    const char* next_k;                     // of the tile that is loaded next
    const char* next_v;
    uint32_t ko[KI], vo[KI];
    uint32_t ahead = 0;                     // the mask's bits of the tile after the one last loaded

    __device__ __forceinline__ KeyTiles(const CrossArgs& a, const CrossTile& t, int keys, int kb, uint32_t lds,
                                        uint64_t* mask_bits)
        : nk(keys), wave(__builtin_amdgcn_readfirstlane(threadIdx.x >> 6)), base(lds), bits(mask_bits),
          mask(a.key_mask + t.s.b * a.mask_batch + t.s.k0), kr(a.ks.row * ES), vr(a.vs.row * ES) {
        const long at = (long)kb * kTileKeys;
        next_k = (const char*)a.k + (t.s.b * a.ks.batch + (t.s.k0 + at) * a.ks.row + t.head * a.ks.head) * ES;
        next_v = (const char*)a.v + (t.s.b * a.vs.batch + (t.s.k0 + at) * a.vs.row + t.head * a.vs.head) * ES;
#pragma unroll
        for (int j = 0; j < KI; ++j) {
            const int i = (wave * KI + j) * 64 + (threadIdx.x & 63);
            const int r = i / CH, c = i % CH;
            const int ck = c ^ Swizzle::key(r), cv = c ^ Swizzle::value(r);
            ko[j] = ck * (16 / ES) < a.d ? (uint32_t)(r * kr) + ck * 16 : kOutside;
            vo[j] = cv * (16 / ES) < a.d ? (uint32_t)(r * vr) + cv * 16 : kOutside;
        }
    }

    __device__ __forceinline__ uint32_t mask_bits(int kt) const {
        return ((const uint32_t*)&bits[kt / 2 % kMaskBits])[kt & 1];
    }

    // keys of tile kt that count, of a mask's `kept`
    __device__ __forceinline__ uint32_t valid(int kt, uint32_t kept) const {
        const int left = nk - kt * kTileKeys;
        const uint32_t v = left >= kTileKeys ? ~0u : (1u << left) - 1;
        return MASK ? v & (uint32_t)__builtin_amdgcn_readfirstlane(kept) : v;
    }
    __device__ __forceinline__ uint32_t valid(int kt) const { return valid(kt, MASK ? mask_bits(kt) : 0u); }

    // the next block of the mask as bits, when the first tile of it is loaded
    __device__ __forceinline__ void read_mask(int kt, bool first) {
        if constexpr (MASK) {
            if (!first && kt % (2 * kMaskWords) != 0) return;
            const int block = kt / 2 / kMaskWords * kMaskWords;
            for (int w = block + wave; w < block + kMaskWords; w += 4) {
                const int key = w * 64 + (threadIdx.x & 63);
                const uint64_t m = __ballot(key < nk && mask[min(key, nk - 1)] != 0);
                if ((threadIdx.x & 63) == 0) bits[w % kMaskBits] = m;
            }
            __syncthreads();
            ahead = mask_bits(kt);
        }
    }

    // Loads tile kt, the next one; all waves.  Returns its keys that count.
    __device__ __forceinline__ uint32_t issue(int kt, int stage, bool first) {
        read_mask(kt, first);
        const uint32_t st = base + stage * SB;
        const i32x4 rk = wave_uniform(buffer_rsrc(next_k, (uint32_t)((kTileKeys - 1) * kr + RB)));
        const i32x4 rv = wave_uniform(buffer_rsrc(next_v, (uint32_t)((kTileKeys - 1) * vr + RB)));
        next_k += kTileKeys * kr;
        next_v += kTileKeys * vr;
        const uint32_t keys = valid(kt, ahead);
        if constexpr (MASK) ahead = mask_bits(kt + 1);   // (of another block: read again with it)
        if (keys == ~0u) {
#pragma unroll
            for (int j = 0; j < KI; ++j)
                lds_dma16(rk, __builtin_amdgcn_readfirstlane(st + (wave * KI + j) * 1024), ko[j], 0);
#pragma unroll
            for (int j = 0; j < KI; ++j)
                lds_dma16(rv, __builtin_amdgcn_readfirstlane(st + KB + (wave * KI + j) * 1024), vo[j], 0);
        } else {
#pragma unroll
            for (int j = 0; j < KI; ++j) {
                const int r = ((wave * KI + j) * 64 + (threadIdx.x & 63)) / CH;
                const uint32_t out = keys >> r & 1 ? 0u : kOutside;
                lds_dma16(rk, __builtin_amdgcn_readfirstlane(st + (wave * KI + j) * 1024), ko[j] | out, 0);
                lds_dma16(rv, __builtin_amdgcn_readfirstlane(st + KB + (wave * KI + j) * 1024), vo[j] | out, 0);
            }
        }
        return keys;
    }

    // Until tile kt is there for all waves; those after it, STAGES - 2 of them at most, may be in
    // flight.
    __device__ __forceinline__ void await(int kt, int ke) const {
        if (kt + STAGES - 1 <= ke)
            asm volatile("s_waitcnt vmcnt(%0)" ::"n"((STAGES - 2) * 2 * KI) : "memory");
        else
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
        asm volatile("s_barrier" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
    }
};

}  // namespace s2
