// Cross attention of 16-bit operands on tiles of rows.
//
// A wave has 32 rows, whose q stays in registers; k and v go through LDS by DMA in tiles of
// 32 keys that the workgroup's four waves share.  S^T = K Q^T and O^T = V^T P^T on 16x16x32
// products: a score accumulator's four registers are four neighbouring keys of one row, and
// two of them, of 16 keys each, are the second product's operand as they stand.  Its other
// operand, four keys by 16 columns of v, is what a transposing LDS read gives of v's rows.
// So weights never leave registers and v is not transposed before.  (32x32x16 products
// leave the matrix cores waiting less, but the chip clocks lower: 3 to 5% slower.)
//
// Softmax in powers of two: weights are 2^(c (s - m)), c = |scale| log2 e (a negative scale turns
// q's signs), m a maximum of scores that follows them only when a row's weight passes 2^8: the
// few rescales cost nothing, and a tile's maxima need not be exchanged between lanes to find
// that none is due.  Weights are rounded to the operands' type for the second product,
// at most half a step each, as independent errors of its terms; their sum stays in fp32.
//
// On long keys the matrix cores and the exponentials beside them bound it, at the clocks that
// their power leaves (1.7 GHz): 4096 on 21600 keys, 20 heads of 128, 0.79 to 0.85 ms by the card,
// 1.1 PFLOP/s; 21600 on 512 120 to 125 us, 0.92.  A wave's rows are 32: with 16 a tile's reads of LDS would bound
// it, 64 do not fit its registers.  Two waves' keys ahead (a second tile's scores before the
// first one's weights) were slower than three workgroups' waves in turn.
#include "cross_attention_device.h"

namespace s2 {

namespace {

typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
    typedef float f2 __attribute__((ext_vector_type(2)));
    if constexpr (T == 1) {
        typedef __bf16 b2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{lo, hi}), b2));
    } else {
        typedef _Float16 h2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(uint32_t, __builtin_convertvector((f2{lo, hi}), h2));
    }
}

// Four keys' values of one column: lane i of each 16 supplies 8 bytes of row i / 4, and gets
// column i of the four rows.
__device__ __forceinline__ uint2 read_columns(const uint8_t* p) {
    typedef __attribute__((address_space(3))) s16x4* Lds;
    return __builtin_bit_cast(uint2, __builtin_amdgcn_ds_read_tr16_b64_v4i16((Lds)p));
}

// fp16 weights reach 2^14 so that its subnormal numbers begin 2^-28 below the largest;
// 2^8 where a row's maximum is 8 past m.
template <int T>
constexpr float kShift = T == 2 ? 6.f : 0.f;

// A read of 16 bytes a lane is done 16 lanes at a time, one of 8 bytes 32 lanes, each 256
// bytes on 64 banks.  Chunk c (16 bytes) of row r of a k tile stands at c ^ key(r):
// 16 rows of one chunk lie on distinct banks.  Of v, eight rows of a pair of chunks do.
template <int DP>
struct Swizzle {
    static __device__ __forceinline__ int key(int r) { return DP == 64 ? (r >> 1) & 7 : r & 15; }
    static __device__ __forceinline__ int value(int r) { return DP == 64 ? ((r >> 1) & 3) * 2 : (r & 7) * 2; }
};

// Two weights' sum and l.
template <int T>
__device__ __forceinline__ float add_pair(uint32_t p, float l) {
    typedef __bf16 b2 __attribute__((ext_vector_type(2)));
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    if constexpr (T == 1)
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(b2, p), __builtin_bit_cast(b2, 0x3f803f80u), l,
                                               false);
    else
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(h2, p), __builtin_bit_cast(h2, 0x3c003c00u), l, false);
}

// Four values as out's 16-bit type.
__device__ __forceinline__ u32x2 out4(const CrossArgs& a, f32x4 v) {
    if (a.out_kind == 1) return u32x2{pack2_bf16_rne(v[0], v[1]), pack2_bf16_rne(v[2], v[3])};
    return u32x2{pack2_f16_rne(v[0], v[1]), pack2_f16_rne(v[2], v[3])};
}

// A wave's 32 rows: q, the sums and softmax's state.  DP: d rounded up to 64, 128 or 256; lds:
// the stages of KeyTiles.
template <int T, int DP>
struct WaveRows {
    static constexpr int RB = DP * 2, KB = kTileKeys * RB;   // bytes of a row in LDS, of a tile of k
    static constexpr int NK = DP / 32, ND = DP / 16;         // product steps over d; column tiles
    static constexpr int NQ = 2;                             // 16-row tiles
    // 256 bytes further in a row the swizzles are the same
    static constexpr int KA = NK < 4 ? NK : 4, VA = ND < 8 ? ND : 8;
    int l16, g;
    uint32_t sign;
    float c;
    uint4 qf[NQ][NK];
    f32x4 o[ND][NQ];
    float m[NQ], l[NQ];   // l: of this lane's keys
    const uint8_t* kl[KA];
    const uint8_t* vl[VA];

    __device__ __forceinline__ WaveRows(const CrossArgs& a, const uint8_t* lds) {
        l16 = threadIdx.x & 15;
        g = (threadIdx.x & 63) >> 4;
        sign = a.scale < 0.f ? 0x80008000u : 0u;
        c = weight_scale(a);
#pragma unroll
        for (int kk = 0; kk < KA; ++kk) kl[kk] = lds + l16 * RB + (((4 * kk + g) ^ Swizzle<DP>::key(l16)) * 16);
        const int vrow = 4 * g + (l16 >> 2);   // of the lane's eight bytes of v, of 16 rows
#pragma unroll
        for (int dt = 0; dt < VA; ++dt)
            vl[dt] = lds + KB + vrow * RB + (l16 & 1) * 8 +
                     ((2 * dt + (l16 >> 1 & 1)) ^ Swizzle<DP>::value(vrow)) * 16;
    }

    // q of rows `first` on of the tile: row l16 of each 16, elements 32 kk + 8 g on; zeros past
    // d, the last row again past the rows
    __device__ __forceinline__ void load(const CrossArgs& a, const CrossTile& t, int first, uint4 (&q)[NQ][NK]) const {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            const uint16_t* p =
                (const uint16_t*)a.q + cross_row(a, a.qs, t, t.row0 + min(first + 16 * i + l16, t.rows - 1));
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                q[i][kk] = make_uint4(0, 0, 0, 0);
                if (32 * kk + 8 * g < a.d) q[i][kk] = *reinterpret_cast<const uint4*>(p + 32 * kk + 8 * g);
            }
        }
    }

    __device__ __forceinline__ void begin(const uint4 (&q)[NQ][NK]) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
#pragma unroll
            for (int kk = 0; kk < NK; ++kk)
                qf[i][kk] = make_uint4(q[i][kk].x ^ sign, q[i][kk].y ^ sign, q[i][kk].z ^ sign, q[i][kk].w ^ sign);
            m[i] = kLowest;
            l[i] = 0.f;
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) o[dt][i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
    }

    __device__ __forceinline__ uint4 key(int h, int kk, int st) const {
        return *(const uint4*)(kl[kk % KA] + (kk / KA * 256 + 16 * h * RB + st));
    }

    __device__ __forceinline__ uint4 value(int dt, int st) const {
        const uint8_t* p = vl[dt % VA] + (dt / VA * 256 + st);
        const uint2 v0 = read_columns(p), v1 = read_columns(p + 16 * RB);
        return make_uint4(v0.x, v0.y, v1.x, v1.y);
    }

    // The tile of keys at LDS offset ST.  between(), after the first reads are on their way,
    // gives the keys that count; MASK: there may be none.
    template <int ST, bool MASK, typename F>
    __device__ __forceinline__ void keys(F&& between) {
        // Reads ahead where registers are left for them: of v under the scores' products and the
        // softmax, where the compiler would read two operands at a time and wait (4096 on 21600
        // keys, 20 heads of 128, 824 us, 792 so; 21600 on 512 124 and 120; with heads of 64, four
        // waves a SIMD, 3% slower)
        constexpr int AHEAD = DP == 256 ? 0 : NK, VAHEAD = DP == 128 ? ND / 2 : 0;
        uint4 kf[2][NK];
#pragma unroll
        for (int kk = 0; kk < AHEAD; ++kk) kf[0][kk] = key(0, kk, ST);
        asm volatile("" ::: "memory");
        const uint32_t valid = between();
        if (MASK && valid == 0) return;
        f32x4 s[2][NQ];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                if (h || kk >= AHEAD) kf[h][kk] = key(h, kk, ST);
#pragma unroll
                for (int i = 0; i < NQ; ++i)
                    s[h][i] = mfma<T>(kf[h][kk], qf[i][kk], kk ? s[h][i] : f32x4{0.f, 0.f, 0.f, 0.f});
            }
        uint4 vf[ND];
#pragma unroll
        for (int dt = 0; dt < VAHEAD; ++dt) vf[dt] = value(dt, ST);
        asm volatile("" ::: "memory");
        if constexpr (VAHEAD != 0) {   // reads between the products
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                __builtin_amdgcn_sched_group_barrier(8, NQ, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
#pragma unroll
            for (int kk = 0; kk < NK; ++kk) {
                __builtin_amdgcn_sched_group_barrier(8, NQ, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 2 * VAHEAD / NK, 0);
            }
        }
        // other waves' products run beside this wave's exponentials
        __builtin_amdgcn_s_setprio(1);
        if (valid != ~0u) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const uint32_t v4 = valid >> (16 * h + 4 * g);
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int i = 0; i < NQ; ++i)
                        if (!(v4 >> r & 1)) s[h][i][r] = -__builtin_inff();
            }
        }
        float top[NQ];
        bool due = false;
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            float x = fmaxf(fmaxf(s[0][i][0], s[0][i][1]), s[0][i][2]);
            x = fmaxf(fmaxf(x, s[0][i][3]), s[1][i][0]);
            x = fmaxf(fmaxf(x, s[1][i][1]), s[1][i][2]);
            top[i] = fmaxf(x, s[1][i][3]);
            due |= (top[i] - m[i]) * c > kLazy;
        }
        if (__any(due)) {
#pragma unroll
            for (int i = 0; i < NQ; ++i) {
                const float x = fmaxf(max_groups(top[i]), m[i]);
                const float fade = __builtin_amdgcn_exp2f((m[i] - x) * c);
                m[i] = x;
                l[i] *= fade;
#pragma unroll
                for (int dt = 0; dt < ND; ++dt) o[dt][i] *= fade;
            }
        }
        uint4 pb[NQ];
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            auto weight = [&](float score) {
                const float x = score - m[i];
                return __builtin_amdgcn_exp2f(kShift<T> != 0.f ? fmaf(x, c, kShift<T>) : x * c);
            };
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
                w[e] = pack2<T>(weight(s[e >> 1][i][2 * (e & 1)]), weight(s[e >> 1][i][2 * (e & 1) + 1]));
            pb[i] = make_uint4(w[0], w[1], w[2], w[3]);
#pragma unroll
            for (int e = 0; e < 4; ++e) l[i] = add_pair<T>(w[e], l[i]);
        }
        __builtin_amdgcn_s_setprio(0);
#pragma unroll
        for (int dt = 0; dt < ND; ++dt) {
            if (dt >= VAHEAD) vf[dt] = value(dt, ST);
#pragma unroll
            for (int i = 0; i < NQ; ++i) o[dt][i] = mfma<T>(vf[dt], pb[i], o[dt][i]);
        }
        if constexpr (VAHEAD != 0) {
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
                __builtin_amdgcn_sched_group_barrier(8, NQ, 0);
                if (dt < ND - VAHEAD) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
            }
        }
    }

    // Rows `first` on of the tile to out, or to their part.
    __device__ __forceinline__ void store(const CrossArgs& a, const CrossTile& t, const CrossParts& parts, int first) {
#pragma unroll
        for (int i = 0; i < NQ; ++i) {
            l[i] = sum_groups(l[i]);
            const int r = first + 16 * i + l16;
            if (r >= t.rows) continue;   // (all four lanes of a row)
            if (parts.parts > 1) {
                const long at = cross_part(a, parts, t, t.row0 + r);
                if (g == 0) parts.weights[at] = make_float2(m[i], l[i]);
#pragma unroll
                for (int dt = 0; dt < ND; ++dt)
                    if (16 * dt + 4 * g < a.d)
                        *reinterpret_cast<f32x4*>(parts.sums + at * a.d + 16 * dt + 4 * g) = o[dt][i];
                continue;
            }
            const float scale = l[i] == 0.f ? 0.f : 1.f / l[i];
            const long at = cross_row(a, a.os, t, t.row0 + r);
            if (a.out_kind == 0) {
#pragma unroll
                for (int dt = 0; dt < ND; ++dt)
                    if (16 * dt + 4 * g < a.d) store4_any<0>(a.out, at + 16 * dt + 4 * g, o[dt][i] * scale);
                continue;
            }
            // two column tiles' values change lanes, so that a lane has eight neighbours
#pragma unroll
            for (int dt = 0; dt < ND; dt += 2) {
                u32x2 x = out4(a, o[dt][i] * scale), y = out4(a, o[dt + 1][i] * scale);
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    auto w = __builtin_amdgcn_permlane32_swap(x[e], y[e], false, false);
                    w = __builtin_amdgcn_permlane16_swap(w[0], w[1], false, false);
                    x[e] = w[0];
                    y[e] = w[1];
                }
                const int col = 16 * (dt + (g >> 1)) + 8 * (g & 1);
                if (col < a.d)
                    *reinterpret_cast<u32x4_at2*>((uint16_t*)a.out + at + col) = u32x4{x[0], x[1], y[0], y[1]};
            }
        }
    }
};

// STAGES: of LDS; WGS: workgroups on a compute unit.
template <int T, int DP, int STAGES, int WGS, bool MASK>
__global__ __launch_bounds__(256, WGS) void cross_tile_kernel(CrossArgs a, int tiles, CrossParts parts) {
    typedef WaveRows<T, DP> Rows;
    constexpr int SB = 2 * Rows::KB;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * SB];
    __shared__ uint64_t bits[MASK ? kMaskBits : 1];
    const CrossTile t = cross_tile(a, kTileRows, tiles, parts.parts);
    if (t.rows <= 0) return;   // the whole workgroup
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int row_w = 32 * wave;   // of the wave's first row in the tile
    const int nk = MASK ? keys_kept(a, t) : __builtin_amdgcn_readfirstlane(t.s.nk);
    const int all = (nk + kTileKeys - 1) / kTileKeys;
    const int kb = (int)((long)all * t.part / parts.parts), ke = (int)((long)all * (t.part + 1) / parts.parts);

    KeyTiles<2, DP, STAGES, MASK, Swizzle<DP>> kv(a, t, nk, kb, (uint32_t)(uintptr_t)lds, bits);
    uint32_t counts[STAGES] = {};   // keys of the stages' tiles that count
    if (kb < ke) counts[0] = kv.issue(kb, 0, true);
    if (STAGES > 2 && kb + 1 < ke) counts[1] = kv.issue(kb + 1, 1, false);

    if (row_w >= t.rows) {   // a wave without rows takes part in loads and barriers alone
        for (int kt = kb; kt < ke; ++kt) {
            kv.await(kt, ke);
            if (kt + STAGES - 1 < ke) kv.issue(kt + STAGES - 1, (kt - kb + STAGES - 1) % STAGES, false);
        }
        return;
    }

    Rows rows(a, lds);
    {
        uint4 q[Rows::NQ][Rows::NK];
        rows.load(a, t, row_w, q);
        rows.begin(q);
    }
    // q is there before the loop, in a way that the compiler sees: with these loads perhaps in
    // flight it would wait for all of the DMA in every tile
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0)

    // unrolled by the stages, so that LDS addresses are registers and constants
    auto tile = [&](int kt, auto stage) {
        constexpr int ST = decltype(stage)::value;
        kv.await(kt, ke);   // and tile kt - 1 is no longer read
        rows.template keys<ST * SB, MASK>([&] {   // the loads' issue
            constexpr int NEXT = (ST + STAGES - 1) % STAGES;
            const uint32_t now = counts[ST];
            if (kt + STAGES - 1 < ke) counts[NEXT] = kv.issue(kt + STAGES - 1, NEXT, false);
            return now;
        });
    };
#pragma unroll 1
    for (int kt = kb; kt < ke; kt += STAGES) {
        tile(kt, std::integral_constant<int, 0>{});
        if (kt + 1 < ke) tile(kt + 1, std::integral_constant<int, 1>{});
        if constexpr (STAGES > 2)
            if (kt + 2 < ke) tile(kt + 2, std::integral_constant<int, 2>{});
    }
    rows.store(a, t, parts, row_w);
}

// Many rows of d from 65 to 128 on few keys: all of a head's keys stay in LDS, up to 128 of
// them, for `run` times 128 rows, so that waves meet at no barrier and q, loaded a turn
// ahead, and out are all that moves (21600 queries on 77 keys, 20 heads of 128: 59 us by the
// kernel above, 52 so, 4.3 TB/s; with heads of 64 no gain).  Samples of more keys are
// read again for every 128 rows.
template <int T, bool MASK>
__global__ __launch_bounds__(256, kShortEach) void cross_short_kernel(CrossArgs a, int tiles, int run) {
    constexpr int DP = 128, TILES = kShortKeys / kTileKeys;
    static_assert(TILES == 4, "the tiles' unrolling");
    typedef WaveRows<T, DP> Rows;
    constexpr int SB = 2 * Rows::KB;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[TILES * SB];
    __shared__ uint64_t bits[MASK ? kMaskBits : 1];
    const CrossTile t = cross_tile(a, kTileRows * run, tiles, 1);
    if (t.rows <= 0) return;   // the whole workgroup
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int nk = MASK ? keys_kept(a, t) : __builtin_amdgcn_readfirstlane(t.s.nk);
    const int all = (nk + kTileKeys - 1) / kTileKeys;
    typedef KeyTiles<2, DP, TILES, MASK, Swizzle<DP>> Keys;
    Keys kv(a, t, nk, 0, (uint32_t)(uintptr_t)lds, bits);
    auto load = [&](int k0) {   // tiles k0 .. k0 + TILES - 1
        for (int s = 0; s < TILES && k0 + s < all; ++s) kv.issue(k0 + s, s, k0 + s == 0);
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __syncthreads();
    };
    Rows rows(a, lds);
    uint4 q[Rows::NQ][Rows::NK];
    rows.load(a, t, min(32 * wave, t.rows - 1), q);
    if (all <= TILES) load(0);
#pragma unroll 1
    for (int first = 32 * wave, r = 0; r < t.rows; r += kTileRows, first += kTileRows) {
        rows.begin(q);
        if (first + kTileRows < t.rows) rows.load(a, t, first + kTileRows, q);
        for (int k0 = 0; k0 < all; k0 += TILES) {
            if (all > TILES) {
                __syncthreads();   // the tiles before are no longer read
                if (k0 == 0) kv = Keys(a, t, nk, 0, (uint32_t)(uintptr_t)lds, bits);
                load(k0);
            }
            if (first >= t.rows) continue;
            auto tile = [&](auto stage) {
                constexpr int ST = decltype(stage)::value;
                if (k0 + ST < all) rows.template keys<ST * SB, MASK>([&] { return kv.valid(k0 + ST); });
            };
            tile(std::integral_constant<int, 0>{});
            tile(std::integral_constant<int, 1>{});
            tile(std::integral_constant<int, 2>{});
            tile(std::integral_constant<int, 3>{});
        }
        if (first < t.rows) rows.store(a, t, CrossParts{1, nullptr, nullptr}, first);
    }
}

template <int T>
hipError_t launch_short(const CrossArgs& a, const CrossPlan& p, hipStream_t stream) {
    return launch_in_turn(a, (long)p.tiles * a.kv_heads, [&](const CrossArgs& part, unsigned nb) {
        if (part.key_mask)
            cross_short_kernel<T, true><<<nb, 256, 0, stream>>>(part, p.tiles, p.run);
        else
            cross_short_kernel<T, false><<<nb, 256, 0, stream>>>(part, p.tiles, p.run);
    });
}

template <int T, int DP, int STAGES, int WGS>
hipError_t launch(const CrossArgs& a, int tiles, const CrossParts& parts, hipStream_t stream) {
    return launch_in_turn(a, (long)tiles * a.kv_heads * parts.parts, [&](const CrossArgs& part, unsigned nb) {
        if (part.key_mask)
            cross_tile_kernel<T, DP, STAGES, WGS, true><<<nb, 256, 0, stream>>>(part, tiles, parts);
        else
            cross_tile_kernel<T, DP, STAGES, WGS, false><<<nb, 256, 0, stream>>>(part, tiles, parts);
    });
}

template <int T>
hipError_t launch_t(const CrossArgs& a, const CrossPlan& p, const CrossParts& parts, hipStream_t stream) {
    if (p.run > 1) return launch_short<T>(a, p, stream);
    if (a.d > 128) return launch<T, 256, 2, 2>(a, p.tiles, parts, stream);
    if (a.d > 64) return launch<T, 128, 3, 3>(a, p.tiles, parts, stream);
    return launch<T, 64, 3, 4>(a, p.tiles, parts, stream);
}

}  // namespace

hipError_t launch_cross_tiles(const CrossArgs& a, const CrossPlan& plan, void* workspace, hipStream_t stream) {
    const CrossParts parts = cross_parts(a, plan, workspace);
    return a.kind == 1 ? launch_t<1>(a, plan, parts, stream) : launch_t<2>(a, plan, parts, stream);
}

}  // namespace s2
