// Cross attention of fp32 operands on tiles of rows.
//
// As the 16-bit kernel, on 16x16x4 products in fp32, whose rate (157 TFLOP/s) bounds it: a
// wave has 16 rows.  A lane takes 16 bytes of k (four elements of d, one for each of four
// products) and 16 bytes of v, four columns of one key: column tile j of 64 columns is 4 i + j,
// i = 0 .. 15, so that the four accumulators of a lane and register are neighbours.
// Scores' registers are the second product's operand as they stand, a key a register, and
// nothing is rounded between.  Long keys run at 127 to 135 TFLOP/s; 1024 on 300, eight heads
// of 64 in two samples, 20 us, a workgroup a unit.
#include "cross_attention_device.h"

namespace s2 {

namespace {

// 16 rows of one chunk of k lie on distinct banks; of v a read takes whole rows.
struct Swizzle32 {
    static __device__ __forceinline__ int key(int r) { return r & 15; }
    static __device__ __forceinline__ int value(int) { return 0; }
};

// DP: d rounded up to 64, 128 or 256.  WGS: workgroups on a compute unit.
template <int DP, int WGS, bool MASK>
__global__ __launch_bounds__(256, WGS) void cross_f32_kernel(CrossArgs a, int tiles, CrossParts parts) {
    constexpr int KT = kTileKeys, BM = kTileRows32, STAGES = 2;
    constexpr int RB = DP * 4, KB = KT * RB, SB = 2 * KB;   // bytes: a row, a tile, a stage
    constexpr int NK = DP / 16, ND = DP / 64;
    __shared__ __attribute__((aligned(1024))) uint8_t lds[STAGES * SB];
    __shared__ uint64_t bits[MASK ? kMaskBits : 1];
    const CrossTile t = cross_tile(a, BM, tiles, parts.parts);
    if (t.rows <= 0) return;   // the whole workgroup
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int l16 = lane & 15, g = lane >> 4;
    const int nk = MASK ? keys_kept(a, t) : __builtin_amdgcn_readfirstlane(t.s.nk);
    const int all = (nk + KT - 1) / KT;
    const int kb = (int)((long)all * t.part / parts.parts), ke = (int)((long)all * (t.part + 1) / parts.parts);
    KeyTiles<4, DP, STAGES, MASK, Swizzle32> kv(a, t, nk, kb, (uint32_t)(uintptr_t)lds, bits);
    uint32_t counts[STAGES] = {};   // keys of the stages' tiles that count
    if (kb < ke) counts[0] = kv.issue(kb, 0, true);
    if (16 * wave >= t.rows) {   // a wave without rows takes part in loads and barriers alone
        for (int kt = kb; kt < ke; ++kt) {
            kv.await(kt, ke);
            if (kt + 1 < ke) kv.issue(kt + 1, (kt + 1 - kb) % STAGES, false);
        }
        return;
    }

    // q: row l16, elements 16 kk + 4 g on; zeros past d, the last row again past the rows
    const int row = 16 * wave + l16;
    const float c = weight_scale(a);
    const float sign = a.scale < 0.f ? -1.f : 1.f;
    f32x4 qf[NK];
    {
        const float* p = (const float*)a.q + cross_row(a, a.qs, t, t.row0 + min(row, t.rows - 1));
#pragma unroll
        for (int kk = 0; kk < NK; ++kk) {
            qf[kk] = f32x4{0.f, 0.f, 0.f, 0.f};
            if (16 * kk + 4 * g < a.d) qf[kk] = *reinterpret_cast<const f32x4*>(p + 16 * kk + 4 * g) * sign;
        }
    }
    __builtin_amdgcn_s_waitcnt(0x0F70);   // vmcnt(0): q, in a way that the compiler sees

    f32x4 o[ND][4];
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int j = 0; j < 4; ++j) o[n][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    float m = kLowest, l = 0.f;   // l: of this lane's keys
    constexpr int KA = NK < 4 ? NK : 4;   // 256 bytes further the swizzle is the same
    const uint8_t* kl[KA];
#pragma unroll
    for (int kk = 0; kk < KA; ++kk) kl[kk] = lds + l16 * RB + (((4 * kk + g) ^ Swizzle32::key(l16)) * 16);
    const uint8_t* vl = lds + KB + 4 * g * RB + l16 * 16;

    auto tile = [&](int kt, auto stage) {
        constexpr int ST = decltype(stage)::value * SB;
        kv.await(kt, ke);   // and tile kt - 1 is no longer read
        constexpr int NEXT = 1 - decltype(stage)::value;
        if (kt + 1 < ke) counts[NEXT] = kv.issue(kt + 1, NEXT, false);
        const uint32_t valid = counts[decltype(stage)::value];
        if (MASK && valid == 0) return;
        f32x4 s[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
        for (int kk = 0; kk < NK; ++kk)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const f32x4 kf = *(const f32x4*)(kl[kk % KA] + (kk / KA * 256 + 16 * h * RB + ST));
#pragma unroll
                for (int e = 0; e < 4; ++e) s[h] = __builtin_amdgcn_mfma_f32_16x16x4f32(kf[e], qf[kk][e], s[h], 0, 0, 0);
            }
        if (valid != ~0u) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int r = 0; r < 4; ++r)
                    if (!(valid >> (16 * h + 4 * g + r) & 1)) s[h][r] = -__builtin_inff();
        }
        float top = fmaxf(fmaxf(s[0][0], s[0][1]), s[0][2]);
        top = fmaxf(fmaxf(top, s[0][3]), s[1][0]);
        top = fmaxf(fmaxf(top, s[1][1]), s[1][2]);
        top = fmaxf(top, s[1][3]);
        if (__any((top - m) * c > kLazy)) {
            const float x = fmaxf(max_groups(top), m);
            const float fade = __builtin_amdgcn_exp2f((m - x) * c);
            m = x;
            l *= fade;
#pragma unroll
            for (int n = 0; n < ND; ++n)
#pragma unroll
                for (int j = 0; j < 4; ++j) o[n][j] *= fade;
        }
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int r = 0; r < 4; ++r) s[h][r] = __builtin_amdgcn_exp2f((s[h][r] - m) * c);
            l += (s[h][0] + s[h][1]) + (s[h][2] + s[h][3]);
        }
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int n = 0; n < ND; ++n) {
                    const f32x4 vf = *(const f32x4*)(vl + ((16 * h + r) * RB + n * 256 + ST));
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        o[n][j] = __builtin_amdgcn_mfma_f32_16x16x4f32(vf[j], s[h][r], o[n][j], 0, 0, 0);
                }
    };
#pragma unroll 1
    for (int kt = kb; kt < ke; kt += STAGES) {
        tile(kt, std::integral_constant<int, 0>{});
        if (kt + 1 < ke) tile(kt + 1, std::integral_constant<int, 1>{});
    }

    l = sum_groups(l);
    if (row >= t.rows) return;
    const float scale = l == 0.f ? 0.f : 1.f / l;
    const long at = parts.parts > 1 ? cross_part(a, parts, t, t.row0 + row) : cross_row(a, a.os, t, t.row0 + row);
    if (parts.parts > 1 && g == 0) parts.weights[at] = make_float2(m, l);
#pragma unroll
    for (int n = 0; n < ND; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int col = 64 * n + 16 * g + 4 * r;
            const f32x4 v = {o[n][0][r], o[n][1][r], o[n][2][r], o[n][3][r]};
            if (col >= a.d) continue;
            if (parts.parts > 1)
                *reinterpret_cast<f32x4*>(parts.sums + at * a.d + col) = v;
            else
                store4_out(a, at + col, v * scale);
        }
}

template <int DP, int WGS>
hipError_t launch(const CrossArgs& a, const CrossPlan& p, const CrossParts& parts, hipStream_t stream) {
    return launch_in_turn(a, (long)p.tiles * a.kv_heads * p.parts, [&](const CrossArgs& part, unsigned nb) {
        if (part.key_mask)
            cross_f32_kernel<DP, WGS, true><<<nb, 256, 0, stream>>>(part, p.tiles, parts);
        else
            cross_f32_kernel<DP, WGS, false><<<nb, 256, 0, stream>>>(part, p.tiles, parts);
    });
}

}  // namespace

hipError_t launch_cross_f32(const CrossArgs& a, const CrossPlan& plan, void* workspace, hipStream_t stream) {
    const CrossParts parts = cross_parts(a, plan, workspace);
    return a.d <= 64    ? launch<64, 4>(a, plan, parts, stream)
           : a.d <= 128 ? launch<128, 2>(a, plan, parts, stream)
                        : launch<256, 1>(a, plan, parts, stream);
}

}  // namespace s2
