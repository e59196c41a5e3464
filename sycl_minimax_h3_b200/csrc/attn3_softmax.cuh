// attn3_softmax.cuh - a half row of 64 scores in a softmax thread's registers: masking and maximum, and the exponentials
// packed to half. Shared by attn_sage3 (attn3.cuh) and attend_tc (attendtc.cu).
#pragma once
#include "attn_common.cuh"

namespace h3 {

// The int32 bits that become -inf once the bias is added: keys past S.
constexpr uint32_t kMaskedRaw = 0xFF800000u - kBias;

// One half row (64 keys) of scores r: keys at or past `valid` are masked. I8: r holds raw int32 sums; masked keys get
// kMaskedRaw, then the bias is added in place; returns the biased max. !I8: r holds fp32 scores; masked keys get -inf;
// returns the max.
template <bool I8>
__device__ __forceinline__ float sage3_bias_max(uint32_t (&r)[2][32], int valid) {
    if (valid < 64) {
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
            for (int i = 0; i < 32; ++i)
                if (c2 * 32 + i >= valid) r[c2][i] = I8 ? kMaskedRaw : 0xFF800000u;
    }
    if (I8) {
#pragma unroll
        for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
            for (int i = 0; i < 32; ++i) r[c2][i] += kBias;
    }
    return fmaxf(max32(r[0]), max32(r[1]));
}
// The exp argument's offset for running max m (log2 units) and scale c: I8 removes the bias too.
template <bool I8>
__device__ __forceinline__ float sage3_offset(float c, float m) {
    if (m == -INFINITY) return 0.0f;           // still no valid key: every weight is 0, not NaN
    return I8 ? -fmaf(kBiasF, c, m) : -m;
}
template <bool I8>
__device__ __forceinline__ float sage3_scaled_max(float bm, float c) {
    if (bm == -INFINITY) return -INFINITY;
    return I8 ? (bm - kBiasF) * c : bm * c;
}

// exp2 of one half row's 64 biased scores: p = 2^(r*c + k), rounded to half and packed two per word into pk; returns
// the sum of the p. FMAs and sums on packed f32x2 instructions.
__device__ __forceinline__ float sage3_exp_half(const uint32_t (&r)[2][32], float c, float k, uint32_t (&pk)[32]) {
    const float2 c2v = make_float2(c, c), k2v = make_float2(k, k);
    float2 sum[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
#pragma unroll
    for (int c2 = 0; c2 < 2; ++c2)
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            const float2 y = __ffma2_rn(make_float2(__uint_as_float(r[c2][2 * e]), __uint_as_float(r[c2][2 * e + 1])), c2v, k2v);
            float2 p;
            p.x = ex2(y.x);
            p.y = ex2(y.y);
            sum[e & 3] = __fadd2_rn(sum[e & 3], p);
            pk[c2 * 16 + e] = pack_half2(p.x, p.y);
        }
    const float2 s01 = __fadd2_rn(sum[0], sum[1]), s23 = __fadd2_rn(sum[2], sum[3]);
    const float2 s = __fadd2_rn(s01, s23);
    return s.x + s.y;
}

}  // namespace h3
