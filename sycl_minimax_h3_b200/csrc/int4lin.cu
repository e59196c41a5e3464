// int4lin.cu - a linear layer with 4-bit weights and a scale (and, where given, a zero point) for each group of inputs
// of an output, for the few rows of a step of the text model: bound by the weights' bytes.
//
//   y[m, n] = sum_groups scale[g, n] * sum_{k in g} x[m, k] (code[n, k] - zero[g, n])  + bias[n]
//
// The codes are kept in tiles of 16 outputs x 64 inputs, 512 bytes that a warp loads with one 16-byte load per lane and
// that are its A fragments of m16n8k16 products as they come: lane (g, t) = (lane / 4, lane % 4) has four words; word w
// holds the inputs 32 (w / 2) + 8 t + 4 (w % 2) + {0, 1, 2, 3} of outputs g and g + 8, nibble j + 4 e (bits 4 (j + 4 e)) the
// output g + 8 (j % 2) at input 2 (j / 2) + e of those four. Then (word >> 4 j) & 0x000f000f are two neighbouring inputs
// in the low bits of two 16-bit halves. Past N or K the code is 8.
//
// (code - 8) is exact in bf16 and fp16, so x in a 16-bit type enters the products as it is; float32 goes in as three
// bf16 terms of 8 bits each, all 24. A group's products are added up in 32 bits, then multiplied by its scale.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "attn_common.cuh"
#include "int4lin.cuh"
#include "prepass.cuh"

namespace h3 {
namespace {

constexpr int kI4Warps = 8;

template <int DT>
__device__ __forceinline__ void mma_x(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (DT == F16)
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                     : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                     : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// a word of codes as an A fragment: code + 1024 (fp16) or + 128 (bf16) in the bits of a number, minus that and 8
template <int DT>
__device__ __forceinline__ void frag(uint32_t word, uint32_t (&a)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t v = (word >> (4 * j)) & 0x000f000fu;
        if constexpr (DT == F16) {
            const uint32_t u = v | 0x64006400u;
            const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6408)));
            a[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const uint32_t u = v | 0x43004300u;
            const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u),
                                             __bfloat162bfloat162(__ushort_as_bfloat16(0x4308)));
            a[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
}

// 8 inputs of x as B fragments of two steps: TERMS sets of four words
template <int DT, int TERMS>
__device__ __forceinline__ void load_x(const Int4Args& a, long long m, int k, uint32_t (&b)[TERMS][4]) {
#pragma unroll
    for (int e = 0; e < TERMS; ++e)
#pragma unroll
        for (int i = 0; i < 4; ++i) b[e][i] = 0;
    if (m >= a.M || k >= a.K) return;
    const size_t at = (size_t) m * a.K + k;
    const bool whole = k + 8 <= a.K;
    if constexpr (DT == F32) {
        float x[8];
        if (whole && a.x_vec) {
            ld16<F32>(reinterpret_cast<const float*>(a.x) + at, x);
            ld16<F32>(reinterpret_cast<const float*>(a.x) + at + 4, x + 4);
        } else
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = k + i < a.K ? ld1<F32>(a.x, at + i) : 0.0f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // 8 bits at a time from the top, cut off: what is left over is exact. An infinity or a NaN stays in the first.
            float r = x[i];
            const bool fin = fabsf(r) <= 3.402823466e38f;
#pragma unroll
            for (int e = 0; e < TERMS; ++e) {
                uint32_t u = __float_as_uint(r) >> 16;
                if (!fin && e == 0 && r != r) u = 0x7fc0;
                b[e][i / 2] |= u << (16 * (i & 1));
                r = fin ? r - __uint_as_float(u << 16) : 0.0f;
            }
        }
    } else {
        const uint16_t* p = reinterpret_cast<const uint16_t*>(a.x) + at;
        if (whole && a.x_vec) {
            const uint4 u = *reinterpret_cast<const uint4*>(p);
            b[0][0] = u.x; b[0][1] = u.y; b[0][2] = u.z; b[0][3] = u.w;
        } else
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (k + i < a.K) b[0][i / 2] |= (uint32_t) p[i] << (16 * (i & 1));
    }
}

__device__ __forceinline__ float ld_dt(const void* p, size_t i, int dt) {
    return dt == F16 ? ld1<F16>(p, i) : dt == BF16 ? ld1<BF16>(p, i) : ld1<F32>(p, i);
}
__device__ __forceinline__ void st_dt(void* p, size_t i, float x, int dt) {
    if (dt == F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
    else if (dt == BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else reinterpret_cast<float*>(p)[i] = x;
}

// 16 outputs x 8 rows of x per CTA; its warps take the 64-input tiles in turn and their sums meet in shared memory.
template <int DT, bool ZERO>
__global__ void __launch_bounds__(kI4Warps * 32) int4_rows(const Int4Args a) {
    constexpr int TERMS = DT == F32 ? 3 : 1;
    constexpr int XT = DT == F16 ? F16 : BF16;
    __shared__ float red[kI4Warps][16][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int nt = (int) blockIdx.x, KT = (a.K + 63) / 64;
    const long long m0 = (long long) blockIdx.y * 8;
    const int n0 = nt * 16 + g, n1 = n0 + 8;
    float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    const uint4* tiles = a.tiles + (size_t) nt * KT * 32 + lane;
    const uint32_t ones[4] = {XT == F16 ? 0x3c003c00u : 0x3f803f80u, XT == F16 ? 0x3c003c00u : 0x3f803f80u,
                              XT == F16 ? 0x3c003c00u : 0x3f803f80u, XT == F16 ? 0x3c003c00u : 0x3f803f80u};
    for (int kt = warp; kt < KT; kt += kI4Warps) {
        const uint4 wv = tiles[(size_t) kt * 32];
        const uint32_t w[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
        for (int half = 0; half < 2; ++half) {
            const int k0 = kt * 64 + half * 32;
            if (k0 >= a.K) break;
            uint32_t b[TERMS][4];
            load_x<DT, TERMS>(a, m0 + g, k0 + 8 * t, b);
            float c[4] = {0.0f, 0.0f, 0.0f, 0.0f}, sx[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                uint32_t f[4];
                frag<XT>(w[half * 2 + u], f);
#pragma unroll
                for (int e = 0; e < TERMS; ++e) {
                    mma_x<XT>(c, f, b[e][2 * u], b[e][2 * u + 1]);
                    if constexpr (ZERO) mma_x<XT>(sx, ones, b[e][2 * u], b[e][2 * u + 1]);
                }
            }
            const size_t gi = (size_t) (k0 / a.group) * a.N;
            const float s0 = n0 < a.N ? ld_dt(a.scale, gi + n0, a.s_dt) : 0.0f;
            const float s1 = n1 < a.N ? ld_dt(a.scale, gi + n1, a.s_dt) : 0.0f;
            if constexpr (ZERO) {
                const float z0 = n0 < a.N ? ld_dt(a.zero, gi + n0, a.s_dt) - 8.0f : 0.0f;
                const float z1 = n1 < a.N ? ld_dt(a.zero, gi + n1, a.s_dt) - 8.0f : 0.0f;
#pragma unroll
                for (int i = 0; i < 4; ++i) c[i] = fmaf(-(i < 2 ? z0 : z1), sx[i], c[i]);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) acc[i] = fmaf(i < 2 ? s0 : s1, c[i], acc[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) red[warp][g + 8 * (i >> 1)][2 * t + (i & 1)] = acc[i];
    __syncthreads();
    if (threadIdx.x < 128) {
        const int n = nt * 16 + (int) (threadIdx.x & 15), col = threadIdx.x >> 4;
        const long long m = m0 + col;
        if (n < a.N && m < a.M) {
            float y = 0.0f;
#pragma unroll
            for (int w = 0; w < kI4Warps; ++w) y += red[w][threadIdx.x & 15][col];
            if (a.bias) y += a.bias[n];
            st_dt(a.out, (size_t) m * a.N + n, y, a.out_dt);
        }
    }
}

// codes [N, K / 2], two to a byte, the even input in the low four bits -> tiles
__global__ void int4_pack(const uint8_t* __restrict__ codes, long long N, long long K, uint32_t* __restrict__ tiles) {
    const long long KT = (K + 63) / 64, words = (N + 15) / 16 * KT * 128;
    for (long long i = blockIdx.x * (long long) blockDim.x + threadIdx.x; i < words; i += (long long) gridDim.x * blockDim.x) {
        const int w = (int) (i & 3), t = (int) (i >> 2) & 3, g = (int) (i >> 4) & 7;
        const long long kt = (i >> 7) % KT, nt = (i >> 7) / KT;
        const long long k = kt * 64 + 32 * (w >> 1) + 8 * t + 4 * (w & 1);
        uint32_t word = 0;
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const long long n = nt * 16 + g + 8 * (j & 1), kk = k + 2 * (j >> 1) + e;
                uint32_t c = 8;
                if (n < N && kk < K) c = (codes[n * (K / 2) + kk / 2] >> (4 * (kk & 1))) & 15u;
                word |= c << (4 * (j + 4 * e));
            }
        tiles[i] = word;
    }
}

}  // namespace

template <int DT>
cudaError_t int4_dt(const Int4Args& a, cudaStream_t st) {
    const dim3 grid((unsigned) ((a.N + 15) / 16), (unsigned) ((a.M + 7) / 8));
    if (a.zero) int4_rows<DT, true><<<grid, kI4Warps * 32, 0, st>>>(a);
    else int4_rows<DT, false><<<grid, kI4Warps * 32, 0, st>>>(a);
    return cudaGetLastError();
}

cudaError_t launch_int4_linear(const Int4Args& a, int, cudaStream_t st) {
    switch (a.x_dt) {
        case F16: return int4_dt<F16>(a, st);
        case BF16: return int4_dt<BF16>(a, st);
        default: return int4_dt<F32>(a, st);
    }
}

cudaError_t launch_int4_pack(const uint8_t* codes, long long N, long long K, void* tiles, int n_sm, cudaStream_t st) {
    int4_pack<<<(unsigned) (n_sm * 8), 256, 0, st>>>(codes, N, K, static_cast<uint32_t*>(tiles));
    return cudaGetLastError();
}

}  // namespace h3
