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
#include <atomic>

#include "attn_common.cuh"
#include "int4lin.cuh"
#include "prepass.cuh"

namespace h3 {
namespace {

constexpr int kI4Warps = 8;
constexpr int kErrInt4 = 128;          // a wait of the 4-bit layer's kernel gave up

template <int XT>
__device__ __forceinline__ void mma_x(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (XT == F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
            : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// the same from zero
template <int XT>
__device__ __forceinline__ void mma_x0(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    if constexpr (XT == F16)
        asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
    else
        asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
            : "=f"(c[0]), "=f"(c[1]), "=f"(c[2]), "=f"(c[3])
            : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1), "f"(0.0f));
}

// a word of codes as an A fragment: code + 1024 (fp16) or + 128 (bf16) in the bits of a number, minus that and 8
template <int XT>
__device__ __forceinline__ void frag(uint32_t word, uint32_t (&a)[4]) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t u = ((word >> (4 * j)) & 0x000f000fu) | (XT == F16 ? 0x64006400u : 0x43004300u);
        if constexpr (XT == F16) {
            const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6408)));
            a[j] = *reinterpret_cast<const uint32_t*>(&h);
        } else {
            const __nv_bfloat162 h = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&u),
                                             __bfloat162bfloat162(__ushort_as_bfloat16(0x4308)));
            a[j] = *reinterpret_cast<const uint32_t*>(&h);
        }
    }
}

// 8 inputs of x as they lie in memory: row m (one of x's) from input k on, past the inputs zeros. whole: all of them are
// there, on 16 bytes.
template <int DT>
struct Raw {
    uint4 u[DT == F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw<DT> load_raw(const Int4Args& a, const char* row, int k, bool whole) {
    Raw<DT> r{};
    const char* p = row + (size_t) k * DtInfo<DT>::ES;
    if (whole) {
        r.u[0] = *reinterpret_cast<const uint4*>(p);
        if constexpr (DT == F32) r.u[1] = *reinterpret_cast<const uint4*>(p + 16);
    } else {
        uint32_t w[8] = {};
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (k + i < a.K) {
                if constexpr (DT == F32) w[i] = reinterpret_cast<const uint32_t*>(p)[i];
                else w[i / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(p)[i] << (16 * (i & 1));
            }
        r.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (DT == F32) r.u[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
    return r;
}
// ... as B fragments of two steps: TERMS sets of four words
template <int DT, int TERMS>
__device__ __forceinline__ void terms(const Raw<DT>& r, uint32_t (&b)[TERMS][4]) {
    if constexpr (DT == F32) {
#pragma unroll
        for (int e = 0; e < TERMS; ++e)
#pragma unroll
            for (int i = 0; i < 4; ++i) b[e][i] = 0;
        const uint32_t w[8] = {r.u[0].x, r.u[0].y, r.u[0].z, r.u[0].w, r.u[1].x, r.u[1].y, r.u[1].z, r.u[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            // 8 bits at a time from the top, cut off: what is left over is exact. An infinity or a NaN stays in the first.
            float x = __uint_as_float(w[i]);
            const bool fin = fabsf(x) <= 3.402823466e38f;
#pragma unroll
            for (int e = 0; e < TERMS; ++e) {
                uint32_t u = __float_as_uint(x) >> 16;
                if (!fin && e == 0 && x != x) u = 0x7fc0;
                b[e][i / 2] |= u << (16 * (i & 1));
                x = fin ? x - __uint_as_float(u << 16) : 0.0f;
            }
        }
    } else {
        b[0][0] = r.u[0].x; b[0][1] = r.u[0].y; b[0][2] = r.u[0].z; b[0][3] = r.u[0].w;
    }
}

// A scale or zero point as its bits, and what they stand for: apart, so that the load is not waited for where it is made.
__device__ __forceinline__ uint32_t ld_bits(const void* p, size_t i, int dt) {
    return dt == F32 ? reinterpret_cast<const uint32_t*>(p)[i] : reinterpret_cast<const uint16_t*>(p)[i];
}
__device__ __forceinline__ float bits_value(uint32_t u, int dt) {
    return dt == F16 ? __half2float(__ushort_as_half((uint16_t) u)) : __uint_as_float(dt == BF16 ? u << 16 : u);
}
__device__ __forceinline__ void st_dt(void* p, size_t i, float x, int dt) {
    if (dt == F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
    else if (dt == BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else reinterpret_cast<float*>(p)[i] = x;
}

// Output n of row m without its bias, term by term as the layer is defined and in 64 bits, for sums that are not finite in
// the kernels. These form sum x (code - 8) and (8 - zero) sum x apart, and multiply by the scale last: an infinite x is then
// 0 times infinity for the code 8, or infinity less infinity, where the definition has an infinity, and a large x passes
// float's largest where scale (code - zero) x does not. One thread reads a whole row for it (some milliseconds for 14,336
// inputs); a finite sum never comes here, and what is not finite on the way to a sum stays not finite.
__device__ __noinline__ float int4_exact(const Int4Args& a, long long m, int n) {
    const long long KT = (a.K + 63) / 64;
    const uint2* tile = reinterpret_cast<const uint2*>(a.tiles + (n / 16) * KT * 32 + (n & 7) * 4);
    const int up = 4 * ((n >> 3) & 1);                     // outputs 8-15 of a strip: the odd nibbles
    double y = 0.0;
    for (int k0 = 0; k0 < a.K; k0 += 8) {                  // 8 inputs: a pair of a lane's words, within one group
        const uint2 u = tile[(k0 / 64) * 64 + (k0 / 8 % 4) * 2 + k0 / 32 % 2];
        const size_t at = (size_t) (k0 >> a.group_shift) * a.N + n;
        const double s = bits_value(ld_bits(a.scale, at, a.s_dt), a.s_dt);
        const double z = a.zero ? bits_value(ld_bits(a.zero, at, a.s_dt), a.s_dt) : 8.0f;
        const int count = min(8, a.K - k0);
        for (int i = 0; i < count; ++i) {
            const uint32_t word = i < 4 ? u.x : u.y;
            const int code = (word >> (8 * (i / 2 % 2) + up + 16 * (i & 1))) & 15;
            const double x = bits_value(ld_bits(a.x, (size_t) m * a.K + k0 + i, a.x_dt), a.x_dt);
            y += s * (((double) code - z) * x);
        }
        if (y != y) break;
    }
    return (float) y;
}
__device__ __forceinline__ bool is_finite(float x) { return fabsf(x) <= 3.402823466e38f; }

// Scales and zero points of two outputs for the halves of a 64-input tile (one for both where a group has more than 32
// inputs), as bits. An output past the last reads the last one's: its sums are not stored.
template <bool ZERO, bool G32>
struct Scales {
    uint32_t s[G32 ? 2 : 1][2];
    uint32_t z[ZERO ? (G32 ? 2 : 1) : 1][2];
};
template <bool ZERO, bool G32>
__device__ __forceinline__ void load_scales(const Int4Args& a, int kt, int n0, int n1, Scales<ZERO, G32>& sc) {
    const size_t i = (size_t) ((kt * 64) >> a.group_shift) * a.N;
#pragma unroll
    for (int half = 0; half < (G32 ? 2 : 1); ++half) {
        if (half == 1 && kt * 64 + 32 >= a.K) break;
        const size_t at = i + (half ? a.N : 0);
        sc.s[half][0] = ld_bits(a.scale, at + n0, a.s_dt);
        sc.s[half][1] = ld_bits(a.scale, at + n1, a.s_dt);
        if constexpr (ZERO) {
            sc.z[half][0] = ld_bits(a.zero, at + n0, a.s_dt);
            sc.z[half][1] = ld_bits(a.zero, at + n1, a.s_dt);
        }
    }
}

// ---- up to 8 rows ----------------------------------------------------------------------------------------------------
// RT strips of 16 outputs per CTA; its 8 warps take the 64-input tiles in turn, each with the loads of the next one under
// way, and their sums meet in shared memory.
// One row of 4096 inputs to 12288 outputs in bf16, groups of 128: 11.2 us (25 MB at 2.25 TB/s; the bytes alone 3.9), 28672
// outputs 22.7 us, 8 rows of 12288 12.0 us; groups of 32 with zero points 17.7 us, float32 22.7 us. Not memory's rate bounds it
// (10.4 us with the codes in L2) but instructions and the waits between them: 27 per word of 8 codes and lane, of which
// unpacking is 11, while the schedulers issue 58 % of the time, for a warp has eight tiles, two of them under way, and starts
// and ends with nothing to do. Codes through a ring of bulk copies, eight tiles ahead, took 14.2 us: more instructions, and
// no wait less.
template <int DT, int SDT, bool ZERO, bool G32, int RT>
__global__ void __launch_bounds__(kI4Warps * 32, DT == F32 ? 2 : 3) int4_few(const __grid_constant__ Int4Args a) {
    constexpr int TERMS = DT == F32 ? 3 : 1, ES = DtInfo<DT>::ES, SES = DtInfo<SDT>::ES, NS = G32 ? 2 : 1;
    constexpr int XT = DT == F16 ? F16 : BF16;
    __shared__ float red[kI4Warps][16 * RT][8];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int KT = (a.K + 63) / 64, strips = (a.N + 15) / 16;
    float acc[RT][4];
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[r][i] = 0.0f;
    // what this lane reads of tile kt = warp: codes, x, scales, zero points; each moves on by as much for every 8 tiles.
    // A strip, an output or a row past the last repeats it, and is not stored.
    const uint4* tp[RT];
    int ns[RT][2];
#pragma unroll
    for (int r = 0; r < RT; ++r) {
        tp[r] = a.tiles + ((size_t) min((int) blockIdx.x * RT + r, strips - 1) * KT + warp) * 32 + lane;
#pragma unroll
        for (int i = 0; i < 2; ++i) ns[r][i] = min((int) (blockIdx.x * RT + r) * 16 + g + 8 * i, a.N - 1) * SES;
    }
    const char* row = static_cast<const char*>(a.x) + (size_t) min((int) a.M - 1, g) * a.K * ES;
    const char* xp = row + (warp * 64 + 8 * t) * ES;
    const size_t grow = (size_t) a.N * SES;                // a group's scales
    size_t sp = (size_t) ((warp * 64) >> a.group_shift) * grow;
    const size_t sstep = (size_t) ((kI4Warps * 64) >> a.group_shift) * grow;
    const int whole = a.x_vec ? a.K / 64 : 0;              // tiles whose inputs are all there, on 16 bytes
    constexpr uint32_t one = XT == F16 ? 0x3c003c00u : 0x3f803f80u;
    const uint32_t ones[4] = {one, one, one, one};
    struct Stage {
        uint4 w[RT];
        Raw<DT> x[2];
        uint32_t s[RT][NS][2], z[ZERO ? RT : 1][NS][2];
    } st[2] = {};
    auto bits = [](const char* p) -> uint32_t {
        if constexpr (SDT == F32) return *reinterpret_cast<const uint32_t*>(p);
        else return *reinterpret_cast<const uint16_t*>(p);
    };
    auto value = [](uint32_t u) { return bits_value(u, SDT); };
    auto load = [&](int kt, Stage& s) {
        if (kt >= KT) return;
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            s.w[r] = __ldcs(tp[r]);
            tp[r] += kI4Warps * 32;
        }
        // an odd last half of 32 inputs has no second group: its scales are read again (x is zero there)
        const size_t next = G32 && kt * 64 + 32 < a.K ? grow : 0;
#pragma unroll
        for (int r = 0; r < RT; ++r)
#pragma unroll
            for (int h = 0; h < NS; ++h)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    s.s[r][h][i] = bits(static_cast<const char*>(a.scale) + sp + (h ? next : 0) + ns[r][i]);
                    if constexpr (ZERO) s.z[r][h][i] = bits(static_cast<const char*>(a.zero) + sp + (h ? next : 0) + ns[r][i]);
                }
        sp += sstep;
        if (kt < whole) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                s.x[h].u[0] = *reinterpret_cast<const uint4*>(xp + 32 * h * ES);
                if constexpr (DT == F32) s.x[h].u[1] = *reinterpret_cast<const uint4*>(xp + 32 * h * ES + 16);
            }
        } else {
            s.x[0] = load_raw<DT>(a, row, kt * 64 + 8 * t, false);
            s.x[1] = load_raw<DT>(a, row, kt * 64 + 32 + 8 * t, false);
            __syncwarp();                                  // the lanes part at the inputs' end, the products are the whole warp's
        }
        xp += kI4Warps * 64 * ES;
    };
    auto add = [&](const Stage& s) {
        uint32_t b[2][TERMS][4];
        terms<DT, TERMS>(s.x[0], b[0]);
        terms<DT, TERMS>(s.x[1], b[1]);
        float sx[2][4];
        if constexpr (ZERO) {
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int e = 0; e < TERMS; ++e) {
                    if (e == 0 && (G32 || h == 0)) mma_x0<XT>(sx[h], ones, b[h][e][0], b[h][e][1]);
                    else mma_x<XT>(sx[G32 ? h : 0], ones, b[h][e][0], b[h][e][1]);
                    mma_x<XT>(sx[G32 ? h : 0], ones, b[h][e][2], b[h][e][3]);
                }
        }
#pragma unroll
        for (int r = 0; r < RT; ++r) {
            const uint32_t w[4] = {s.w[r].x, s.w[r].y, s.w[r].z, s.w[r].w};
            float c[4];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    uint32_t f[4];
                    frag<XT>(w[h * 2 + u], f);
#pragma unroll
                    for (int e = 0; e < TERMS; ++e) {
                        if (u == 0 && e == 0 && (G32 || h == 0)) mma_x0<XT>(c, f, b[h][e][2 * u], b[h][e][2 * u + 1]);
                        else mma_x<XT>(c, f, b[h][e][2 * u], b[h][e][2 * u + 1]);
                    }
                }
                if (!G32 && h == 0) continue;
                const int sh = G32 ? h : 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if constexpr (ZERO) c[i] = fmaf(8.0f - value(s.z[r][sh][i >> 1]), sx[sh][i], c[i]);
                    acc[r][i] = fmaf(value(s.s[r][sh][i >> 1]), c[i], acc[r][i]);
                }
            }
        }
    };
    load(warp, st[0]);
    for (int kt = warp; kt < KT; kt += 2 * kI4Warps) {
        load(kt + kI4Warps, st[1]);
        add(st[0]);
        if (kt + kI4Warps >= KT) break;
        load(kt + 2 * kI4Warps, st[0]);
        add(st[1]);
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < 4; ++i) red[warp][r * 16 + g + 8 * (i >> 1)][2 * t + (i & 1)] = acc[r][i];
    __syncthreads();
    if (threadIdx.x < 128 * RT) {
        const int c = threadIdx.x % (16 * RT), n = (int) blockIdx.x * 16 * RT + c, m = threadIdx.x / (16 * RT);
        if (n < a.N && m < a.M) {
            float y = 0.0f;
#pragma unroll
            for (int w = 0; w < kI4Warps; ++w) y += red[w][c][m];
            if (!is_finite(y)) y = int4_exact(a, m, n);
            if (a.bias) y += a.bias[n];
            st_dt(a.out, (size_t) m * a.N + n, y, a.out_dt);
        }
    }
}

// ---- 9 to 16 rows, and any number of rows of float32 -------------------------------------------------------------------------------------------------------
// 128 outputs x up to 64 rows per CTA: a warp has 16 outputs and every row, so that a tile is unpacked once for all of
// them; x comes through a ring in shared memory, 128 inputs at a time, of which warps 0-7 take the first 64 and warps
// 8-15 the others. A cluster of `split` CTAs divides the inputs. The sums meet in shared memory, always in one order.
// 16 rows of 14336 inputs to 4096 outputs in bf16 22.0 us (29 MB at 1.33 TB/s), with zero points 26.3; float32 33.8, 48 rows 79.
// A stage's barrier and the unpacking behind it bound it: the schedulers issue 46 % of the time with 16 warps on an SM.
constexpr int kRowsN = 128, kRowsM = 64, kRowsThreads = 512;

template <int TERMS>
struct RowsSmem {
    static constexpr int STAGES = TERMS == 1 ? 4 : 3;
    union {
        // [row][16-byte piece of 8 inputs]: odd rows have the halves of every 64 exchanged, so that the 8 lanes that read
        // together (two rows, four pieces) meet different banks
        uint4 x[STAGES][TERMS][kRowsM][16];
        float part[2 * kRowsM * kRowsN];                   // [source][row][output]
    };
};

template <int DT, bool ZERO, bool G32, int MT>
__global__ void __launch_bounds__(kRowsThreads, 1) int4_rows(const __grid_constant__ Int4Args a, int split) {
    constexpr int TERMS = DT == F32 ? 3 : 1;
    constexpr int XT = DT == F16 ? F16 : BF16;
    constexpr int ROWS = 8 * MT, STAGES = RowsSmem<TERMS>::STAGES, AHEAD = 3;
    constexpr int PIECES = (ROWS * 16 + kRowsThreads - 1) / kRowsThreads;
    constexpr uint32_t one = XT == F16 ? 0x3c003c00u : 0x3f803f80u;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    RowsSmem<TERMS>& sm = *reinterpret_cast<RowsSmem<TERMS>*>(smem_raw);
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3, wg = warp >> 3;
    const int part = (int) (blockIdx.x % split), KT = (a.K + 63) / 64, KP = (KT + 1) / 2;
    const int per = (KP + split - 1) / split, kp0 = min(KP, part * per), kp1 = min(KP, kp0 + per);
    const int block = (int) (blockIdx.x / split), strips = (a.N + 15) / 16;
    const int nt = min(block * (kRowsN / 16) + (warp & 7), strips - 1);    // a strip past the last repeats it, unstored
    const int n0 = min(nt * 16 + g, a.N - 1), n1 = min(nt * 16 + g + 8, a.N - 1);
    const long long m0 = (long long) blockIdx.y * ROWS;
    const uint4* tiles = a.tiles + (size_t) nt * KT * 32 + lane;
    const uint32_t ones[4] = {one, one, one, one};
    float acc[MT][4];
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int u = 0; u < 4; ++u) acc[i][u] = 0.0f;
    // this thread's pieces of a stage: row and first input, where they lie and where they go
    const char* src[PIECES];
    int kc[PIECES], dst[PIECES];
#pragma unroll
    for (int j = 0; j < PIECES; ++j) {
        const int i = threadIdx.x + j * kRowsThreads, r = i >> 4, c = i & 15;
        const long long m = min(m0 + r, a.M - 1);
        src[j] = static_cast<const char*>(a.x) + (size_t) m * a.K * DtInfo<DT>::ES;
        kc[j] = r < ROWS ? c * 8 : 1 << 30;                // no such piece: never inside
        dst[j] = r * 16 + (c ^ (4 * (r & 1)));
    }
    auto stage = [&](int kp, int slot) {                   // inputs 128 kp .. of x into a slot
        if (kp < kp1) {
#pragma unroll
            for (int j = 0; j < PIECES; ++j) {
                const int k = kp * 128 + kc[j];
                if (kc[j] > 128) continue;
                uint4* to = &sm.x[slot][0][0][0] + dst[j];
                if (DT != F32 && a.x_vec) {                // K is a multiple of 8: a piece is inside or outside
                    const uint32_t bytes = k < a.K ? 16 : 0;
                    const char* from = bytes ? src[j] + (size_t) k * 2 : src[j];
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_u32(to)), "l"(from), "r"(bytes) : "memory");
                } else {
                    uint32_t b[TERMS][4];
                    terms<DT, TERMS>(load_raw<DT>(a, src[j], k, a.x_vec && k + 8 <= a.K), b);
#pragma unroll
                    for (int e = 0; e < TERMS; ++e) to[e * kRowsM * 16] = make_uint4(b[e][0], b[e][1], b[e][2], b[e][3]);
                    __syncwarp();                          // (a warp has whole rows) the lanes part at the inputs' end
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    uint4 w[AHEAD];
    Scales<ZERO, G32> sc[AHEAD] = {};
    auto fetch = [&](int kp, int u) {
        const int kt = min(2 * kp + wg, KT - 1);           // past the last tile x is zeros
        if (kp < kp1) {
            w[u] = __ldcs(tiles + kt * 32);
            load_scales<ZERO, G32>(a, kt, n0, n1, sc[u]);
        }
    };
#pragma unroll
    for (int i = 0; i < STAGES - 1; ++i) stage(kp0 + i, i);
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) fetch(kp0 + u, u);
    int slot = 0;
    for (int base = kp0; base < kp1; base += AHEAD) {
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            const int kp = base + u;
            if (kp >= kp1) break;
            asm volatile("cp.async.wait_group %0;" ::"n"(STAGES - 2) : "memory");
            __syncthreads();                               // this stage is here, and nobody reads the one before any more
            stage(kp + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
            const uint32_t words[4] = {w[u].x, w[u].y, w[u].z, w[u].w};
            float sv[G32 ? 2 : 1][2], zv[G32 ? 2 : 1][2];
#pragma unroll
            for (int i = 0; i < (G32 ? 2 : 1); ++i)
#pragma unroll
                for (int r = 0; r < 2; ++r) {
                    sv[i][r] = bits_value(sc[u].s[i][r], a.s_dt);
                    zv[i][r] = ZERO ? 8.0f - bits_value(sc[u].z[ZERO ? i : 0][r], a.s_dt) : 0.0f;
                }
            const uint4* xs = &sm.x[slot][0][0][0] + g * 16 + wg * 8 + t;
            float c[MT][4], sx[ZERO ? MT : 1][4];
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                const int piece = 4 * (half ^ (g & 1));
                uint32_t f[2][4];
                frag<XT>(words[half * 2], f[0]);
                frag<XT>(words[half * 2 + 1], f[1]);
#pragma unroll
                for (int e = 0; e < TERMS; ++e) {
                    uint4 b[MT];                           // the rows' products side by side: MT sums that do not wait
#pragma unroll
                    for (int i = 0; i < MT; ++i) b[i] = xs[e * kRowsM * 16 + i * 128 + piece];
                    const bool first = e == 0 && (G32 || half == 0);
#pragma unroll
                    for (int i = 0; i < MT; ++i) {
                        if (first) mma_x0<XT>(c[i], f[0], b[i].x, b[i].y);
                        else mma_x<XT>(c[i], f[0], b[i].x, b[i].y);
                    }
#pragma unroll
                    for (int i = 0; i < MT; ++i) mma_x<XT>(c[i], f[1], b[i].z, b[i].w);
                    if constexpr (ZERO) {
#pragma unroll
                        for (int i = 0; i < MT; ++i) {
                            if (first) mma_x0<XT>(sx[i], ones, b[i].x, b[i].y);
                            else mma_x<XT>(sx[i], ones, b[i].x, b[i].y);
                        }
#pragma unroll
                        for (int i = 0; i < MT; ++i) mma_x<XT>(sx[i], ones, b[i].z, b[i].w);
                    }
                }
                if (!G32 && half == 0) continue;
                const int sh = G32 ? half : 0;
#pragma unroll
                for (int i = 0; i < MT; ++i)
#pragma unroll
                    for (int q = 0; q < 4; ++q) {
                        if constexpr (ZERO) c[i][q] = fmaf(zv[sh][q >> 1], sx[i][q], c[i][q]);
                        acc[i][q] = fmaf(sv[sh][q >> 1], c[i][q], acc[i][q]);
                    }
            }
            fetch(kp + AHEAD, u);
            slot = slot == STAGES - 1 ? 0 : slot + 1;
        }
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    // x is no longer read, in any CTA of the cluster: its memory takes the sums. CTA p finishes the rows p, p + split, ...;
    // every warp group of every CTA has a place there of its own, [source][row / split][output].
    if (split > 1) cluster_sync();
    else __syncthreads();
    const int rows = ROWS / split, source = part * 2 + wg, col = (warp & 7) * 16 + g;
    const uint32_t mine = smem_u32(&sm.part[0]);
#pragma unroll
    for (int i = 0; i < MT; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int r = 8 * i + 2 * t + (q & 1);
            const uint32_t at = mine + (uint32_t) ((source * rows + r / split) * kRowsN + col + 8 * (q >> 1)) * 4;
            asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(mapa_shared(at, (uint32_t) (r % split))), "f"(acc[i][q]) : "memory");
        }
    if (split > 1) cluster_sync();
    else __syncthreads();
    for (int i = threadIdx.x; i < rows * kRowsN; i += kRowsThreads) {
        const int c = i % kRowsN, r = i / kRowsN, n = block * kRowsN + c;
        const long long m = m0 + r * split + part;
        if (n >= a.N || m >= a.M) continue;
        float y = 0.0f;
        for (int p = 0; p < 2 * split; ++p) y += sm.part[(p * rows + r) * kRowsN + c];
        if (!is_finite(y)) y = int4_exact(a, m, n);
        if (a.bias) y += a.bias[n];
        st_dt(a.out, (size_t) m * a.N + n, y, a.out_dt);
    }
}

#include "int4tc.cuh"

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

template <typename... A>
cudaError_t in_clusters(void (*kernel)(A..., int), int blocks, long long chunks, int split, int threads, size_t smem,
                        cudaStream_t st, const A&... a) {
    cudaLaunchConfig_t c{};
    c.gridDim = dim3((unsigned) (blocks * split), (unsigned) chunks);
    c.blockDim = dim3((unsigned) threads);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = (unsigned) split;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    c.attrs = at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, a..., split);
}

template <int DT, bool ZERO, bool G32, int MT>
cudaError_t rows_mt(const Int4Args& a, int n_sm, cudaStream_t st) {
    constexpr int TERMS = DT == F32 ? 3 : 1;
    static std::atomic<uint64_t> ready{0};
    const cudaError_t e = allow_smem(ready, int4_rows<DT, ZERO, G32, MT>, sizeof(RowsSmem<TERMS>));
    if (e != cudaSuccess) return e;
    const int blocks = (a.N + kRowsN - 1) / kRowsN, KP = (a.K + 127) / 128;
    const long long chunks = (a.M + 8 * MT - 1) / (8 * MT);
    // as many CTAs as there are SMs, or half again as many; a part of the inputs has at least two stages
    int split = 1;
    while (split < 8 && blocks * chunks * split * 2 <= n_sm + n_sm / 2 && KP / (split * 2) >= 2) split *= 2;
    return in_clusters<Int4Args>(int4_rows<DT, ZERO, G32, MT>, blocks, chunks, split, kRowsThreads, sizeof(RowsSmem<TERMS>), st, a);
}

template <int DT, bool ZERO, int US, int NC>
cudaError_t tc_nc(const Int4Args& a, int n_sm, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    constexpr size_t bytes = sizeof(TcSmem) + 1024;
    const cudaError_t e = allow_smem(ready, int4_tc<DT, ZERO, US, NC>, bytes);
    if (e != cudaSuccess) return e;
    const int blocks = (a.N + 127) / 128, KT = (a.K + 63) / 64;
    const long long chunks = (a.M + 32 * NC - 1) / (32 * NC);
    // a CTA per SM, as far as a part of the inputs has at least four stages
    int split = 1;
    while (split < 8 && blocks * chunks * split * 2 <= n_sm && KT / (split * 2) >= 4) split *= 2;
    CUtensorMap tx{};
    if (a.x_vec) {                                         // x as [M, K]: boxes of 64 inputs x ROWS rows, 128-byte swizzle
        auto enc = tensor_map_encoder();
        if (!enc) return cudaErrorNotSupported;
        const cuuint64_t dims[2] = {(cuuint64_t) a.K, (cuuint64_t) a.M}, strides[1] = {(cuuint64_t) a.K * 2};
        const cuuint32_t box[2] = {64, 32 * NC}, steps[2] = {1, 1};
        if (enc(&tx, DT == F16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, const_cast<void*>(a.x), dims, strides,
                box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            return cudaErrorInvalidValue;
    }
    return in_clusters<Int4Args, CUtensorMap>(int4_tc<DT, ZERO, US, NC>, blocks, chunks, split, kTcThreads, bytes, st, a, tx);
}

template <int DT, int SDT, bool ZERO, bool G32>
cudaError_t few_s(const Int4Args& a, int n_sm, cudaStream_t st) {
    const int strips = (a.N + 15) / 16;
    // Two strips to a CTA share what is done for x, where there are enough of them for every SM: float32, whose x is three
    // terms, 22.7 us against 29.9 for 12288 outputs of 4096 inputs; 16-bit types 11.3 against 11.8 (28672: 23.0 and 23.6; 9600
    // 11.0 and 10.5). With zero points or groups of 32 a 16-bit type has not the registers for it: 16.5 against 13.9, and 25.3
    // against 17.7 with both.
    if constexpr (DT == F32 || (!ZERO && !G32)) {
        if (strips >= 4 * n_sm) {
            int4_few<DT, SDT, ZERO, G32, 2><<<(unsigned) ((strips + 1) / 2), kI4Warps * 32, 0, st>>>(a);
            return cudaGetLastError();
        }
    }
    int4_few<DT, SDT, ZERO, G32, 1><<<(unsigned) strips, kI4Warps * 32, 0, st>>>(a);
    return cudaGetLastError();
}

template <int DT, bool ZERO, bool G32>
cudaError_t int4_dt(const Int4Args& a, int n_sm, cudaStream_t st) {
    if (a.M <= 8) {
        switch (a.s_dt) {
            case F16: return few_s<DT, F16, ZERO, G32>(a, n_sm, st);
            case BF16: return few_s<DT, BF16, ZERO, G32>(a, n_sm, st);
            default: return few_s<DT, F32, ZERO, G32>(a, n_sm, st);
        }
    }
    // Up to 16 rows of a 16-bit type mma.sync is the quicker, its stages being shorter. 16 rows in bf16, groups of 128, against
    // tcgen05, us: 4096 inputs to 4096 outputs 9.0 and 11.4, to 12288 26.9 and 25.7, to 28672 45.5 and 49.7; 14336 to 4096 22.1
    // and 23.9; with groups of 32 9.7 and 15.2, 28.4 and 45.4, 49.3 and 87.5, 23.6 and 39.4. At 17 rows this kernel's next size,
    // 32 rows, was 11.8 against 11.7 and 34.6 against 26.6 (12288).
    if (a.M <= 16) return rows_mt<DT, ZERO, G32, 2>(a, n_sm, st);
    if constexpr (DT == F32) {
        if (a.M <= 32) return rows_mt<DT, ZERO, G32, 4>(a, n_sm, st);
        if (a.M <= 48) return rows_mt<DT, ZERO, G32, 6>(a, n_sm, st);
        return rows_mt<DT, ZERO, G32, 8>(a, n_sm, st);
    } else {
        // 4, 2 or 1 units in a stage
        if constexpr (G32) return a.M <= 32 ? tc_nc<DT, ZERO, 2, 1>(a, n_sm, st) : tc_nc<DT, ZERO, 2, 2>(a, n_sm, st);
        else if (a.group_shift == 6) return a.M <= 32 ? tc_nc<DT, ZERO, 1, 1>(a, n_sm, st) : tc_nc<DT, ZERO, 1, 2>(a, n_sm, st);
        else return a.M <= 32 ? tc_nc<DT, ZERO, 0, 1>(a, n_sm, st) : tc_nc<DT, ZERO, 0, 2>(a, n_sm, st);
    }
}

template <int DT>
cudaError_t int4_type(const Int4Args& a, int n_sm, cudaStream_t st) {
    if (a.group_shift == 5) return a.zero ? int4_dt<DT, true, true>(a, n_sm, st) : int4_dt<DT, false, true>(a, n_sm, st);
    return a.zero ? int4_dt<DT, true, false>(a, n_sm, st) : int4_dt<DT, false, false>(a, n_sm, st);
}

cudaError_t launch_int4_linear(const Int4Args& a, int n_sm, cudaStream_t st) {
    switch (a.x_dt) {
        case F16: return int4_type<F16>(a, n_sm, st);
        case BF16: return int4_type<BF16>(a, n_sm, st);
        default: return int4_type<F32>(a, n_sm, st);
    }
}

cudaError_t launch_int4_pack(const uint8_t* codes, long long N, long long K, void* tiles, int n_sm, cudaStream_t st) {
    int4_pack<<<(unsigned) (n_sm * 8), 256, 0, st>>>(codes, N, K, static_cast<uint32_t*>(tiles));
    return cudaGetLastError();
}

}  // namespace h3
