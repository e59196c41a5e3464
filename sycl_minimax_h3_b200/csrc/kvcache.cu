// kvcache.cu - a key/value cache in 8 bits, with one scale for each 64-token page and head, for the text model's
// grouped heads: writing to it, causal attention over it, and eviction by the weight that tokens received.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <type_traits>

#include "attn_common.cuh"
#include "kvcache.cuh"
#include "kvcommon.cuh"

namespace h3 {
namespace {

// The codes of eight values x times sc in a block whose largest magnitude is top > 0: 127 x sc / top rounded to the nearest
// whole number, half way to even, as if the ratio were exact. ratio = 127 sc / top as a float is off by 2^-23 of itself at
// most, so x * ratio by less than 4e-5: where it lies within 1e-4 of half way between two codes, the ratio is taken
// again in 64 bits, which hold x sc 127 exactly (24 + 24 + 7 bits at most where x is a float and sc = 1, or x a code).
// Adding 1.5 2^23 rounds to a whole number in the low bits. odd: x may hold infinities (+-127) and NaN (0).
// The long way is a call of its own: inlined, its registers would halve the CTAs of an SM for one chunk in a few hundred.
__device__ __noinline__ uint2 codes8_long(float4 lo, float4 hi, double sc, double top) {
    const float x[8] = {lo.x, lo.y, lo.z, lo.w, hi.x, hi.y, hi.z, hi.w};
    uint32_t o[2] = {0, 0};
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        int q = 0;
        if (!finite(x[u])) q = x[u] > 0.0f ? 127 : x[u] < 0.0f ? -127 : 0;
        else q = (int) fmin(fmax(rint((double) x[u] * sc * 127.0 / top), -127.0), 127.0);
        o[u / 4] |= (uint32_t) (q & 255) << (8 * (u % 4));
    }
    return make_uint2(o[0], o[1]);
}
__device__ __forceinline__ uint2 codes8(const float (&x)[8], float ratio, double sc, double top, bool odd) {
    constexpr float kRound = 12582912.0f;
    int q[8];
    float far = 0.0f;
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const float n = fmaf(x[u], ratio, kRound);
        q[u] = __float_as_int(n);
        far = fmaxf(far, fabsf(fmaf(x[u], ratio, kRound - n)));
    }
    if (odd || far > 0.4999f)
        return codes8_long(make_float4(x[0], x[1], x[2], x[3]), make_float4(x[4], x[5], x[6], x[7]), sc, top);
    uint2 o;
    o.x = __byte_perm(__byte_perm(q[0], q[1], 0x0040), __byte_perm(q[2], q[3], 0x0040), 0x5410);
    o.y = __byte_perm(__byte_perm(q[4], q[5], 0x0040), __byte_perm(q[6], q[7], 0x0040), 0x5410);
    return o;
}

template <typename T>
__device__ __forceinline__ T block_max(T x, T* red) {     // over 256 threads; every thread gets the result
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const T y = __shfl_xor_sync(0xffffffffu, x, o);
        x = y > x ? y : x;
    }
    __syncthreads();                                       // red may still be read from the call before
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
    __syncthreads();
    x = red[0];
#pragma unroll
    for (int i = 1; i < 8; ++i) x = red[i] > x ? red[i] : x;
    return x;
}

// ---- writing ---------------------------------------------------------------------------------------------------------
// A block of 64 slots that is full becomes a page: a = max|x| over its 64 x D values of a head, scale = a / 127, codes as
// codes8. What does not fill a block stays in the tail in its own type, so a token is rounded once, when its block is
// full, and the cache does not depend on how the tokens were spread over calls. Infinities take the code +-127 and NaN 0;
// neither counts for a.
// One CTA per (sequence, head), block, and K or V. The CTA of the sequence's first block reads the old tail and, after
// that, writes the new one: the two share slots.
// A block's rows are read once, into registers (16 KB a CTA of 256 threads, four to an SM), since the maximum comes before
// the codes: a CTA's loads, maximum and conversions (product, rounding check, packing) follow one another. Three prompts of
// 700 to 4,133 tokens, 8 heads of 128 in fp16, 58 MB, are 25 us (2.3 TB/s; the bytes alone 9; float32 28 us): the schedulers
// issue 64 % of the time with 37 % of an SM's warps, and wait for the loads and the barriers for most of the rest. A step of
// 48 single tokens is 7 us (float32 5): three loads that follow from one another (start, length, page) in 768 CTAs of 256
// threads, 1.3 rounds of what is resident, of which 16 threads have a row to move.
constexpr int kAppThreads = 256;

template <int DT, int D>
__global__ void __launch_bounds__(kAppThreads, DT == F32 ? 3 : 4) kv_append(const __grid_constant__ KvArgs kv, const void* __restrict__ krows,
                                                         const void* __restrict__ vrows, long long T, long long stride,
                                                         const int* __restrict__ starts, int vec) {
    constexpr int C8 = D / 8;                              // 8-value chunks of a row
    constexpr int PER = 64 * C8 / kAppThreads;
    __shared__ float red[8];
    const int j = blockIdx.y, J = gridDim.y, which = blockIdx.z;
    const int b = (int) (blockIdx.x / kv.heads), h = (int) (blockIdx.x % kv.heads);
    const Seq s = load_seq(kv, starts, T, b);
    if (!s.ok || s.L < s.n) {
        if (threadIdx.x == 0) atomicOr(kv.err, kErrLen);
        return;
    }
    if (s.n == 0) return;
    const int L0 = s.L - s.n, first = L0 / kPage, full = s.L / kPage;
    const void* rows = which ? vrows : krows;
    void* tail = which ? kv.tv : kv.tk;
    const size_t tbase = ((size_t) b * kv.heads + h) * kPage;
    auto row = [&](int slot) { return (size_t) (s.s0 + (slot - L0)) * stride + (size_t) h * D; };
    for (int blk = first + j; blk < full; blk += J) {
        const int page = kv.table[(size_t) b * kv.width + blk];
        const bool ok = page_ok(kv, page);
        Raw8<DT> raw[PER];
        float top = 0.0f, odd = 0.0f;                      // odd: NaN once a value is infinite or NaN
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = threadIdx.x + i * kAppThreads, r = c / C8, d = c % C8 * 8, slot = blk * kPage + r;
            if (slot < L0) raw[i] = raw8<DT>(tail, (tbase + r) * D + d, true);
            else raw[i] = raw8<DT>(rows, row(slot) + d, vec);
        }
        if (!ok) {
            if (threadIdx.x == 0) atomicOr(kv.err, kErrPage);
            continue;
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            float x[8];
            floats8(raw[i], x);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                top = fmaxf(top, fabsf(x[u]));
                odd = fmaf(x[u], 0.0f, odd);
            }
        }
        const bool any_odd = __syncthreads_or(odd != 0.0f);
        if (any_odd) {
            top = 0.0f;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                float x[8];
                floats8(raw[i], x);
#pragma unroll
                for (int u = 0; u < 8; ++u)
                    if (finite(x[u])) top = fmaxf(top, fabsf(x[u]));
            }
        }
        top = block_max(top, red);
        const size_t pbase = (size_t) page * kv.heads + h;
        if (threadIdx.x == 0) (which ? kv.vs : kv.ks)[pbase] = __fdiv_rn(top, 127.0f);
        // a largest value below 2^-100 has no float 127 / a: every code goes the long way
        const bool small = top < 7.9e-31f;
        const float ratio = small ? 0.0f : __fdiv_rn(127.0f, top);
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = threadIdx.x + i * kAppThreads, r = c / C8, d = c % C8 * 8;
            uint2 o = make_uint2(0, 0);
            float x[8];
            floats8(raw[i], x);
            if (top > 0.0f) o = codes8(x, ratio, 1.0, (double) top, any_odd || small);
            *reinterpret_cast<uint2*>((which ? kv.v : kv.k) + (pbase * kPage + r) * D + d) = o;
        }
        if (kv.tw && which == 0 && threadIdx.x < kPage)
            kv.w[pbase * kPage + threadIdx.x] = blk * kPage + (int) threadIdx.x < L0 ? kv.tw[tbase + threadIdx.x] : 0.0f;
    }
    if (j != 0 || s.L == full * kPage) return;
    __syncthreads();                                       // the old tail has been read
    const int from = max(L0, full * kPage);
    for (int c = threadIdx.x; c < (s.L - from) * C8; c += kAppThreads) {
        const int slot = from + c / C8, d = c % C8 * 8;
        const Raw8<DT> x = raw8<DT>(rows, row(slot) + d, vec);
        uint4* to = reinterpret_cast<uint4*>(static_cast<char*>(tail) + ((tbase + slot % kPage) * D + d) * DtInfo<DT>::ES);
        to[0] = x.u[0];
        if constexpr (DT == F32) to[1] = x.u[1];
    }
    if (kv.tw && which == 0)
        for (int slot = from + threadIdx.x; slot < s.L; slot += kAppThreads) kv.tw[tbase + slot % kPage] = 0.0f;
}

// ---- attention -------------------------------------------------------------------------------------------------------
// The query rows of a kv head are its group's heads of every new token, row r = token * group + head, in tiles of 8 NB:
// the columns of m16n8k16 products whose 16 rows are keys (scores) or features (output), so that one tile of codes
// serves 8 or 16 queries and a step's few queries leave little of a product empty.
//   s_ji = (kc_j . q_i) * ks * log2(e)/sqrt(D)     p_ji = 2^(s_ji - m_i)     acc_i = acc_i 2^(m_old - m_i) + vs * sum_j vc_j p_ji
//
// Codes as fp16 operands: u = code + 128 in the low bits of 1024's mantissa, less 1152, is exact; one logic instruction
// places u (flipped top bit, mask and the bits of 1024 at once), one subtracts. For the scores of 16-bit rows the
// subtraction is saved: the bits 0x00 uu of a half are u 2^-24 exactly, and sum_d q_d (u_d - 128) starts from -128 sum q
// instead of 0. Its partial sums are some four times as large, 2^-21 of the score or less beside the 2^-11 of p's
// rounding; not so for P.V, whose p have one sign (sums of 128 p are 2^5 and more times the result), nor for float32.
// q is brought to fp16 times a power of two per row, so that the row's largest value lies in [2^13, 2^14): exact for
// fp16 and bf16 (what is more than 2^27 times smaller than the row's largest loses bits that a 32-bit sum would not
// hold either); float32 takes two terms, 22 bits. p is rounded to fp16 (at most 2^-11 of it, beside 2^-8 or 2^-11 of the
// output); for float32 it takes two terms too.
//
// Nothing is ordered inside a row's features: lane (g, t) of a warp reads 16-byte pieces of K (key g, features 16 t..),
// and the query's fragment uses the same order. For P.V it reads features D/8 g.. of four keys, and accumulators
// [i][..][e] of a lane are feature D/8 g + 2 i + e / 2 of query 2 t + e % 2.
//
// Four warps per CTA take the pages of a piece in turn, each with a ring of two 8 KB tiles of its own that bulk copies fill:
// no warp waits for another before the end. What bounds it, by lengths (bf16, 8 heads of 128, 4 queries each): 48 sequences
// of 2,048 tokens 41 us (4.9 TB/s of codes; the bytes alone 31; float32 44 us), of 200 to 8,191 94 us (4.6 TB/s; 66: pieces are
// whole pages and their ends leave SMs idle), one of 131,037 52 us (5.2 TB/s; 41; float32 57); one of 64 to 4,096 tokens 6 to 10
// us (77: 8.3), which are the loads that follow from one another, start and length, page id, codes and scale, tail, and the
// joining launch. 32 rows behind 16,384 tokens are 26 us (the bytes alone 5): each tile of 16 rows reads and unpacks the
// codes for itself.

__device__ __forceinline__ void mma16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    // volatile: in the order written, which keeps four sums in flight and the operands' registers few
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// an 8 x 8 matrix of halves, lane (g, t) holding row g's columns 2 t and 2 t + 1, transposed
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
__device__ __forceinline__ uint32_t half2_bits(__half2 h) { return *reinterpret_cast<const uint32_t*>(&h); }

// per bit: 0 where m and k are 0, 1 where only k is, x where only m is, ~x where both are
__device__ __forceinline__ uint32_t place(uint32_t x, uint32_t m, uint32_t k) {
    uint32_t y;
    asm("lop3.b32 %0, %1, %2, %3, 0x6a;" : "=r"(y) : "r"(x), "r"(m), "r"(k));
    return y;
}
// bytes 0 and 2 of x as two halves: their codes, or (SHORT) code + 128 in units of 2^-24
template <bool SHORT>
__device__ __forceinline__ uint32_t codes02(uint32_t x) {
    if constexpr (SHORT) return place(x, 0x00ff00ffu, 0x00800080u);
    const uint32_t u = place(x, 0x00ff00ffu, 0x64806480u);
    return half2_bits(__hsub2(*reinterpret_cast<const __half2*>(&u), __half2half2(__ushort_as_half(0x6480))));
}
constexpr float kCodeUnit = 16777216.0f;                   // 2^24
// keeps the compiler from loading shared memory ahead of this point, which would cost more registers than there are
__device__ __forceinline__ void load_fence() { asm volatile("" ::: "memory"); }

constexpr int kAttWarps = 4;

// Which piece the flat-th of a call is. A sequence has tiles x heads units of `length` pages each (its whole pages, and the
// tail as kTailPages more), cut into nz pieces; a piece has about as many pages as the sum over all units divided by
// `room`, but kChunk at least: so unequal sequences give nearly equal pieces, and a short one is one piece. Up to 32
// sequences are a warp's, a lane each, and every warp finds the piece for itself; more are the 128 threads' together.
constexpr int kTailPages = 2, kChunk = 6;
struct Piece {
    int b, tile, h, z, nz;             // b < 0: there are no more
    Seq s;
};
constexpr int kWhole = 0;              // no chunk: every unit is one piece
__device__ __forceinline__ int pieces_of_unit(int length, int chunk) {   // rounded
    return chunk == kWhole ? 1 : max(1, (2 * length + chunk) / (2 * chunk));
}
// (starts that run backwards can stand for any number of pages: the chunk stays where twice of it is an int)
__device__ __forceinline__ int chunk_pages(float all, int room) { return max(kChunk, (int) fminf(ceilf(all / (float) room), 1 << 28)); }
template <int ROWS>
__device__ __forceinline__ Piece find_piece(const AttendArgs& a, int flat, int group, int* scan) {
    const KvArgs& kv = a.kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto units_of = [&](int i, int& length) {
        length = 0;
        if (i >= kv.seqs) return 0;
        const Seq s = load_seq(kv, a.starts, a.T, i);
        if (!s.ok) {
            atomicOr(kv.err, kErrLen);
            return 0;
        }
        length = max(1, s.L / kPage + (s.L % kPage ? kTailPages : 0));
        return (s.n * group + ROWS - 1) / ROWS * kv.heads;
    };
    if (kv.seqs <= 32) {
        Seq s{0, 0, 0, false};
        int units = 0, length = 0, nz = 1;
        if (lane < kv.seqs) {
            s = load_seq(kv, a.starts, a.T, lane);
            length = max(1, s.L / kPage + (s.L % kPage ? kTailPages : 0));
            if (s.ok) units = (s.n * group + ROWS - 1) / ROWS * kv.heads;
            else atomicOr(kv.err, kErrLen);
        }
        if (a.plan.room > 0) {
            float all = (float) units * (float) length;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
            nz = pieces_of_unit(length, chunk_pages(all, a.plan.room));
        }
        int upto = units * nz;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const int from = upto - units * nz;
        const uint32_t here = __ballot_sync(0xffffffffu, flat >= from && flat < upto);
        Piece p{-1, 0, 0, 0, 1, s};
        if (here == 0) return p;
        const int i = __ffs((int) here) - 1, at = flat - __shfl_sync(0xffffffffu, from, i);
        p.nz = __shfl_sync(0xffffffffu, nz, i);
        if (a.plan.joined && at == 0 && (int) threadIdx.x == i)
            reinterpret_cast<int2*>(a.part + (size_t) a.plan.entries * (kv.dim + 2))[i] = make_int2(flat, nz);
        p.b = i;
        p.s.s0 = __shfl_sync(0xffffffffu, s.s0, i);
        p.s.n = __shfl_sync(0xffffffffu, s.n, i);
        p.s.L = __shfl_sync(0xffffffffu, s.L, i);
        p.s.ok = true;
        // the heads side by side: they lie side by side in a page, and are read at about the same time
        const int zt = quotient(at, kv.heads, a.head_shift);
        p.h = at - zt * kv.heads;
        p.tile = p.nz == 1 ? zt : zt / p.nz;
        p.z = zt - p.tile * p.nz;
        return p;
    }
    int length0 = 0, units0 = units_of((int) threadIdx.x, length0);      // the first 128 sequences' are kept
    int chunk = kWhole;
    if (a.plan.room > 0) {
        float all = 0.0f;                                  // pages in all: a float is exact enough to divide them
        for (int b0 = 0; b0 < kv.seqs; b0 += kAttWarps * 32) {
            int length = length0;
            const int units = b0 == 0 ? units0 : units_of(b0 + (int) threadIdx.x, length);
            all += (float) units * (float) length;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        if (lane == 0) scan[warp] = __float_as_int(all);
        __syncthreads();
        all = __int_as_float(scan[0]) + __int_as_float(scan[1]) + __int_as_float(scan[2]) + __int_as_float(scan[3]);
        chunk = chunk_pages(all, a.plan.room);
    }
    int* found = scan + 2 * kAttWarps;
    if (threadIdx.x == 0) found[0] = -1;
    int before = 0;
    for (int b0 = 0; b0 < kv.seqs; b0 += kAttWarps * 32) {
        int length = length0;
        const int units = b0 == 0 ? units0 : units_of(b0 + (int) threadIdx.x, length);
        const int nz = pieces_of_unit(length, chunk), n = units * nz;
        int upto = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        if (b0 > 0) __syncthreads();                       // the sums of the sequences before have been read
        if (lane == 31) scan[kAttWarps + warp] = upto;
        __syncthreads();
        int from = before + upto - n, sum = 0;
#pragma unroll
        for (int w = 0; w < kAttWarps; ++w) {
            if (w < warp) from += scan[kAttWarps + w];
            sum += scan[kAttWarps + w];
        }
        if (flat >= from && flat < from + n) {
            found[0] = b0 + (int) threadIdx.x;
            const int i = flat - from, h = i % kv.heads, zt = i / kv.heads;
            found[1] = zt / nz;
            found[2] = zt % nz;
            found[3] = nz;
            found[4] = h;
            if (a.plan.joined && flat == from)
                reinterpret_cast<int2*>(a.part + (size_t) a.plan.entries * (kv.dim + 2))[found[0]] = make_int2(from, nz);
        }
        before += sum;
    }
    __syncthreads();
    Piece p{found[0], found[1], found[4], found[2], found[3], {0, 0, 0, false}};
    if (p.b >= 0) p.s = load_seq(kv, a.starts, a.T, p.b);
    return p;
}
// p is 2^(s - m) with m the largest score less this, so at most 2^14: fp16 then keeps its 11 bits of every p down to
// 2^-28 of the row's largest (2^-14 without it), and 2^-39 of the largest is what it drops
constexpr float kPTop = 14.0f;

// The query rows of a tile as B fragments in shared memory, which a CTA's warps share: step ks of rows 8 nb + g is two words
// of lane (g, t), hi[nb][ks][lane]; TWO: and the second terms. rs: what a row's scores are multiplied by, with a page's scale; s0:
// where its sums start.
template <int D, int NB, bool TWO>
struct QFrag {
    uint2 hi[NB][D / 16][32];
    uint2 lo[TWO ? NB : 1][TWO ? D / 16 : 1][32];
    float rs[8 * NB], s0[8 * NB];
};
// D / 8 threads to a row, 8 features to a thread; T threads. The loads apart from what makes fragments of them, so that
// others can be made while these are under way. qoff: the rows' element offsets, or -1 for a row of zeros.
template <int DT, int D, int NB, int T>
struct QRows {
    static constexpr int PER = (8 * NB * D / 8 + T - 1) / T;
    Raw8<DT> x[PER];
};
template <int DT, int D, int NB, int T>
__device__ __forceinline__ void load_q(QRows<DT, D, NB, T>& r, const void* q, const long long* qoff, bool vec) {
#pragma unroll
    for (int j = 0; j < QRows<DT, D, NB, T>::PER; ++j) {
        const int i = (int) threadIdx.x % T + j * T, row = i / (D / 8);
        const long long at = row < 8 * NB ? qoff[row] : -1;
        if (at >= 0) r.x[j] = raw8<DT>(q, (size_t) at + i % (D / 8) * 8, vec);
        else
#pragma unroll
            for (int u = 0; u < (DT == F32 ? 2 : 1); ++u) r.x[j].u[u] = make_uint4(0, 0, 0, 0);
    }
}
template <int DT, int D, int NB, bool TWO, int T>
__device__ __forceinline__ void make_q(QFrag<D, NB, TWO>& f, const QRows<DT, D, NB, T>& r, float scale) {
#pragma unroll
    for (int j = 0; j < QRows<DT, D, NB, T>::PER; ++j) {
        const int i = (int) threadIdx.x % T + j * T, row = i / (D / 8), d = i % (D / 8) * 8;
        float x[8], top = 0.0f;
        floats8(r.x[j], x);
#pragma unroll
        for (int u = 0; u < 8; ++u)
            if (finite(x[u])) top = fmaxf(top, fabsf(x[u]));
#pragma unroll
        for (int o = 1; o < D / 8; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        // 2^e in two factors: each is a normal float, whatever the row's size (e from -162 to 114)
        int e = 0;
        if (top > 0.0f) e = ilogbf(top) - 13;
        const int e1 = e / 2, e2 = e - e1;
        const float m1 = __int_as_float((127 - e1) << 23), m2 = __int_as_float((127 - e2) << 23);
        float sum = 0.0f;
        // features d .. d + 7 are two steps (four each) of lane (row % 8, d % 64 / 16); 0 and 2, 1 and 3 of four, as codes02
        const int ks = d / 64 * 4 + d % 16 / 4, lane = row % 8 * 4 + d % 64 / 16;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            uint32_t hi[2], lo[2];
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const float y0 = x[k * 4 + u] * m1 * m2, y1 = x[k * 4 + u + 2] * m1 * m2;
                const __half2 h = __floats2half2_rn(y0, y1);
                const float2 back = __half22float2(h);
                hi[u] = half2_bits(h);
                if constexpr (TWO) lo[u] = half2_bits(__floats2half2_rn(finite(y0) ? y0 - back.x : 0.0f, finite(y1) ? y1 - back.y : 0.0f));
                else sum += back.x + back.y;
            }
            if (row < 8 * NB) {
                f.hi[row / 8][ks + k][lane] = make_uint2(hi[0], hi[1]);
                if constexpr (TWO) f.lo[row / 8][ks + k][lane] = make_uint2(lo[0], lo[1]);
            }
        }
#pragma unroll
        for (int o = 1; o < D / 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (d == 0 && row < 8 * NB) {
            f.rs[row] = scale * (TWO ? 1.0f : kCodeUnit) * __int_as_float((127 + e1) << 23) * __int_as_float((127 + e2) << 23);
            f.s0[row] = TWO ? 0.0f : sum * (-128.0f / kCodeUnit);
        }
    }
}

// s[mt][nb] = the scores of keys 16 mt + g (elements 0, 1) and + 8 (2, 3) with queries 8 nb + 2 t + {0, 1}, unscaled
template <int D, int NB, bool TWO>
__device__ __forceinline__ void page_scores(const QFrag<D, NB, TWO>& f, const int8_t* kp, float (&s)[4][NB][4]) {
    const int g = (threadIdx.x & 31) >> 2, t = threadIdx.x & 3;
#pragma unroll
    for (int mt = 0; mt < 4; ++mt)
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int i = 0; i < 4; ++i) s[mt][nb][i] = f.s0[8 * nb + 2 * t + (i & 1)];
#pragma unroll
    for (int c = 0; c < D / 64; ++c) {
        load_fence();
        uint32_t w[4][2][4];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                const uint4 u = *reinterpret_cast<const uint4*>(kp + (mt * 16 + r * 8 + g) * D + c * 64 + t * 16);
                w[mt][r][0] = u.x; w[mt][r][1] = u.y; w[mt][r][2] = u.z; w[mt][r][3] = u.w;
            }
        // the key tiles' products side by side: sums that do not wait for one another
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int ks = c * 4 + i, lane = threadIdx.x & 31;
            uint2 q[NB], q2[NB];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                q[nb] = f.hi[nb][ks][lane];
                if constexpr (TWO) q2[nb] = f.lo[nb][ks][lane];
            }
#pragma unroll
            for (int mt = 0; mt < 4; ++mt) {
                const uint32_t a0 = codes02<!TWO>(w[mt][0][i]), a2 = codes02<!TWO>(w[mt][0][i] >> 8);
                const uint32_t a1 = codes02<!TWO>(w[mt][1][i]), a3 = codes02<!TWO>(w[mt][1][i] >> 8);
#pragma unroll
                for (int nb = 0; nb < NB; ++nb) {
                    mma16816(s[mt][nb], a0, a1, a2, a3, q[nb].x, q[nb].y);
                    if constexpr (TWO) mma16816(s[mt][nb], a0, a1, a2, a3, q2[nb].x, q2[nb].y);
                }
            }
        }
    }
}

// A page's codes come into shared memory by bulk copies, K and V of a page in turn through a ring of two 64 x D tiles per
// warp: one or two are in flight while one is read.
constexpr int kSlots = 2;

// four neighbouring outputs, with one store where vec
template <int DT>
__device__ __forceinline__ void st4(void* p, size_t i, float x, float y, float z, float w, bool vec) {
    if (!vec) {
        st1<DT>(p, i, x);
        st1<DT>(p, i + 1, y);
        st1<DT>(p, i + 2, z);
        st1<DT>(p, i + 3, w);
    } else if constexpr (DT == F32) {
        *reinterpret_cast<float4*>(static_cast<float*>(p) + i) = make_float4(x, y, z, w);
    } else if constexpr (DT == F16) {
        *reinterpret_cast<uint2*>(static_cast<__half*>(p) + i) = make_uint2(pack_half2(x, y), pack_half2(z, w));
    } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(x, y), b = __floats2bfloat162_rn(z, w);
        *reinterpret_cast<uint2*>(static_cast<__nv_bfloat16*>(p) + i) =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
    }
}

template <int D, int NB, bool TWO>
struct AttSmem {
    union {
        int8_t ring[kAttWarps][kSlots][kPage * D];
        float acc[kAttWarps + 1][8 * NB][D];               // the warps' accumulators, then the tail's
        unsigned char tail[2][(kPage - 1) * D * 4];        // the tail's keys and values
    };
    QFrag<D, NB, TWO> f;
    float q[8 * NB][D];
    float sc[kPage][8 * NB];                               // the tail's scores, then its p: [key][row]
    float m[kAttWarps + 1][8 * NB], l[kAttWarps + 1][8 * NB];
    int pos[8 * NB];
    int row[8 * NB];                                       // token * Hq + head, or -1
    long long qoff[8 * NB];                                // the query row's first element, or -1
    uint64_t full[kAttWarps][kSlots];
    uint64_t tail_full;
    int scan[3 * kAttWarps + 4];
    // what the epilogue needs again
    int L, b, h, nrow, nu, tail_here;
};

// The codes leave L2 first: a step reads them once, and what every CTA waits for at its start (lengths, tables, scales,
// queries) should not make room for them.
__device__ __forceinline__ uint64_t leave_first() {
    uint64_t p;
    asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(p));
    return p;
}
__device__ __forceinline__ void bulk_load(void* dst, const void* src, uint32_t bytes, uint64_t* bar, uint64_t policy) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1], %2, [%3], %4;" ::"r"(smem_u32(dst)),
                 "l"(__cvta_generic_to_global(src)), "r"(bytes), "r"(smem_u32(bar)), "l"(policy)
                 : "memory");
}

// Scores of the tail's keys in plain 32-bit arithmetic, sc[key][row] in log2 units: qf [rows][D] as floats, kt the tail's
// rows in dt (shared memory). 128 threads, each a key and half of the rows; a thread starts at the 16-byte piece that its
// key's number names, so that neighbouring keys, whose rows start in the same banks, read different ones.
// No branch per row: with one, every load was waited for, and 13 keys of 4 rows took 1.8 us, now 0.7.
template <int DT, int D, int ROWS>
__device__ __forceinline__ void tail_scores(const float (*qf)[D], const unsigned char* kt, int nrow, int nkey, float scale,
                                            float (*sc)[ROWS]) {
    constexpr int E = 16 / DtInfo<DT>::ES, N = D / E;      // elements of a piece, pieces of a row
    const int key = threadIdx.x & 63, half = threadIdx.x >> 6, per = (nrow + 1) / 2;
    const int r0 = half * per, r1 = min(nrow, r0 + per);
    if (key >= nkey) return;
    // rows past the last are computed from what lies there, and not stored
    auto rows = [&](auto count) {
        constexpr int R = decltype(count)::value;
        float acc[R];
#pragma unroll
        for (int r = 0; r < R; ++r) acc[r] = 0.0f;
#pragma unroll 4
        for (int i = 0; i < N; ++i) {
            const int d = (i + key) % N * E;
            float x[E];
            cvt16<DT>(*reinterpret_cast<const uint4*>(kt + (key * D + d) * DtInfo<DT>::ES), x);
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int u = 0; u < E; u += 4) {
                    const float4 y = *reinterpret_cast<const float4*>(&qf[r0 + r][d + u]);
                    acc[r] = fmaf(y.x, x[u], acc[r]);
                    acc[r] = fmaf(y.y, x[u + 1], acc[r]);
                    acc[r] = fmaf(y.z, x[u + 2], acc[r]);
                    acc[r] = fmaf(y.w, x[u + 3], acc[r]);
                }
        }
#pragma unroll
        for (int r = 0; r < R; ++r)
            if (r0 + r < r1) sc[key][r0 + r] = acc[r] * scale;
    };
    if (per <= 2) rows(std::integral_constant<int, 2>{});
    else rows(std::integral_constant<int, ROWS / 2>{});
}

// The tail of the piece at hand as one more partial result, sm.acc[kAttWarps]: on CUDA cores, in 32 bits, since it is in
// its own type and has at most 63 keys. A function of its own, whose registers the loop over pages need not make room for.
template <int DT, int D, int NB>
__device__ __noinline__ void attend_tail(const AttendArgs& a) {
    constexpr int ROWS = 8 * NB, TR = ROWS * D / (kAttWarps * 32);   // the rows in a thread, of one feature
    extern __shared__ __align__(128) unsigned char smem_raw[];
    AttSmem<D, NB, DT == F32>& sm = *reinterpret_cast<AttSmem<D, NB, DT == F32>*>(smem_raw);
    const KvArgs& kv = a.kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, L = sm.L, nrow = sm.nrow, b = sm.b, h = sm.h;
    float ot[TR];
    const int full = L / kPage, nkey = L - full * kPage;
    __syncthreads();                               // the ring has been read
    if (threadIdx.x == 0) {
        const size_t tb = ((size_t) b * kv.heads + h) * kPage * D * DtInfo<DT>::ES;
        const uint32_t bytes = (uint32_t) (nkey * D * DtInfo<DT>::ES);
        mbar_expect_tx(&sm.tail_full, 2 * bytes);
        bulk_load(sm.tail[0], static_cast<const char*>(kv.tk) + tb, bytes, &sm.tail_full, leave_first());
        bulk_load(sm.tail[1], static_cast<const char*>(kv.tv) + tb, bytes, &sm.tail_full, leave_first());
    }
    for (int i = threadIdx.x; i < nrow * D; i += kAttWarps * 32)
        sm.q[i / D][i % D] = ld1<DT>(a.q, (size_t) sm.qoff[i / D] + i % D);
    if (!mbar_wait(&sm.tail_full, 0, a.wait_ns, nullptr)) atomicOr(a.wait_err, kErrCache);
    __syncthreads();
    tail_scores<DT, D, ROWS>(sm.q, sm.tail[0], nrow, nkey, a.scale_log2, sm.sc);
    __syncthreads();
    for (int r = warp; r < nrow; r += kAttWarps) {
        const int see = min(nkey, sm.pos[r] + 1 - full * kPage);
        const float x0 = lane < see ? sm.sc[lane][r] : -INFINITY, x1 = lane + 32 < see ? sm.sc[lane + 32][r] : -INFINITY;
        float mx = fmaxf(x0, x1);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        const float mu = mx == -INFINITY ? 0.0f : mx;
        const float e0 = ex2(x0 - mu), e1 = ex2(x1 - mu);
        float sum = e0 + e1;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        sm.sc[lane][r] = e0;
        sm.sc[lane + 32][r] = e1;
        if (lane == 0) { sm.m[kAttWarps][r] = mx; sm.l[kAttWarps][r] = sum; }
    }
    __syncthreads();
    // a thread has one feature and TR rows
    const int d = threadIdx.x % D, rb = threadIdx.x / D * TR;
#pragma unroll
    for (int r = 0; r < TR; ++r) ot[r] = 0.0f;
    float odd = 0.0f;                              // NaN once a value is infinite or NaN
#pragma unroll
    for (int r = 0; r < TR; r += 4) {
        if (rb + r >= nrow) break;
#pragma unroll 8
        for (int key = 0; key < nkey; ++key) {
            const float x = ld1<DT>(sm.tail[1], (size_t) key * D + d);
            const float4 e = *reinterpret_cast<const float4*>(&sm.sc[key][rb + r]);
            ot[r] = fmaf(e.x, x, ot[r]);
            ot[r + 1] = fmaf(e.y, x, ot[r + 1]);
            ot[r + 2] = fmaf(e.z, x, ot[r + 2]);
            ot[r + 3] = fmaf(e.w, x, ot[r + 3]);
            odd = fmaf(x, 0.0f, odd);
        }
    }
    if (odd != 0.0f) {                           // again, without what a row does not see, and 0 times infinity an infinity
#pragma unroll
        for (int r = 0; r < TR; ++r) {
            if (rb + r >= nrow) break;
            const int see = min(nkey, sm.pos[rb + r] + 1 - full * kPage);
            ot[r] = 0.0f;
#pragma unroll 4
            for (int key = 0; key < see; ++key) ot[r] = add_weighted(sm.sc[key][rb + r], ld1<DT>(sm.tail[1], (size_t) key * D + d), ot[r]);
        }
    }
    __syncthreads();                                       // the tail has been read, its memory becomes accumulators
#pragma unroll
    for (int r = 0; r < TR; ++r) sm.acc[kAttWarps][threadIdx.x / D * TR + r][threadIdx.x % D] = ot[r];
}

template <int DT, int D, int NB>
__global__ void __launch_bounds__(kAttWarps * 32, NB == 1 ? 3 : 2) attend(const __grid_constant__ AttendArgs a) {
    constexpr bool TWO = DT == F32;
    constexpr int DG = D / 8, ROWS = 8 * NB;
    constexpr uint32_t TILE = kPage * D;
    extern __shared__ __align__(128) unsigned char smem_raw[];
    AttSmem<D, NB, DT == F32>& sm = *reinterpret_cast<AttSmem<D, NB, DT == F32>*>(smem_raw);
    const KvArgs& kv = a.kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = quotient(a.Hq, kv.heads, a.head_shift);
    let_next_launch();
    if (threadIdx.x == 0) {
        for (int w = 0; w < kAttWarps; ++w)
            for (int i = 0; i < kSlots; ++i) mbar_init(&sm.full[w][i], 1);
        mbar_init(&sm.tail_full, 1);
        fence_barrier_init();
    }
    uint32_t used = 0, issued = 0;                         // tiles of this warp read and asked for
    const int flat = (int) blockIdx.x;                     // the grid has room for every piece there can be
    const Piece pcs = find_piece<ROWS>(a, flat, group, sm.scan);
    if (pcs.b < 0) return;
    {
        const int b = pcs.b, nz = pcs.nz, z = pcs.z, h = pcs.h, tile = pcs.tile;
        const Seq s = pcs.s;
        const int R = s.n * group;
        const int r0 = tile * ROWS, nrow = min(R - r0, ROWS);
        const int last_pos = s.L - s.n + quotient(r0 + nrow - 1, group, a.group_shift);
        const Pieces pc = pieces(s.L, last_pos, nz);
        if (z >= max(pc.nu, 1)) return;
        __syncthreads();                                   // the barriers are made
        if (threadIdx.x == 0) {
            sm.L = s.L;
            sm.b = b;
            sm.h = h;
            sm.nrow = nrow;
            sm.nu = pc.nu;
            sm.tail_here = z == pc.tail_at;
        }
        if (threadIdx.x < ROWS) {
            const int r = threadIdx.x;
            const bool in = r < nrow;
            const int tok = quotient(r0 + r, group, a.group_shift), hq = h * group + r0 + r - tok * group;
            sm.pos[r] = in ? s.L - s.n + tok : -1;
            sm.row[r] = in ? (s.s0 + tok) * a.Hq + hq : -1;
            sm.qoff[r] = in ? (long long) (s.s0 + tok) * a.qs + hq * D : -1;
        }
        __syncthreads();
        float acc[DG / 2][NB][4], m[NB][2], l[NB][2];
        const int p0 = z * pc.cz, p1 = min(pc.np, p0 + pc.cz);
        // up to 32 pages of this warp at a time, from page `sub` on: lane i keeps the i-th one's id and scales. Their first
        // tiles are asked for at once.
        int sub = p0, id = -1;
        float ks = 0.0f, vs = 0.0f;
        uint32_t ask = 0, todo = 0;
        bool ask_v = false;
        auto next = [&]() {                                // the next tile into the slot that was freed last
            if (ask == 0) return;
            const int i = __ffs((int) ask) - 1, pid = __shfl_sync(0xffffffffu, id, i), slot = (int) (issued % kSlots);
            if (lane == 0) {
                mbar_expect_tx(&sm.full[warp][slot], TILE);
                bulk_load(sm.ring[warp][slot], (ask_v ? kv.v : kv.k) + ((size_t) pid * kv.heads + h) * TILE, TILE, &sm.full[warp][slot], leave_first());
            }
            ++issued;
            if (ask_v) ask &= ask - 1;
            ask_v = !ask_v;
        };
        auto begin = [&]() {
            const int mine = sub + warp + kAttWarps * lane;
            id = -1;
            if (mine < p1) {
                id = kv.table[(size_t) b * kv.width + mine];
                if (!page_ok(kv, id)) {
                    atomicOr(kv.err, kErrPage);
                    id = -1;
                }
            }
            ask = todo = __ballot_sync(0xffffffffu, id >= 0);
#pragma unroll
            for (int i = 0; i < kSlots; ++i) next();
            if (id >= 0) {
                ks = kv.ks[(size_t) id * kv.heads + h];
                vs = kv.vs[(size_t) id * kv.heads + h];
            }
        };
        if (p0 < p1) {
            QRows<DT, D, NB, kAttWarps * 32> rows;
            load_q(rows, a.q, sm.qoff, a.q_vec);
            begin();
            make_q(sm.f, rows, a.scale_log2);
        }
        __syncthreads();
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            m[nb][0] = m[nb][1] = -INFINITY;
            l[nb][0] = l[nb][1] = 0.0f;
#pragma unroll
            for (int i = 0; i < DG / 2; ++i)
#pragma unroll
                for (int u = 0; u < 4; ++u) acc[i][nb][u] = 0.0f;
        }
        if (p0 < p1) {
            int pos[NB][2];
            float rs[NB][2];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    pos[nb][c] = sm.pos[8 * nb + 2 * t + c];
                    rs[nb][c] = sm.f.rs[8 * nb + 2 * t + c];
                }
            const int first_pos = sm.pos[0];
            while (true) {
                auto arrived = [&]() {
                    if (warp_wait(&sm.full[warp][used % kSlots], (used / kSlots) & 1, a.wait_ns, nullptr)) return true;
                    if (lane == 0) atomicOr(a.wait_err, kErrCache);
                    // give up: the copies in flight land before the memory is used for anything else
                    for (uint32_t u = used; u < issued; ++u)
                        warp_wait(&sm.full[warp][u % kSlots], (u / kSlots) & 1, a.wait_ns, nullptr);
                    return false;
                };
                while (todo) {
                    const int i = __ffs((int) todo) - 1, p = sub + warp + kAttWarps * i;
                    todo &= todo - 1;
                    const float kscale = __shfl_sync(0xffffffffu, ks, i), vscale = __shfl_sync(0xffffffffu, vs, i);
                    if (!arrived()) { used = issued; break; }
                    float sc[4][NB][4];
                    page_scores<D, NB, TWO>(sm.f, sm.ring[warp][used % kSlots], sc);
                    __syncwarp();
                    ++used;
                    next();
                    const bool mask = nrow < ROWS || p * kPage + kPage - 1 > first_pos;
                    float al[NB][2];
                    uint32_t ph[4][NB][2], pl[TWO ? 4 : 1][NB][2];
#pragma unroll
                    for (int nb = 0; nb < NB; ++nb) {
                        float mu[2];
#pragma unroll
                        for (int c = 0; c < 2; ++c) {
                            const float fs = kscale * rs[nb][c];
                            float mx = -INFINITY;
#pragma unroll
                            for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                                for (int r = 0; r < 2; ++r) {
                                    float x = sc[mt][nb][2 * r + c] * fs;
                                    if (mask && p * kPage + mt * 16 + r * 8 + g > pos[nb][c]) x = -INFINITY;
                                    sc[mt][nb][2 * r + c] = x;
                                    mx = fmaxf(mx, x);
                                }
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                            const float mn = fmaxf(m[nb][c], mx - kPTop);
                            mu[c] = mn == -INFINITY ? 0.0f : mn;   // a query that sees nothing yet: every p is 2^-inf = 0
                            al[nb][c] = ex2(m[nb][c] - mu[c]);
                            m[nb][c] = mn;
                            l[nb][c] *= al[nb][c];
                        }
#pragma unroll
                        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                            for (int r = 0; r < 2; ++r) {
                                const float e0 = ex2(sc[mt][nb][2 * r] - mu[0]), e1 = ex2(sc[mt][nb][2 * r + 1] - mu[1]);
                                l[nb][0] += e0;
                                l[nb][1] += e1;
                                const __half2 hh = __floats2half2_rn(e0, e1);
                                ph[mt][nb][r] = transpose8(half2_bits(hh));
                                if constexpr (TWO) {
                                    const float2 back = __half22float2(hh);
                                    pl[mt][nb][r] = transpose8(half2_bits(__floats2half2_rn(e0 - back.x, e1 - back.y)));
                                }
                            }
                    }
                    if (!arrived()) { used = issued; break; }
                    const int8_t* vp = sm.ring[warp][used % kSlots];
#pragma unroll
                    for (int hf = 0; hf < DG / 8; ++hf) {  // 8 features of each lane's DG at a time
                        load_fence();
                        uint32_t w[4][4][2];               // 16 keys x 4 of them in this lane x 8 features
#pragma unroll
                        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                            for (int kk = 0; kk < 4; ++kk) {
                                const int key = mt * 16 + (kk >> 1) * 8 + 2 * t + (kk & 1);
                                const uint2 u = *reinterpret_cast<const uint2*>(vp + key * D + g * DG + hf * 8);
                                w[mt][kk][0] = u.x;
                                w[mt][kk][1] = u.y;
                            }
                        float c[2][2][NB][4];
#pragma unroll
                        for (int wd = 0; wd < 2; ++wd)
#pragma unroll
                            for (int u = 0; u < 2; ++u)
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) c[wd][u][nb][e] = 0.0f;
#pragma unroll
                        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                            for (int wd = 0; wd < 2; ++wd) {
                                uint32_t v[2][4];          // [keys 2t.. / 8 + 2t..][feature of the word]
#pragma unroll
                                for (int k2 = 0; k2 < 2; ++k2) {
                                    const uint32_t x = w[mt][2 * k2][wd], y = w[mt][2 * k2 + 1][wd];
                                    v[k2][0] = codes02<false>(__byte_perm(x, y, 0x5410));   // x's byte, y's byte at 0 and 2
                                    v[k2][1] = codes02<false>(__byte_perm(x, y, 0x6521));
                                    v[k2][2] = codes02<false>(__byte_perm(x, y, 0x7632));
                                    v[k2][3] = codes02<false>(__byte_perm(x, y, 0x3743));
                                }
#pragma unroll
                                for (int u = 0; u < 2; ++u)
#pragma unroll
                                    for (int nb = 0; nb < NB; ++nb) {
                                        mma16816(c[wd][u][nb], v[0][2 * u], v[0][2 * u + 1], v[1][2 * u], v[1][2 * u + 1], ph[mt][nb][0], ph[mt][nb][1]);
                                        if constexpr (TWO)
                                            mma16816(c[wd][u][nb], v[0][2 * u], v[0][2 * u + 1], v[1][2 * u], v[1][2 * u + 1], pl[mt][nb][0], pl[mt][nb][1]);
                                    }
                            }
#pragma unroll
                        for (int wd = 0; wd < 2; ++wd)
#pragma unroll
                            for (int u = 0; u < 2; ++u)
#pragma unroll
                                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                                    for (int e = 0; e < 4; ++e) {
                                        float& y = acc[hf * 4 + wd * 2 + u][nb][e];
                                        y = fmaf(vscale, c[wd][u][nb][e], y * al[nb][e & 1]);
                                    }
                    }
                    __syncwarp();
                    ++used;
                    next();
                }
                sub += 32 * kAttWarps;
                if (sub >= p1) break;
                begin();
            }
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float x = l[nb][c];
                x += __shfl_xor_sync(0xffffffffu, x, 4);
                x += __shfl_xor_sync(0xffffffffu, x, 8);
                x += __shfl_xor_sync(0xffffffffu, x, 16);
                if (g == 0) {
                    sm.m[warp][8 * nb + 2 * t + c] = m[nb][c];
                    sm.l[warp][8 * nb + 2 * t + c] = x;
                }
            }
        const bool tail = sm.tail_here != 0;
        if (tail) attend_tail<DT, D, NB>(a);
        else __syncthreads();                              // the ring has been read: it becomes accumulators
#pragma unroll
        for (int i = 0; i < DG / 2; ++i)
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int c = 0; c < 2; ++c)
                    *reinterpret_cast<float2*>(&sm.acc[warp][8 * nb + 2 * t + c][DG * g + 2 * i]) = make_float2(acc[i][nb][c], acc[i][nb][2 + c]);
        __syncthreads();
        // the pieces of this CTA as one: rows straight out, or a partial result per split; four features to a thread
        const int parts = kAttWarps + (tail ? 1 : 0);
        const int n_rows = sm.nrow;
        const bool whole = sm.nu <= 1;
        for (int i = threadIdx.x; i < n_rows * (D / 4); i += kAttWarps * 32) {
            const int r = i / (D / 4), d = i % (D / 4) * 4;
            float mx = -INFINITY;
            for (int p = 0; p < parts; ++p) mx = fmaxf(mx, sm.m[p][r]);
            // NaN scores leave the maximum alone and come out of the sums
            const float mu = mx == -INFINITY ? 0.0f : mx;
            float sum = 0.0f;
            float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            for (int p = 0; p < parts; ++p) {
                const float e = ex2(sm.m[p][r] - mu);
                const float4 x = *reinterpret_cast<const float4*>(&sm.acc[p][r][d]);
                sum = fmaf(e, sm.l[p][r], sum);
                o.x = add_weighted(e, x.x, o.x);
                o.y = add_weighted(e, x.y, o.y);
                o.z = add_weighted(e, x.z, o.z);
                o.w = add_weighted(e, x.w, o.w);
            }
            const size_t gr = (size_t) sm.row[r];
            if (whole) {
                const bool none = sum == 0.0f;
                const float inv = none ? 0.0f : 1.0f / sum;
                st4<DT>(a.out, gr * D + d, none ? 0.0f : o.x * inv, none ? 0.0f : o.y * inv, none ? 0.0f : o.z * inv,
                        none ? 0.0f : o.w * inv, a.out_vec);
                if (a.lse && d == 0) a.lse[gr] = none ? INFINITY : mu + log2f(sum);
            } else {
                const size_t at = (size_t) blockIdx.x * ROWS + r;
                *reinterpret_cast<float4*>(a.part + at * D + d) = o;
                if (d == 0) {
                    float* ml = a.part + (size_t) a.plan.entries * D + at * 2;
                    ml[0] = mx;
                    ml[1] = sum;
                }
            }
        }
    }
}

// The splits' partial results of a row as one: a CTA per row, whose warps take the splits in turn and then meet. The
// partial results lie in L2; a launch that is ready when the pieces end makes it 2 to 3 us. Not made for many rows: 16,000 of
// two splits each (500 tokens behind 3,500, 32 heads) are 124 us, most of them a CTA's start and its loads one after another.
constexpr int kJoinWarps = 8;
template <int DT, int D>
__global__ void __launch_bounds__(kJoinWarps * 32) attend_join(const __grid_constant__ AttendArgs a) {
    __shared__ float so[kJoinWarps][D], sl[kJoinWarps], sx[kJoinWarps];
    const KvArgs& kv = a.kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, group = a.Hq / kv.heads, rows = a.plan.rows;
    const int b = blockIdx.x;
    const Seq s = load_seq(kv, a.starts, a.T, b);
    let_next_launch();
    wait_for_previous();
    if (!s.ok || s.n == 0) return;
    const float* mls = a.part + (size_t) a.plan.entries * D;
    int2 pieces_of = make_int2(0, a.plan.nz);              // this sequence's first piece, the pieces of a unit
    if (rows != 256) pieces_of = reinterpret_cast<const int2*>(mls + (size_t) a.plan.entries * 2)[b];
    if (pieces_of.y <= 1) return;
    // row starts that run backwards can stand for more pieces than the call has rows: the call has reported them, and what
    // was not written is not followed
    const long long units = (long long) ((s.n * group + rows - 1) / rows) * kv.heads;
    if (rows != 256 && (pieces_of.x < 0 || pieces_of.x + units * pieces_of.y > a.plan.grid)) return;
    for (int i = blockIdx.y; i < s.n * a.Hq; i += gridDim.y) {
        const int tok = i / a.Hq, hq = i % a.Hq;
        const int R = s.n * group, row = tok * group + hq % group, tile = row / rows, r0 = tile * rows;
        const int last_pos = s.L - s.n + (min(R, r0 + rows) - 1) / group;
        const Pieces pc = pieces(s.L, last_pos, pieces_of.y);
        if (pc.nu <= 1) continue;
        const size_t gr = (size_t) (s.s0 + tok) * a.Hq + hq;
        // the row's partial results: entries at, at + step, ...
        const size_t step = rows == 256 ? 1 : (size_t) kv.heads * rows;
        const size_t at = rows == 256 ? gr * a.plan.nz
                                      : (size_t) (pieces_of.x + tile * pieces_of.y * kv.heads + hq / group) * rows + (row - r0);
        // each warp its own splits, up to 8 at a time under way
        float m = -INFINITY, sum = 0.0f, o[D / 32];
#pragma unroll
        for (int u = 0; u < D / 32; ++u) o[u] = 0.0f;
        for (int z0 = warp; z0 < pc.nu; z0 += 8 * kJoinWarps) {
            float2 ml[8];
            float x[8][D / 32];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int z = z0 + i * kJoinWarps;
                const size_t w = at + (size_t) min(z, pc.nu - 1) * step;
                ml[i] = *reinterpret_cast<const float2*>(mls + w * 2);
                if (z >= pc.nu) ml[i] = make_float2(-INFINITY, 0.0f);
#pragma unroll
                for (int u = 0; u < D / 32; ++u) x[i][u] = z < pc.nu ? a.part[w * D + lane + 32 * u] : 0.0f;
            }
            float mn = m;
#pragma unroll
            for (int i = 0; i < 8; ++i) mn = fmaxf(mn, ml[i].x);
            const float mu = mn == -INFINITY ? 0.0f : mn, al = ex2(m - mu);
            sum *= al;
#pragma unroll
            for (int u = 0; u < D / 32; ++u) o[u] = add_weighted(al, o[u], 0.0f);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float e = ex2(ml[i].x - mu);
                sum = fmaf(e, ml[i].y, sum);
#pragma unroll
                for (int u = 0; u < D / 32; ++u) o[u] = add_weighted(e, x[i][u], o[u]);
            }
            m = mn;
        }
        __syncthreads();                                   // the row before has been written
        if (lane == 0) {
            sl[warp] = sum;
            sx[warp] = m;
        }
#pragma unroll
        for (int u = 0; u < D / 32; ++u) so[warp][lane + 32 * u] = o[u];
        __syncthreads();
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) mx = fmaxf(mx, sx[w]);
        const float mu = mx == -INFINITY ? 0.0f : mx;
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < kJoinWarps; ++w) sum = fmaf(ex2(sx[w] - mu), sl[w], sum);
        if (threadIdx.x < D) {
            const int d = threadIdx.x;
            float y = 0.0f;
#pragma unroll
            for (int w = 0; w < kJoinWarps; ++w) y = add_weighted(ex2(sx[w] - mu), so[w][d], y);
            st1<DT>(a.out, gr * D + d, sum == 0.0f ? 0.0f : y / sum);
        }
        if (a.lse && threadIdx.x == 0) a.lse[gr] = sum == 0.0f ? INFINITY : mu + log2f(sum);
    }
}

// weight[slot] += the sum over the group's query rows of p = 2^(s - lse): the scores once more, against the finished
// sums. One CTA per (sequence, kv head, piece of the pages), the last piece also the tail; a page's sums stay in one warp.
// Reading the keys again costs less than keeping every score of the first pass would. 16 sequences of 100 to 4,500 tokens,
// 2 heads of 64 with 8 queries each in float32: 13 us of the call's 23, all of its kernels bound by their first loads (here the
// schedulers issue 23 % of the time). Not made for prompts: a row's query is laid out again for every page and 8 rows, and
// 1,999 tokens behind 15,002 (32 heads of 128 over 8, fp16) take 4.24 ms with weights, 0.65 without. Pages that sequences
// share take their sums in any order.
template <int DT, int D>
__global__ void __launch_bounds__(kAttWarps * 32) attend_weights(const __grid_constant__ AttendArgs a, int nzw) {
    constexpr bool TWO = DT == F32;
    constexpr int NB = 1, ROWS = 8;
    __shared__ __align__(16) float qs[ROWS][D];
    __shared__ __align__(16) float sc[kPage][ROWS];
    __shared__ QFrag<D, NB, TWO> fr[kAttWarps];
    __shared__ long long qoff[kAttWarps][ROWS];
    extern __shared__ __align__(16) unsigned char kt[];
    const KvArgs& kv = a.kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    const int group = a.Hq / kv.heads;
    const int z = (int) (blockIdx.x % nzw), h = (int) (blockIdx.x / nzw % kv.heads), b = (int) (blockIdx.x / nzw / kv.heads);
    const Seq s = load_seq(kv, a.starts, a.T, b);
    wait_for_previous();
    if (!s.ok || s.n == 0) return;
    const int R = s.n * group;
    const int full = s.L / kPage;
    auto place = [&](int r, int& pos, long long& off, float& lse) {
        pos = -1;
        off = -1;
        lse = INFINITY;
        if (r >= R) return;
        const int tok = r / group, hq = h * group + r % group;
        pos = s.L - s.n + tok;
        off = (long long) (s.s0 + tok) * a.qs + (long long) hq * D;
        lse = a.lse[(size_t) (s.s0 + tok) * a.Hq + hq];
    };
    for (int p = z * kAttWarps + warp; p < full; p += nzw * kAttWarps) {
        const int page = kv.table[(size_t) b * kv.width + p];
        if (!page_ok(kv, page)) continue;                  // already recorded by the attention
        const size_t pb = (size_t) page * kv.heads + h;
        const float ks = kv.ks[pb];
        float sum[4][2];
#pragma unroll
        for (int mt = 0; mt < 4; ++mt) sum[mt][0] = sum[mt][1] = 0.0f;
        // from the first row that sees slot 64 p on
        for (int r0 = max(0, p * kPage - (s.L - s.n)) * group / ROWS * ROWS; r0 < R; r0 += ROWS) {
            int pos, pos2[2];
            long long off;
            float lse, lse2[2];
            place(r0 + g, pos, off, lse);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                pos2[c] = __shfl_sync(0xffffffffu, pos, 8 * t + 4 * c);
                lse2[c] = __shfl_sync(0xffffffffu, lse, 8 * t + 4 * c);
            }
            __syncwarp();                                  // the rows before have been read
            if (t == 0) qoff[warp][g] = off;
            __syncwarp();
            QRows<DT, D, NB, 32> rows;
            load_q(rows, a.q, qoff[warp], a.q_vec);
            QFrag<D, NB, TWO>& f = fr[warp];
            make_q(f, rows, a.scale_log2);
            __syncwarp();
            float x[4][NB][4];
            page_scores<D, NB, TWO>(f, kv.k + pb * kPage * D, x);
#pragma unroll
            for (int mt = 0; mt < 4; ++mt)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float e = ex2(x[mt][0][i] * (ks * f.rs[2 * t + (i & 1)]) - lse2[i & 1]);
                    if (p * kPage + mt * 16 + (i >> 1) * 8 + g <= pos2[i & 1]) sum[mt][i >> 1] += e;
                }
        }
#pragma unroll
        for (int mt = 0; mt < 4; ++mt)
#pragma unroll
            for (int r = 0; r < 2; ++r) {
                float y = sum[mt][r];
                y += __shfl_xor_sync(0xffffffffu, y, 1);
                y += __shfl_xor_sync(0xffffffffu, y, 2);
                if (t == 0) atomicAdd(&kv.w[pb * kPage + mt * 16 + r * 8 + g], y);
            }
    }
    const int nkey = s.L - full * kPage;
    if (z != nzw - 1 || nkey == 0) return;
    const size_t tb = ((size_t) b * kv.heads + h) * kPage;
    float sum = 0.0f;
    for (int i = threadIdx.x; i < nkey * D * DtInfo<DT>::ES / 16; i += kAttWarps * 32)
        reinterpret_cast<uint4*>(kt)[i] = reinterpret_cast<const uint4*>(static_cast<const char*>(kv.tk) + tb * D * DtInfo<DT>::ES)[i];
    for (int r0 = max(0, full * kPage - (s.L - s.n)) * group / ROWS * ROWS; r0 < R; r0 += ROWS) {
        const int nrow = min(R - r0, ROWS);
        __syncthreads();
        for (int i = threadIdx.x; i < nrow * D; i += kAttWarps * 32) {
            int pos;
            long long off;
            float lse;
            place(r0 + i / D, pos, off, lse);
            qs[i / D][i % D] = ld1<DT>(a.q, (size_t) off + i % D);
        }
        __syncthreads();
        tail_scores<DT, D, ROWS>(qs, kt, nrow, nkey, a.scale_log2, sc);
        __syncthreads();
        if (threadIdx.x < nkey)
            for (int r = 0; r < nrow; ++r) {
                int pos;
                long long off;
                float lse;
                place(r0 + r, pos, off, lse);
                if (full * kPage + (int) threadIdx.x <= pos) sum += ex2(sc[threadIdx.x][r] - lse);
            }
    }
    if (threadIdx.x < nkey) kv.tw[tb + threadIdx.x] += sum;
}

// ---- eviction --------------------------------------------------------------------------------------------------------
// Of a sequence longer than the budget, each kv head keeps its first `sinks` and last `recent` tokens and, of the ones
// between, those with the largest weight (of equal ones the earlier), in their order, budget tokens in all. They are
// quantised again, 64 to a page with a new scale, into the sequence's spare pages.

// weights in an order of whole numbers: larger weight, larger key; NaN below everything
__device__ __forceinline__ uint32_t weight_key(float w) {
    if (w != w) return 0;
    const uint32_t u = __float_as_uint(w == 0.0f ? 0.0f : w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelThreads = 1024;
constexpr int kLeftAlone = INT32_MIN;
constexpr int kSelKeys = 48 * 1024;    // keys that fit shared memory; those of a longer sequence are read again each time

// kept[seq, head, 0..budget): where the kept tokens are, in order: 64 page + place, or -1 - place in the tail;
// kept[..][0] = kLeftAlone where the sequence is left alone. One CTA per
// (sequence, head). The weights' keys are read once into shared memory; the key of the last kept one is found by four
// passes over 8 bits of them each; then every thread counts the kept ones in a run of slots of its own, one scan over
// the threads gives the places, and the runs are written down. Few CTAs with scans in a row bound it: 18 us for 12 sequences
// of 3,500 to 8,111 tokens and 8 heads, 96 CTAs on 148 SMs.
__global__ void __launch_bounds__(kSelThreads) evict_select(const __grid_constant__ KvArgs kv, const int* spare,
                                                            int budget, int sinks, int recent, int* kept, int room) {
    extern __shared__ uint32_t keys[];
    __shared__ int hist[256];
    __shared__ int ssum[32], esum[32];
    __shared__ uint32_t s_prefix;
    __shared__ int s_need;
    const int h = (int) (blockIdx.x % kv.heads), b = (int) (blockIdx.x / kv.heads);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int L = kv.lens[b];
    let_next_launch();
    int* out = kept + (size_t) blockIdx.x * budget;
    const int* table = kv.table + (size_t) b * kv.width;
    const int full = L / kPage;
    if (L <= budget || full > kv.width) {
        if (tid == 0) {
            out[0] = kLeftAlone;
            if (L < 0 || full > kv.width) atomicOr(kv.err, kErrLen);
        }
        return;
    }
    bool bad = false;
    for (int i = tid; i < full; i += kSelThreads) bad |= !page_ok(kv, table[i]);
    for (int i = tid; i < budget / kPage; i += kSelThreads) bad |= !page_ok(kv, spare[(size_t) b * (budget / kPage) + i]);
    if (__syncthreads_or(bad)) {
        if (tid == 0) {
            out[0] = kLeftAlone;
            atomicOr(kv.err, kErrPage);
        }
        return;
    }
    auto read = [&](int slot) {
        const float w = slot < full * kPage ? kv.w[((size_t) table[slot / kPage] * kv.heads + h) * kPage + slot % kPage]
                                            : kv.tw[((size_t) b * kv.heads + h) * kPage + slot - full * kPage];
        return weight_key(w);
    };
    const bool held = L <= room;
    if (held) {
#pragma unroll 4
        for (int i = tid; i < L; i += kSelThreads) keys[i] = read(i);
        __syncthreads();
    }
    auto key = [&](int slot) { return held ? keys[slot] : read(slot); };
    const int lo = sinks, hi = L - recent;                 // sinks + recent <= budget < L: lo < hi
    // the need-th largest key of the middle
    const int middle = budget - sinks - recent;
    uint32_t prefix = 0;
    int need = middle;
    if (need > 0) {
        for (int shift = 24; shift >= 0; shift -= 8) {
            if (tid < 256) hist[tid] = 0;
            __syncthreads();
            for (int i = lo + tid; i < hi; i += kSelThreads) {
                const uint32_t k = key(i);
                if (shift == 24 || (k >> (shift + 8)) == (prefix >> (shift + 8))) atomicAdd(&hist[(k >> shift) & 255], 1);
            }
            __syncthreads();
            if (warp == 0) {                               // from the top: the bin in which the need-th falls
                int mine = 0;
#pragma unroll
                for (int i = 0; i < 8; ++i) mine += hist[255 - lane * 8 - i];
                int above = mine;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int y = __shfl_up_sync(0xffffffffu, above, o);
                    if (lane >= o) above += y;
                }
                above -= mine;                             // keys in higher bins than this lane's
                if (above < need && above + mine >= need) {
                    int left = need - above;
                    for (int i = 0; i < 8; ++i) {
                        const int c = hist[255 - lane * 8 - i];
                        if (left <= c) {
                            s_prefix = prefix | (uint32_t) (255 - lane * 8 - i) << shift;
                            s_need = left;
                            break;
                        }
                        left -= c;
                    }
                }
            }
            __syncthreads();
            prefix = s_prefix;
            need = s_need;
        }
    }
    // now `need` of the keys equal to prefix are kept (the first ones), and all larger ones. A thread's run has an odd
    // length, so that the threads of a warp read different banks.
    const int run = ((L + kSelThreads - 1) / kSelThreads) | 1, i0 = min(L, tid * run), i1 = min(L, i0 + run);
    auto look = [&](int i, bool& sure, bool& equal) {
        sure = i < lo || i >= hi;
        equal = false;
        if (!sure && middle > 0) {
            const uint32_t k = key(i);
            sure = k > prefix;
            equal = k == prefix;
        }
    };
    int n_sure = 0, n_equal = 0;
    for (int i = i0; i < i1; ++i) {
        bool sure, equal;
        look(i, sure, equal);
        n_sure += sure;
        n_equal += equal;
    }
    int before_sure = n_sure, before_equal = n_equal;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, before_sure, o), y = __shfl_up_sync(0xffffffffu, before_equal, o);
        if (lane >= o) {
            before_sure += x;
            before_equal += y;
        }
    }
    if (lane == 31) {
        ssum[warp] = before_sure;
        esum[warp] = before_equal;
    }
    __syncthreads();
    before_sure -= n_sure;
    before_equal -= n_equal;
    for (int w = 0; w < warp; ++w) {
        before_sure += ssum[w];
        before_equal += esum[w];
    }
    int at = before_sure + min(before_equal, need);
    for (int i = i0; i < i1; ++i) {
        bool sure, equal;
        look(i, sure, equal);
        if (sure || (equal && before_equal < need)) out[at++] = i < full * kPage ? table[i / kPage] * kPage + i % kPage : full * kPage - 1 - i;
        before_equal += equal;
    }
}

// 64 kept tokens of a (sequence, head) into one spare page, K and V side by side so that their loads are under way
// together. TAIL: some of them lie in the tail (a sequence's last page or two).
// A kept token's row is 128 bytes anywhere in the old pages. 12 sequences cut to 4,096 tokens, 8 heads of 128, are 188 MB in 89
// us (2.1 TB/s; the bytes alone 29): a CTA's loads, its pass for the maximum (twice, K and V) and its pass for the codes follow
// one another with barriers between, and four CTAs are what an SM holds; the schedulers issue 62 % of the time and wait for
// the barriers and the loads about equally. Both passes take the codes exactly, code x scale in 64 bits where 32 are not
// sure of the rounding.
template <int DT, int D, bool TAIL>
__device__ __forceinline__ void gather_page(const KvArgs& kv, int h, size_t tbase, int page, const int* loc) {
    constexpr int C8 = D / 8, PER = 64 * C8 / 256;
    __shared__ double red[8];
    __shared__ float scale[2][kPage], ratio[2][kPage];
    if (threadIdx.x < 2 * kPage) {
        const int which = threadIdx.x / kPage, at = loc[threadIdx.x % kPage];
        scale[which][threadIdx.x % kPage] = at >= 0 ? (which ? kv.vs : kv.ks)[(size_t) (at / kPage) * kv.heads + h] : 1.0f;
    }
    struct Chunk {
        uint2 c;                       // a page's codes
        Raw8<DT> t[1];                 // or, with TAIL, the tail's values
    } raw[2][PER];
#pragma unroll
    for (int which = 0; which < 2; ++which)
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = threadIdx.x + i * 256, d = c % C8 * 8, at = loc[c / C8];
            if (!TAIL || at >= 0)
                raw[which][i].c = *reinterpret_cast<const uint2*>(
                    (which ? kv.v : kv.k) + (((size_t) (at / kPage) * kv.heads + h) * kPage + at % kPage) * D + d);
            else if constexpr (TAIL)
                raw[which][i].t[0] = raw8<DT>(which ? kv.tv : kv.tk, (tbase - 1 - at) * D + d, true);
        }
    auto values = [&](int which, int i, float (&x)[8]) {
        if (!TAIL || loc[(threadIdx.x + i * 256) / C8] >= 0) {
            const uint32_t w[2] = {raw[which][i].c.x ^ 0x80808080u, raw[which][i].c.y ^ 0x80808080u};
            // code + 128 in the low bits of 2^23
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = __uint_as_float(__byte_perm(w[e / 4], 0x4b000000u, 0x7650 | (e % 4))) - 8388736.0f;
        } else if constexpr (TAIL) {
            floats8(raw[which][i].t[0], x);
        }
    };
    __syncthreads();
    const size_t pb = (size_t) page * kv.heads + h;
#pragma unroll
    for (int which = 0; which < 2; ++which) {
        double top = 0.0;
        bool odd = false;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            float x[8], m = 0.0f;
            values(which, i, x);
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                if (!TAIL || finite(x[u])) m = fmaxf(m, fabsf(x[u]));
                else odd = true;
            }
            const double v = (double) m * (double) scale[which][(threadIdx.x + i * 256) / C8];   // exact: 24 bits times 24 at most
            if (v > top) top = v;
        }
        if (TAIL) odd = __syncthreads_or(odd);
        top = block_max(top, red);
        if (threadIdx.x == 0) (which ? kv.vs : kv.ks)[pb] = (float) (top / 127.0);
        // where a float cannot hold 127 scale / top every code goes the long way
        const bool far = top < 1e-30;
        if (threadIdx.x < kPage) ratio[which][threadIdx.x] = far ? 0.0f : (float) ((double) scale[which][threadIdx.x] * 127.0 / top);
        __syncthreads();
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int c = threadIdx.x + i * 256, r = c / C8, d = c % C8 * 8;
            uint2 o = make_uint2(0, 0);
            float x[8];
            values(which, i, x);
            if (top > 0.0) o = codes8(x, ratio[which][r], (double) scale[which][r], top, odd || far);
            *reinterpret_cast<uint2*>((which ? kv.v : kv.k) + (pb * kPage + r) * D + d) = o;
        }
    }
    if (threadIdx.x < kPage) {
        const int at = loc[threadIdx.x];
        kv.w[pb * kPage + threadIdx.x] = at >= 0 ? kv.w[((size_t) (at / kPage) * kv.heads + h) * kPage + at % kPage] : kv.tw[tbase - 1 - at];
    }
}

template <int DT, int D>
__global__ void __launch_bounds__(256, 4) evict_gather(const __grid_constant__ KvArgs kv, const int* spare, int budget,
                                                       const int* kept) {
    __shared__ int loc[kPage];
    const int nb = budget / kPage, blk = blockIdx.y;
    const int b = (int) (blockIdx.x / kv.heads), h = (int) (blockIdx.x % kv.heads);
    const int* mine = kept + (size_t) blockIdx.x * budget;
    let_next_launch();
    wait_for_previous();
    if (fresh(mine) == kLeftAlone) return;
    const int page = spare[(size_t) b * nb + blk];
    int at = 0;
    if (threadIdx.x < kPage) loc[threadIdx.x] = at = fresh(mine + blk * kPage + threadIdx.x);
    const size_t tbase = (size_t) blockIdx.x * kPage;
    if (__syncthreads_or(at < 0)) gather_page<DT, D, true>(kv, h, tbase, page, loc);
    else gather_page<DT, D, false>(kv, h, tbase, page, loc);
}

// the new pages take the old ones' place in the table, which take theirs among the spare ones
__global__ void __launch_bounds__(256) evict_swap(const KvArgs kv, int* spare, int budget, const int* kept) {
    const int b = (int) blockIdx.x, nb = budget / kPage;
    wait_for_previous();
    if (fresh(kept + (size_t) b * kv.heads * budget) == kLeftAlone) return;
    for (int i = threadIdx.x; i < nb; i += 256) {
        int* p = kv.table + (size_t) b * kv.width + i;
        int* q = spare + (size_t) b * nb + i;
        const int x = *p;
        *p = *q;
        *q = x;
    }
    if (threadIdx.x == 0) kv.lens[b] = budget;
}

}  // namespace

// ---- launchers -------------------------------------------------------------------------------------------------------

template <int DT>
cudaError_t append_dt(const KvArgs& kv, const void* k, const void* v, long long T, long long stride, const int* starts,
                      long long max_new, bool vec, cudaStream_t st) {
    const dim3 grid((unsigned) (kv.seqs * kv.heads), (unsigned) std::min(std::max(1ll, (max_new + kPage - 1) / kPage), 65535ll), 2);
    if (kv.dim == 64) kv_append<DT, 64><<<grid, kAppThreads, 0, st>>>(kv, k, v, T, stride, starts, vec);
    else kv_append<DT, 128><<<grid, kAppThreads, 0, st>>>(kv, k, v, T, stride, starts, vec);
    return cudaGetLastError();
}

cudaError_t launch_kv_append(const KvArgs& kv, const void* k, const void* v, long long T, long long stride, const int* starts,
                             long long max_new, bool vec, cudaStream_t st) {
    switch (kv.dt) {
        case F16: return append_dt<F16>(kv, k, v, T, stride, starts, max_new, vec, st);
        case BF16: return append_dt<BF16>(kv, k, v, T, stride, starts, max_new, vec, st);
        default: return append_dt<F32>(kv, k, v, T, stride, starts, max_new, vec, st);
    }
}

// Rows of a tile by how many rows a sequence brings (new tokens times the heads of a group): up to 8, 16, and for 16-bit
// types from kTcRows on 256, on tcgen05. Tiles of 16 against tcgen05, us, 8 kv heads, at 32 / 48 / 64 / 96 / 128 rows of each:
//   128 wide   1 x 16,384 tokens   26 / 37 / 44 / 61 / 75   against 44 / 47 / 47 / 51 / 54
//              4 x 2,048           31 / 42 / 46 / 47 / 51           38 / 43 / 46 / 55 / 64
//              16 x 300            25 / 48 / 50 / 39 / 57           22 / 22 / 23 / 22 / 22
//   64 wide    1 x 16,384          19 / 25 / 30 / 39 / 49           39 / 39 / 41 / 43 / 43
//              4 x 2,048           22 / 29 / 32 / 31 / 33           31 / 34 / 37 / 43 / 48
//              16 x 300            16 / 30 / 31 / 26 / 37           18 / 18 / 18 / 18 / 18
// and one of 131,072 at 48 / 64 / 128 rows 174 / 213 / 411 against 226 / 226 / 222 (64 wide: 109 / 135 / 259 against 207 / 208 / 204).
// No one number is right for all: 48 is where many short sequences gain half, which for one long sequence costs a quarter up
// to 60 rows, and more with 64-wide heads, up to some 100.
constexpr int64_t kTcRows = 48;
AttendPlan attend_plan(int n_sm, int dt, int64_t seqs, int64_t heads, int64_t group, int64_t T, int64_t max_new, int64_t max_len) {
    AttendPlan p{};
    const int64_t rows = std::min(max_new, T) * group, pages = (max_len + kPage - 1) / kPage;
    p.rows = rows <= 8 ? 8 : dt != F32 && rows >= kTcRows ? 256 : 16;
    // as many tiles as there can be, of all sequences together
    const int64_t tiles = T * group / p.rows + seqs;
    if (p.rows == 256) {
        p.grid = (int) tiles;
        // (at least the tiles that T rows make: with a hint far below them the splits' partial results would grow with both)
        const int64_t units = heads * std::max(seqs * std::max<int64_t>(1, (rows + 255) / 256), T * group / 256);
        p.nz = (int) std::max<int64_t>(1, std::min<int64_t>({(pages + kMinPages - 1) / kMinPages, n_sm / units, 512}));
        p.joined = p.nz > 1;
        p.entries = p.joined ? T * heads * group * p.nz : 0;
        return p;
    }
    // two or three CTAs are resident on an SM. Units that are many, or as short as a piece may be, stay whole. Even batches
    // would rather stay whole from twice the room on (100 sequences of 100 to 1,500 tokens and 8 heads: 49 us whole, 56 cut;
    // 200 of 500 to 3,000: 140 and 152), but one long sequence among many then holds its few CTAs long after the others have
    // ended (the 100 with one of 60,000: 427 us whole, 77 cut; 200: 543 and 116).
    const int64_t room = (int64_t) n_sm * (p.rows == 8 ? 3 : 2), units = tiles * heads;
    p.nz = 1;
    p.joined = units <= 8 * room && 2 * (pages + kTailPages) >= 3 * kChunk;
    // five sixths of that: pieces are rounded up to whole ones, and those that then find no room run after all the others
    // (48 sequences of 200 to 8,191 tokens: 94 us, all of it 100; one of 131,037: 52.1 and 53.3; 48 of 2,048 40.5 both; 16 of 500
    // to 20,000: 73.4 and 73.0)
    p.room = p.joined ? (int) (room * 5 / 6) : 0;
    p.grid = (int) (units + p.room);                       // (the caller has seen to it that it is one)
    p.entries = p.joined ? (units + room) * p.rows : 0;
    return p;
}

template <int DT, int D, int NB>
cudaError_t attend_nb(const AttendArgs& a, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};                 // a bit per device: the attribute belongs to a device
    const cudaError_t e = allow_smem(ready, attend<DT, D, NB>, sizeof(AttSmem<D, NB, DT == F32>));
    if (e != cudaSuccess) return e;
    attend<DT, D, NB><<<(unsigned) a.plan.grid, kAttWarps * 32, sizeof(AttSmem<D, NB, DT == F32>), st>>>(a);
    return cudaGetLastError();
}

template <int DT, int D>
cudaError_t attend_dt(const AttendArgs& a, int n_sm, cudaStream_t st) {
    const KvArgs& kv = a.kv;
    cudaError_t e = a.plan.rows == 256 ? launch_attend_tc(a, st) : a.plan.rows == 8 ? attend_nb<DT, D, 1>(a, st) : attend_nb<DT, D, 2>(a, st);
    if (e != cudaSuccess) return e;
    if (a.plan.joined) {
        const dim3 grid((unsigned) kv.seqs, (unsigned) std::min(a.max_new * a.Hq, 65535ll));
        if ((e = launch_after(attend_join<DT, D>, grid, kJoinWarps * 32, 0, st, a)) != cudaSuccess) return e;
    }
    if (a.lse) {
        const long long units = (long long) kv.seqs * kv.heads;
        const int nzw = (int) std::max(1ll, std::min<long long>((kv.width + kAttWarps - 1) / kAttWarps, (n_sm * 4 + units - 1) / units));
        constexpr size_t tail = (kPage - 1) * D * DtInfo<DT>::ES;
        static std::atomic<uint64_t> ready{0};
        if ((e = allow_smem(ready, attend_weights<DT, D>, tail)) != cudaSuccess) return e;
        e = launch_after(attend_weights<DT, D>, dim3((unsigned) (units * nzw)), kAttWarps * 32, tail, st, a, nzw);
    }
    return e;
}

cudaError_t launch_attend(const AttendArgs& a, int n_sm, cudaStream_t st) {
    const bool narrow = a.kv.dim == 64;
    switch (a.kv.dt) {
        case F16: return narrow ? attend_dt<F16, 64>(a, n_sm, st) : attend_dt<F16, 128>(a, n_sm, st);
        case BF16: return narrow ? attend_dt<BF16, 64>(a, n_sm, st) : attend_dt<BF16, 128>(a, n_sm, st);
        default: return narrow ? attend_dt<F32, 64>(a, n_sm, st) : attend_dt<F32, 128>(a, n_sm, st);
    }
}

template <int DT>
cudaError_t evict_dt(const KvArgs& kv, const int* spare, int budget, const int* kept, cudaStream_t st) {
    const dim3 grid((unsigned) (kv.seqs * kv.heads), (unsigned) (budget / kPage));
    if (kv.dim == 64) return launch_after(evict_gather<DT, 64>, grid, 256, 0, st, kv, spare, budget, kept);
    return launch_after(evict_gather<DT, 128>, grid, 256, 0, st, kv, spare, budget, kept);
}

cudaError_t launch_kv_evict(const KvArgs& kv, int* spare, int budget, int sinks, int recent, int* kept, cudaStream_t st) {
    static std::atomic<uint64_t> ready{0};
    cudaError_t e = allow_smem(ready, evict_select, kSelKeys * 4);
    if (e != cudaSuccess) return e;
    // room for the longest sequence that the table allows, as far as it goes
    const int room = (int) std::min<long long>((long long) kv.width * kPage + kPage, kSelKeys);
    evict_select<<<(unsigned) (kv.seqs * kv.heads), kSelThreads, (size_t) room * 4, st>>>(kv, spare, budget, sinks, recent, kept, room);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    switch (kv.dt) {
        case F16: e = evict_dt<F16>(kv, spare, budget, kept, st); break;
        case BF16: e = evict_dt<BF16>(kv, spare, budget, kept, st); break;
        default: e = evict_dt<F32>(kv, spare, budget, kept, st); break;
    }
    if (e != cudaSuccess) return e;
    return launch_after(evict_swap, dim3((unsigned) kv.seqs), 256, 0, st, kv, spare, budget, kept);
}

}  // namespace h3
