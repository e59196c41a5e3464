// kvcommon.cuh - what the kernels over the 8-bit key/value cache share: a sequence's bounds, loads of eight values of a
// type, and how the keys of a query tile are divided.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "attn_common.cuh"
#include "kvcache.cuh"
#include "prepass.cuh"

namespace h3 {

// The kernels of one call after its first are launched while the one before still runs (launch_after): they wait here for
// all of it, and every kernel that one follows lets it be launched from its start on. Between calls nothing changes.
// What they read of the one before they read through no const __restrict__ pointer: that would promise that nobody writes
// there while the kernel runs, and lets the compiler load ahead of the wait.
__device__ __forceinline__ void wait_for_previous() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_launch() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
template <typename... P, typename... A>
cudaError_t launch_after(void (*kernel)(P...), dim3 grid, unsigned threads, size_t smem, cudaStream_t st, A... args) {
    cudaLaunchConfig_t c{};
    c.gridDim = grid;
    c.blockDim = dim3(threads);
    c.dynamicSmemBytes = smem;
    c.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    c.attrs = at;
    c.numAttrs = 1;
    return cudaLaunchKernelEx(&c, kernel, static_cast<P>(args)...);
}

// Sequence b's new rows [s0, s0 + n) and its length L, checked against the call's rows and the table's width.
struct Seq {
    int s0, n, L;
    bool ok;
};
__device__ __forceinline__ Seq load_seq(const KvArgs& kv, const int* starts, long long T, int b) {
    Seq s;
    s.s0 = starts[b];
    const int s1 = starts[b + 1];
    s.n = s1 - s.s0;
    s.L = kv.lens[b];
    s.ok = s.s0 >= 0 && s1 >= s.s0 && s1 <= T && s.L >= 0 && s.L / kPage <= kv.width;
    return s;
}
// A load that stays where it is written, and sees what was written before a wait_for_previous().
__device__ __forceinline__ int fresh(const int* p) {
    int x;
    asm volatile("ld.relaxed.gpu.global.s32 %0, [%1];" : "=r"(x) : "l"(__cvta_generic_to_global(p)) : "memory");
    return x;
}
__device__ __forceinline__ int quotient(int x, int d, int shift) { return shift >= 0 ? x >> shift : x / d; }   // x >= 0
__device__ __forceinline__ bool page_ok(const KvArgs& kv, int page) { return page >= 0 && page < kv.pages; }

template <int DT>
__device__ __forceinline__ void st1(void* p, size_t i, float x) {
    if constexpr (DT == F16) reinterpret_cast<__half*>(p)[i] = __float2half_rn(x);
    else if constexpr (DT == BF16) reinterpret_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
    else reinterpret_cast<float*>(p)[i] = x;
}
// 8 consecutive values at element i, with 16-byte loads where vec
template <int DT>
__device__ __forceinline__ void ld8(const void* p, size_t i, bool vec, float* x) {
    if (vec) {
        const char* c = reinterpret_cast<const char*>(p) + i * DtInfo<DT>::ES;
        ld16<DT>(c, x);
        if constexpr (DT == F32) ld16<DT>(c + 16, x + 4);
    } else {
#pragma unroll
        for (int u = 0; u < 8; ++u) x[u] = ld1<DT>(p, i + u);
    }
}

// 8 values as they lie in memory, and as floats
template <int DT>
struct Raw8 {
    uint4 u[DT == F32 ? 2 : 1];
};
template <int DT>
__device__ __forceinline__ Raw8<DT> raw8(const void* p, size_t i, bool vec) {
    Raw8<DT> r;
    const char* c = reinterpret_cast<const char*>(p) + i * DtInfo<DT>::ES;
    if (vec) {
        r.u[0] = *reinterpret_cast<const uint4*>(c);
        if constexpr (DT == F32) r.u[1] = *reinterpret_cast<const uint4*>(c + 16);
    } else {
        uint32_t w[8] = {};
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if constexpr (DT == F32) w[u] = reinterpret_cast<const uint32_t*>(c)[u];
            else w[u / 2] |= (uint32_t) reinterpret_cast<const uint16_t*>(c)[u] << (16 * (u & 1));
        }
        r.u[0] = make_uint4(w[0], w[1], w[2], w[3]);
        if constexpr (DT == F32) r.u[1] = make_uint4(w[4], w[5], w[6], w[7]);
    }
    return r;
}
template <int DT>
__device__ __forceinline__ void floats8(const Raw8<DT>& r, float (&x)[8]) {
    cvt16<DT>(r.u[0], x);
    if constexpr (DT == F32) cvt16<DT>(r.u[1], x + 4);
}

__device__ __forceinline__ bool finite(float x) { return fabsf(x) <= 3.402823466e38f; }
// o + e x for a weight e that may have come out 0 for being small: an infinity (or a NaN) in x is one in o all the same
__device__ __forceinline__ float add_weighted(float e, float x, float o) { return finite(x) ? fmaf(e, x, o) : o + x; }

// The keys that a tile of query rows sees, and how they are divided: np whole pages in pieces of cz pages, and the tail
// (when seen) as a piece of its own, or with the last piece where no split is left.
struct Pieces {
    int np, cz, nu, tail_at;           // nu pieces; the tail is read by piece tail_at (-1: not seen)
};
constexpr int kMinPages = 4;           // a piece has at least a page for each of attend's warps, two key tiles of attend_tc's
__device__ __forceinline__ Pieces pieces(int L, int last_pos, int nz) {
    Pieces p;
    const int seen = min(L, last_pos + 1), full = L / kPage;
    if (seen <= 0) { p.np = 0; p.cz = 1; p.nu = 0; p.tail_at = -1; return p; }
    p.np = min(full, (seen + kPage - 1) / kPage);
    p.cz = max(kMinPages, nz == 1 ? p.np : (p.np + nz - 1) / nz);
    const int nc = nz == 1 ? (p.np > 0) : (p.np + p.cz - 1) / p.cz;
    const bool tail = seen > full * kPage;
    p.nu = tail ? min(nc + 1, nz) : nc;
    p.tail_at = tail ? p.nu - 1 : -1;
    return p;
}

}  // namespace h3
